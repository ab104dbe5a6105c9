"""nrs_dropout_forward / _backward: the mask word for word, and the bits of
the kept values (one f32 product, one f32 sum)."""
import numpy as np
import pytest

import philox

pytestmark = pytest.mark.gpu


def keep_mask(n, p, seed, call):
    return philox.words(n, seed, call) >= np.uint64(int(float(np.float32(p)) * 2 ** 32 + 0.5))


def expected(x, add, p, seed, call):
    p = np.float32(p)
    inv = np.float32(1.0 / (1.0 - float(p))) if p < 1 else np.float32(0)
    with np.errstate(all="ignore"):
        v = np.where(keep_mask(x.size, p, seed, call), x * inv, np.float32(0)).astype(np.float32)
        return v if add is None else (v + add).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 63, 255, 1000, 4096, 100003, 2100001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_bits(hip, n, p):
    rng = np.random.default_rng(n)
    x, res, grad, old = (rng.standard_normal(n).astype(np.float32) for _ in range(4))
    seed, call = 0x0123456789ABCDEF + n, 2 ** 40 + 3
    print(f"dropout {n} p {p}", flush=True)
    up = hip.DeviceBuffer.from_host
    out = up(np.full(n, np.nan, np.float32))
    hip.dropout_forward(out, up(x), None, n, p, seed, call)
    assert np.array_equal(out.to_host(), expected(x, None, p, seed, call))
    hip.dropout_forward(out, up(x), up(res), n, p, seed, call)
    assert np.array_equal(out.to_host(), expected(x, res, p, seed, call))
    gin = up(np.full(n, np.nan, np.float32))
    hip.dropout_backward(gin, up(grad), n, p, seed, call)
    assert np.array_equal(gin.to_host(), expected(grad, None, p, seed, call))
    gin = up(old)
    hip.dropout_backward(gin, up(grad), n, p, seed, call, beta=1.0)
    assert np.array_equal(gin.to_host(), expected(grad, old, p, seed, call))


def test_any_alignment_and_in_place(hip):
    n, p, seed, call = 1003, 0.3, 5, 6
    x, r = (np.random.default_rng(s).standard_normal(n + 8).astype(np.float32) for s in (1, 2))
    for at in range(4):
        for ra in range(2):
            d_x, d_r = hip.DeviceBuffer.from_host(x), hip.DeviceBuffer.from_host(r)
            hip.dropout_forward(d_x.ptr + 4 * at, d_x.ptr + 4 * at, d_r.ptr + 4 * ra, n, p, seed, call)
            want = x.copy()
            want[at:at + n] = expected(x[at:at + n], r[ra:ra + n], p, seed, call)
            assert np.array_equal(d_x.to_host(), want)
    d_x, d_r = hip.DeviceBuffer.from_host(x), hip.DeviceBuffer.from_host(r)
    hip.dropout_forward(d_r, d_x, d_r, n, p, seed, call)  # out over the residual
    want = r.copy()
    want[:n] = expected(x[:n], r[:n], p, seed, call)
    assert np.array_equal(d_r.to_host(), want)


def test_dropped_values_may_be_anything(hip):
    n = 4096
    x = np.full(n, np.nan, np.float32)
    kept = keep_mask(n, 0.5, 9, 1)
    x[kept] = 1.0
    x[np.flatnonzero(~kept)[::2]] = np.inf
    out = hip.DeviceBuffer(n)
    hip.dropout_forward(out, hip.DeviceBuffer.from_host(x), None, n, 0.5, 9, 1)
    assert np.array_equal(out.to_host(), np.where(kept, np.float32(2), np.float32(0)))


def test_step_is_added_to_the_call(hip):
    n, p = 5000, 0.4
    x = np.ones(n, np.float32)
    d_x, out = hip.DeviceBuffer.from_host(x), hip.DeviceBuffer(n)
    for step, call in ((0, 3), (5, 3), (2 ** 33, 2 ** 63), (2 ** 64 - 2, 3)):  # wraps at 2^64
        d_step = hip.DeviceBuffer.from_host(np.array([step], np.uint64), np.uint64)
        hip.dropout_forward(out, d_x, None, n, p, 11, call, d_step)
        assert np.array_equal(out.to_host(), expected(x, None, p, 11, step + call))


def test_past_32_bits_of_elements(hip):
    """The words of the last elements of a call of more than 2^32 of them."""
    n, p, seed, call = 2 ** 32 + 37, 0.25, 21, 4
    tail = 4096
    buf = hip.DeviceBuffer(n)
    hip.call("nrs_memset_zero", buf.ptr, 4 * n)
    ones = np.ones(tail, np.float32)
    hip.call("nrs_memcpy_htod", buf.ptr + 4 * (n - tail), ones.ctypes.data, ones.nbytes)
    hip.dropout_forward(buf, buf, None, n, p, seed, call)
    got = np.empty(tail, np.float32)
    hip.call("nrs_memcpy_dtoh", got.ctypes.data, buf.ptr + 4 * (n - tail), got.nbytes)
    kept = philox.words(tail, seed, call, n - tail) >= np.uint64(2 ** 30)
    assert np.array_equal(got, np.where(kept, np.float32(1.0 / 0.75), np.float32(0)))
    buf.free()
    hip.call("nrs_empty_cache")


def test_gradient_against_differences(hip):
    """Dropout is linear: f(x + d) - f(x - d) is 2 d times the gradient, on
    small integers and p = 1/2 without rounding."""
    n = 1001
    rng = np.random.default_rng(3)
    x, d = (rng.integers(-9, 10, n).astype(np.float32) for _ in range(2))
    outs = []
    for sign in (1, -1):
        out = hip.DeviceBuffer(n)
        hip.dropout_forward(out, hip.DeviceBuffer.from_host(x + sign * d), None, n, 0.5, 8, 2)
        outs.append(out.to_host())
    gin = hip.DeviceBuffer(n)
    hip.dropout_backward(gin, hip.DeviceBuffer.from_host(np.ones(n, np.float32)), n, 0.5, 8, 2)
    assert np.array_equal((outs[0] - outs[1]) / 2, d * gin.to_host())
