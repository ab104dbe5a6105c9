"""nrs_rotary_forward / _backward against complex numbers in 64 bits.

Tolerance: cos and sin are rounded from an angle that is off by 2^-30 of a turn at
most here (64-bit products of turns up to 2^20, then a rounding to a float of at most
half a turn: 2^-26), and have two units of 2^-24 of their own; a product and a sum
round once each: 2^-24 (|a| + |b|) times 2 (products, sum) + 2 (functions) + 2 pi 2^-2
(angle) < 6.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def turned(x, positions, freq, axis, heads, d, pairs, interleaved, sign=1.0):
    rows = x.shape[0]
    y = x[:, :heads * d].astype(np.float64).reshape(rows, heads, d).copy()
    size = np.abs(y)
    for j in range(pairs):
        a = 0 if axis is None else axis[j]
        if a < 0 or a >= positions.shape[0]:
            continue
        angle = sign * positions[a].astype(np.float64) * float(freq[j])
        c = (2 * j, 2 * j + 1) if interleaved else (j, pairs + j)
        z = (y[:, :, c[0]] + 1j * y[:, :, c[1]]) * np.exp(1j * angle)[:, None]
        both = size[:, :, c[0]] + size[:, :, c[1]]
        y[:, :, c[0]], y[:, :, c[1]] = z.real, z.imag
        size[:, :, c[0]] = size[:, :, c[1]] = both
    return y.reshape(rows, heads * d), 6 * U * size.reshape(rows, heads * d)


def inputs(rows, heads, d, pairs, axes, seed, far=100000, pad=0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, heads * d + pad)).astype(np.float32)
    positions = rng.integers(-far, far, (axes, rows)).astype(np.int32)
    freq = (10000.0 ** -(np.arange(pairs) / max(1, pairs))).astype(np.float32)
    axis = rng.integers(0, axes, max(1, pairs)).astype(np.int32)
    return x, positions, freq, axis


def upload(hip, *arrays):
    return [None if a is None else hip.DeviceBuffer.from_host(a, a.dtype) for a in arrays]


CASES = [
    # rows, heads, d_head, pairs, axes
    (1, 1, 2, 1, 1), (3, 2, 16, 8, 1), (5, 3, 32, 16, 2), (17, 4, 24, 9, 3), (33, 5, 7, 3, 1),
    (2, 1, 1, 0, 1), (100, 8, 64, 20, 3), (9, 2, 80, 40, 2), (257, 3, 128, 64, 1), (4, 40, 33, 16, 2),
    (1000, 20, 12, 5, 4), (64, 1, 200, 99, 2), (3, 7, 9, 4, 1),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_backward(hip, case, interleaved):
    rows, heads, d, pairs, axes = case
    x, pos, freq, axis = inputs(rows, heads, d, pairs, axes, seed=sum(case), pad=3)
    n = heads * d
    dx, dpos, dfreq, daxis = upload(hip, x, pos, freq, axis)
    print(f"rotary {case} {interleaved}", flush=True)
    out = hip.DeviceBuffer.from_host(np.full((rows, n + 5), 7.0))
    hip.rotary_forward(out, dx, dpos, dfreq, daxis, *case, n + 3, n + 5, interleaved=interleaved)
    got = out.to_host((rows, n + 5))
    want, tol = turned(x, pos, freq, axis, heads, d, pairs, interleaved)
    assert np.all(np.abs(got[:, :n] - want) <= tol)
    assert np.all(got[:, n:] == 7.0)
    rng = np.random.default_rng(1)
    old = rng.standard_normal((rows, n + 5)).astype(np.float32)
    want, tol = turned(x, pos, freq, axis, heads, d, pairs, interleaved, -1.0)
    for beta in (0.0, 1.0, -0.5):
        start = old.copy()
        if beta == 0.0:
            start[:, :n] = np.nan
        gin = hip.DeviceBuffer.from_host(start)
        hip.rotary_backward(gin, dx, dpos, dfreq, daxis, *case, n + 5, n + 3,
                            interleaved=interleaved, beta=beta)
        got = gin.to_host((rows, n + 5))
        was = beta * old[:, :n].astype(np.float64)
        assert np.all(np.abs(got[:, :n] - (want + was)) <= tol + 2 * U * (np.abs(want) + np.abs(was)))
        assert np.array_equal(got[:, n:], old[:, n:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_has_the_same_bits(hip, interleaved):
    case = (77, 6, 40, 13, 2)
    x, pos, freq, axis = inputs(*case, seed=3)
    dx, dpos, dfreq, daxis = upload(hip, x, pos, freq, axis)
    out = hip.DeviceBuffer(x.size)
    hip.rotary_forward(out, dx, dpos, dfreq, daxis, *case, 240, 240, interleaved=interleaved)
    hip.rotary_forward(dx, dx, dpos, dfreq, daxis, *case, 240, 240, interleaved=interleaved)
    assert np.array_equal(out.to_host(), dx.to_host())
    hip.rotary_backward(out, dx, dpos, dfreq, daxis, *case, 240, 240, interleaved=interleaved)
    hip.rotary_backward(dx, dx, dpos, dfreq, daxis, *case, 240, 240, interleaved=interleaved)
    assert np.array_equal(out.to_host(), dx.to_host())


def test_axes_out_of_range_are_not_turned(hip):
    case = (11, 2, 16, 8, 2)
    x, pos, freq, _ = inputs(*case, seed=4)
    axis = np.array([0, 1, -1, 2, 1, 2 ** 31 - 1, -2 ** 31, 0], np.int32)
    bufs = upload(hip, x, pos, freq, axis)
    out = hip.DeviceBuffer(x.size)
    hip.rotary_forward(out, *bufs, *case, 32, 32)
    want, tol = turned(x, pos, freq, axis, 2, 16, 8, False)
    assert np.all(np.abs(out.to_host(x.shape) - want) <= tol)
    y, z = out.to_host((11, 2, 16)), x.reshape(11, 2, 16)
    for j in (2, 3, 5, 6):
        assert np.array_equal(y[:, :, [j, 8 + j]], z[:, :, [j, 8 + j]])


def test_no_axis_means_the_first(hip):
    case = (11, 2, 16, 8, 1)
    x, pos, freq, axis = inputs(*case, seed=5)
    bufs = upload(hip, x, pos, freq, axis)
    out = [hip.DeviceBuffer(x.size) for _ in range(2)]
    hip.rotary_forward(out[0], *bufs, *case, 32, 32)
    hip.rotary_forward(out[1], *bufs[:3], None, *case, 32, 32)
    assert np.array_equal(out[0].to_host(), out[1].to_host())


def test_far_positions(hip):
    """At the ends of int32 an angle of 2^31 / 2 pi turns has 2^-53 of itself: 2^-24
    of a turn, 2 pi 2^-24 in the results beside what is counted above."""
    case = (8, 1, 4, 2, 1)
    x, _, _, _ = inputs(*case, seed=6)
    pos = np.array([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 10 ** 9 + 7, -10 ** 8]], np.int32)
    freq = np.array([1.0, 0.123456789], np.float32)
    bufs = upload(hip, x, pos, freq)
    out = hip.DeviceBuffer(x.size)
    hip.rotary_forward(out, *bufs, None, *case, 4, 4)
    want, tol = turned(x, pos, freq, None, 1, 4, 2, False)
    # the reference's own angle, in 64 bits too, is off by as much
    assert np.all(np.abs(out.to_host(x.shape) - want) <= tol + 2 * 2 * np.pi * U * np.abs(x).max() * 2)


def test_lengths_are_kept(hip):
    """Zero angle leaves the bits; any angle keeps NaN and infinities in their pair."""
    case = (4, 2, 8, 4, 1)
    x, pos, freq, axis = inputs(*case, seed=7)
    x[1, 2], x[2, 13] = np.nan, np.inf
    pos[:] = 0
    bufs = upload(hip, x, pos, freq)
    out = hip.DeviceBuffer(x.size)
    hip.rotary_forward(out, *bufs, None, *case, 16, 16)
    got = out.to_host(x.shape)
    other = np.ones(x.shape, bool)
    for r, c in ((1, 2), (1, 6), (2, 13), (2, 9)):
        other[r, c] = False
    assert np.array_equal(got[other], x[other])


def test_positions_past_2_31_floats(hip):
    """Rows whose offsets pass 32 bits: two million rows of a stride of 2048."""
    rows, ld = 2 ** 21 + 5, 1024
    x = hip.DeviceBuffer(rows * ld)
    hip.call("nrs_memset_zero", x, rows * ld * 4)
    tail = np.arange(1, 9, dtype=np.float32)
    hip.call("nrs_memcpy_htod", x.ptr + (rows - 1) * ld * 4, tail.ctypes.data, 32)
    pos = np.full((1, rows), 5, np.int32)
    freq = np.array([1.0, 0.5], np.float32)
    dpos, dfreq = upload(hip, pos, freq)
    hip.rotary_forward(x, x, dpos, dfreq, None, rows, 1, 8, 2, 1, ld, ld)
    got = np.empty(8, np.float32)
    hip.call("nrs_memcpy_dtoh", got.ctypes.data, x.ptr + (rows - 1) * ld * 4, 32)
    want, tol = turned(tail[None], pos[:, -1:], freq, None, 1, 8, 2, False)
    assert np.all(np.abs(got - want[0]) <= tol[0])
    x.free()
    hip.call("nrs_empty_cache")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
def test_bad_numbers_stay_in_their_pair(hip, bad, interleaved):
    """Turned by angles that are not zero: the other pairs of the row, of its heads and of
    other rows, and the columns that are not turned, keep their bits; both ways."""
    case = (5, 2, 22, 10, 2)  # two columns of a head are copied
    x, pos, freq, axis = inputs(*case, seed=8)
    pos[pos == 0] = 1
    clean, dirty = x.copy(), x.copy()
    partner = lambda c: (c // 2 * 2 + 1 - c % 2) if interleaved else (c + 10) % 20
    hit = np.zeros(x.shape, bool)
    for row, head, c in ((1, 0, 2), (2, 1, 13), (2, 0, 0), (4, 1, 19), (3, 0, 9)):
        dirty[row, head * 22 + c] = bad
        hit[row, [head * 22 + c, head * 22 + partner(c)]] = True
    dirty[0, 21] = bad  # copied: alone
    hit[0, 21] = True
    _, dpos, dfreq, daxis = upload(hip, x, pos, freq, axis)
    for turn in (hip.rotary_forward, hip.rotary_backward):
        got = []
        for a in (clean, dirty):
            out = hip.DeviceBuffer(a.size)
            turn(out, upload(hip, a)[0], dpos, dfreq, daxis, *case, 44, 44, interleaved=interleaved)
            got.append(out.to_host(a.shape))
        assert np.isfinite(got[0]).all()
        assert np.array_equal(got[0][~hit], got[1][~hit])
        assert not np.isfinite(got[1][hit]).any()
