"""nrs_embedding_forward / _backward against the definition in 64 bits.

The forward rounds one product: exact against an f32 product. The gradient of
a token that n positions hold is a sum of n floats in some fixed order, times
the scale, plus beta times the old value: off by at most (n + 2) half steps
(2^-24) of the sum of magnitudes, and one of the old value's product."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make_ids(rng, count, vocab, how):
    if how == "uniform":
        return rng.integers(0, vocab, count).astype(np.int32)
    if how == "one":
        return np.full(count, vocab - 1, np.int32)
    if how == "outside":  # every id beyond the table, at either side
        return rng.choice([-1, vocab, -2 ** 31, 2 ** 31 - 1, -vocab], count).astype(np.int32)
    # word frequencies fall off as one over their rank, with padding
    rank = np.minimum((np.exp(rng.random(count) * np.log(vocab + 1.0)) - 1).astype(np.int64), vocab - 1)
    ids = rng.permutation(vocab)[rank].astype(np.int32)
    ids[rng.random(count) < 0.1] = -1
    return ids


def reference(ids, grad, vocab, scale):
    """Sums, sums of magnitudes and counts per token, in 64 bits."""
    keep = (ids >= 0) & (ids < vocab)
    order = np.flatnonzero(keep)[np.argsort(ids[keep], kind="stable")]
    total, size = np.zeros((vocab, grad.shape[1])), np.zeros((vocab, grad.shape[1]))
    n = np.bincount(ids[keep], minlength=vocab)
    if len(order):
        starts = np.concatenate([[0], np.cumsum(n)])[:-1][n > 0]
        g = grad[order].astype(np.float64)
        total[n > 0] = np.add.reduceat(g, starts, axis=0)
        size[n > 0] = np.add.reduceat(np.abs(g), starts, axis=0)
    return scale * total, abs(scale) * size, n


CASES = [
    (1, 1, 1, "uniform"), (5, 3, 7, "uniform"), (64, 10, 16, "zipf"), (100, 1000, 33, "zipf"),
    (257, 2, 256, "uniform"), (1000, 1, 12, "one"), (4096, 512, 260, "zipf"),
    (3000, 70000, 64, "uniform"), (2000, 50021, 1000, "zipf"), (300, 40, 5, "outside"),
    (20000, 259, 128, "zipf"), (9000, 100, 30, "one"), (70001, 33000, 9, "zipf"),
    (513, 513, 2048, "zipf"), (63, 4000, 1027, "uniform"), (100000, 17, 3, "uniform"),
    (256, 1, 4096, "one"), (256, 1500, 70, "zipf"), (250, 20, 4100, "zipf"), (256, 3000, 1025, "uniform"),
    (200, 3000, 5, "one"), (255, 9, 130, "outside"), (130, 5000, 2, "zipf"),
]


@pytest.mark.parametrize("count,vocab,dim,how", CASES)
def test_forward_and_backward(hip, count, vocab, dim, how):
    rng = np.random.default_rng(count + vocab)
    ids = make_ids(rng, count, vocab, how)
    table = rng.standard_normal((vocab, dim)).astype(np.float32)
    grad = rng.standard_normal((count, dim)).astype(np.float32)
    scale = np.float32(np.sqrt(dim))
    print(f"embedding {count} of {vocab} x {dim} {how}", flush=True)
    d_ids, d_table, d_grad = (hip.DeviceBuffer.from_host(x, x.dtype) for x in (ids, table, grad))
    out = hip.DeviceBuffer.from_host(np.full((count, dim), np.nan, np.float32))
    hip.embedding_forward(out, d_table, d_ids, count, vocab, dim, scale)
    keep = ((ids >= 0) & (ids < vocab))[:, None]
    want = np.where(keep, table[np.where(keep[:, 0], ids, 0)] * scale, np.float32(0))
    assert np.array_equal(out.to_host((count, dim)), want)

    value, size, n = reference(ids, grad, vocab, float(scale))
    old = rng.standard_normal((vocab, dim)).astype(np.float32)
    for beta in (0.0, 1.0, 0.5):
        start = np.full_like(old, np.nan) if beta == 0.0 else old
        dtable = hip.DeviceBuffer.from_host(start)
        hip.embedding_backward(dtable, d_grad, d_ids, count, vocab, dim, scale, beta)
        got = dtable.to_host((vocab, dim))
        was = beta * old.astype(np.float64) if beta else np.zeros_like(value)
        tol = (n[:, None] + 4) * U * (size + np.abs(was)) + 1e-37
        bad = ~(np.abs(got - (value + was)) <= tol)
        assert not bad.any(), (beta, np.argwhere(bad)[:3], bad.sum())
        if beta == 1.0:
            assert np.array_equal(got[n == 0], old[n == 0])
        if beta == 0.0:
            assert np.all(got[n == 0] == 0)
        # the same bits again
        hip.call("nrs_memcpy_htod", dtable.ptr, start.ctypes.data, start.nbytes)
        hip.embedding_backward(dtable, d_grad, d_ids, count, vocab, dim, scale, beta)
        assert np.array_equal(dtable.to_host((vocab, dim)), got)


def test_integer_sums_are_exact(hip):
    """Small integers add without rounding, in any order."""
    rng = np.random.default_rng(2)
    count, vocab, dim = 30011, 97, 40
    ids = make_ids(rng, count, vocab, "zipf")
    grad = rng.integers(-8, 9, (count, dim)).astype(np.float32)
    value, _, _ = reference(ids, grad, vocab, 2.0)
    dtable = hip.DeviceBuffer(vocab * dim)
    hip.embedding_backward(dtable, hip.DeviceBuffer.from_host(grad),
                           hip.DeviceBuffer.from_host(ids, np.int32), count, vocab, dim, 2.0)
    assert np.array_equal(dtable.to_host((vocab, dim)), value.astype(np.float32))


def test_no_tokens(hip):
    old = np.arange(12, dtype=np.float32).reshape(4, 3)
    for beta in (0.0, 1.0, 2.0):
        dtable = hip.DeviceBuffer.from_host(old)
        hip.embedding_backward(dtable, None, None, 0, 4, 3, 1.0, beta)
        assert np.array_equal(dtable.to_host((4, 3)), beta * old)
    hip.embedding_forward(None, None, None, 0, 4, 3)


def test_unaligned_rows(hip):
    """Buffers that start at any float."""
    rng = np.random.default_rng(3)
    count, vocab, dim = 200, 50, 36
    ids = make_ids(rng, count, vocab, "zipf")
    table, grad = (rng.standard_normal((n, dim)).astype(np.float32) for n in (vocab, count))
    d_ids = hip.DeviceBuffer.from_host(np.concatenate([[7], ids]).astype(np.int32), np.int32)
    d_table = hip.DeviceBuffer.from_host(np.concatenate([[1, 2, 3], table.ravel()]))
    d_grad = hip.DeviceBuffer.from_host(np.concatenate([[1], grad.ravel()]))
    out, dtable = hip.DeviceBuffer.zeros(count * dim + 2), hip.DeviceBuffer.zeros(vocab * dim + 3)
    hip.embedding_forward(out.ptr + 4, d_table.ptr + 12, d_ids.ptr + 4, count, vocab, dim, 3.0)
    got = out.to_host()
    want = np.where((ids >= 0)[:, None], table[np.maximum(ids, 0)] * np.float32(3), np.float32(0))
    assert np.array_equal(got[1:-1].reshape(count, dim), want) and got[0] == 0 and got[-1] == 0
    hip.embedding_backward(dtable.ptr + 4, d_grad.ptr + 4, d_ids.ptr + 4, count, vocab, dim, 1.0)
    got = dtable.to_host()
    value, size, n = reference(ids, grad, vocab, 1.0)
    assert np.all(np.abs(got[1:-2].reshape(vocab, dim) - value) <= (n[:, None] + 4) * U * size + 1e-37)
    assert got[0] == 0 and np.all(got[-2:] == 0)


def test_own_scratch(hip):
    rng = np.random.default_rng(4)
    for count, vocab, dim in ((5000, 300, 64), (33, 20000, 16), (40000, 2000, 100)):
        ids = make_ids(rng, count, vocab, "zipf")
        grad = hip.DeviceBuffer.from_host(rng.standard_normal((count, dim)).astype(np.float32))
        d_ids = hip.DeviceBuffer.from_host(ids, np.int32)
        a, b = hip.DeviceBuffer(vocab * dim), hip.DeviceBuffer(vocab * dim)
        hip.embedding_backward(a, grad, d_ids, count, vocab, dim)
        need = hip.embedding_workspace(count, vocab, dim)
        fill = np.full((need + 3) // 4 + 64, np.float32(7))
        work = hip.DeviceBuffer.from_host(fill)
        hip.embedding_backward(b, grad, d_ids, count, vocab, dim, work=work)
        assert np.array_equal(a.to_host(), b.to_host())
        assert np.all(work.to_host()[(need + 3) // 4:] == 7)


# Long runs of one token, over many tiles and several blocks of columns, beside
# the cases above.
LONG = [(30000, 1, 515, "one"), (20011, 3, 600, "uniform"), (300000, 5, 300, "uniform"),
        (65536, 259, 512, "zipf"), (12345, 7, 257, "zipf"), (1100, 2, 1024, "uniform"),
        # more tokens than 1024 for each of 256 workgroups, and very wide rows
        (5000, 300007, 8, "zipf"), (70000, 2000003, 3, "uniform"), (300, 4, 20000, "uniform"),
        (2, 3, 100001, "one"),
        # a workgroup's tokens just fit, and do not fit, a wave's registers and the LDS
        (16385, 16384, 20, "zipf"), (16384, 16640, 20, "zipf"), (3001, 262144, 5, "uniform"),
        (3001, 262145, 5, "zipf"), (256, 16385, 9, "zipf"), (257, 2, 1030, "uniform")]


@pytest.mark.parametrize("count,vocab,dim,how", CASES + LONG)
@pytest.mark.parametrize("beta", [0.0, 1.0, 0.5])
def test_integer_gradients_are_exact(hip, count, vocab, dim, how, beta):
    """Integers of up to 8, at most 300000 of them to a sum, whose partial sums
    all lie below 2^24: no order rounds, and a row that is lost or taken twice
    shows. The scale is a power of two and the old values are even. The scratch holds
    NaN: nothing is read that the call did not write."""
    rng = np.random.default_rng(count + dim)
    ids = make_ids(rng, count, vocab, how)
    grad = rng.integers(-8, 9, (count, dim)).astype(np.float32)
    old = 2 * rng.integers(-50, 51, (vocab, dim)).astype(np.float32)
    print(f"embedding, integers, {count} of {vocab} x {dim} {how} beta {beta}", flush=True)
    value, _, _ = reference(ids, grad, vocab, 2.0)
    dtable = hip.DeviceBuffer.from_host(old if beta else np.full_like(old, np.nan))
    work = hip.DeviceBuffer.from_host(np.full(hip.embedding_workspace(count, vocab, dim) // 4, np.nan))
    hip.embedding_backward(dtable, hip.DeviceBuffer.from_host(grad),
                           hip.DeviceBuffer.from_host(ids, np.int32), count, vocab, dim, 2.0, beta, work)
    assert np.array_equal(dtable.to_host((vocab, dim)), (value + beta * old).astype(np.float32))


@pytest.mark.parametrize("count,dim,constant", [(1 << 24, 1, True), (1 << 22, 5, True), (3 << 20, 4, False)])
def test_error_of_a_long_run_is_that_of_a_tile(hip, count, dim, constant):
    """Tiles of at most 256 positions are added one after another: 255 half steps
    of the sum of magnitudes at most, and a few for what comes after, however many
    tiles a token's run has. Equal gradients round all in one direction."""
    rng = np.random.default_rng(dim)
    grad = np.full((count, dim), 1.1, np.float32)
    if not constant:
        grad = rng.uniform(0.5, 1.5, (count, dim)).astype(np.float32)
    ids = np.full(count, 1, np.int32)
    print(f"embedding, {count} positions of one token x {dim}", flush=True)
    dtable = hip.DeviceBuffer(3 * dim)
    hip.embedding_backward(dtable, hip.DeviceBuffer.from_host(grad),
                           hip.DeviceBuffer.from_host(ids, np.int32), count, 3, dim, 1.0)
    got = dtable.to_host((3, dim))
    want = grad.astype(np.float64).sum(axis=0)
    assert np.all(got[[0, 2]] == 0)
    error = np.abs(got[1] - want) / want
    assert np.all(error <= (255 + 8) * U), error.max() / U


@pytest.mark.parametrize("count", [200, 40000])
def test_gradients_that_are_not_finite(hip, count):
    """An infinity stays one, in its own column of its own token; two of different
    sign, or a NaN, give NaN."""
    rng = np.random.default_rng(5)
    dim, vocab = 260, 3
    ids = np.full(count, 2, np.int32)
    ids[::7] = 0
    grad = rng.standard_normal((count, dim)).astype(np.float32)
    grad[count // 2 // 7 * 7 + 1, 3] = np.inf
    grad[[1, count - count % 7 - 3], 8] = np.inf, -np.inf
    grad[count // 3 // 7 * 7 + 2, 259] = np.nan
    print(f"embedding, infinities, {count}", flush=True)
    dtable = hip.DeviceBuffer(vocab * dim)
    hip.embedding_backward(dtable, hip.DeviceBuffer.from_host(grad),
                           hip.DeviceBuffer.from_host(ids, np.int32), count, vocab, dim, 1.0)
    got = dtable.to_host((vocab, dim))
    assert got[2, 3] == np.inf and np.isnan(got[2, [8, 259]]).all()
    got[2, [3, 8, 259]] = 0
    assert np.isfinite(got).all()
