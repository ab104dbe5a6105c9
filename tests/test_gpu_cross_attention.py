"""nrs_cross_attention_forward / _backward against the same algebra in 64
bits (tests/attention_ref.py, which also derives how far f32 may be off).
Every problem's dead keys hold NaN, every output buffer starts as a marker
that shows what was written."""
import numpy as np
import pytest

from attention_ref import Problem, backward, forward

pytestmark = pytest.mark.gpu

MARK = np.float32(-12345.0)


class Device:
    """A problem's tensors on the device."""

    def __init__(self, hip, p):
        self.hip, self.p = hip, p
        up = hip.DeviceBuffer.from_host
        self.q, self.dout, self.kbuf = up(p.q), up(p.dout), up(p.k)
        self.vbuf = self.kbuf if p.packed else up(p.v)
        self.k, self.v = self.kbuf.ptr, self.vbuf.ptr + 4 * p.v_at
        self.lens = None if p.lens is None else up(p.lens, np.int32)
        self.out = up(np.full((p.batch * p.sq, p.ld_out), MARK))
        self.stats = up(np.full(max(1, p.batch * p.heads * p.sq * 2), MARK))

    def forward(self, stats=True, work=None):
        self.hip.cross_attention_forward(self.out, self.stats if stats else None, self.q, self.k,
                                         self.v, self.lens, *self.p.shape(), self.p.scale, work)

    def backward(self, dq, dk, dv, beta_q=0.0, beta_kv=0.0, work=None):
        self.hip.cross_attention_backward(dq, dk, dv, self.dout, self.out, self.q, self.k, self.v,
                                          self.stats, self.lens, *self.p.shape(), self.p.scale,
                                          beta_q, beta_kv, work)


def compare(got, value, bound, what):
    """Within the bound (plus what a float of the value's size rounds)."""
    tol = bound + 2.0 ** -24 * np.abs(value) + 2.0 ** -126
    bad = ~(np.abs(got - value) <= tol)
    assert not bad.any(), (
        f"{what}: {bad.sum()} of {bad.size} off; worst {np.nanmax(np.abs(got - value) / tol):.3g} of "
        f"its bound, first at {np.argwhere(bad)[0]}: {got[tuple(np.argwhere(bad)[0])]} for "
        f"{value[tuple(np.argwhere(bad)[0])]}")


def check(hip, p, beta_q=0.0, beta_kv=0.0):
    print(f"cross attention {p.shape()} lens {p.lens} beta {beta_q} {beta_kv}", flush=True)
    ref = p.reference()
    dev = Device(hip, p)
    dev.forward()
    hd, kd = p.heads * p.d, p.kv * p.d
    out = dev.out.to_host((p.batch * p.sq, p.ld_out))
    compare(out[:, :hd], *ref["out"], "out")
    assert np.all(out[:, hd:] == MARK)
    stats = dev.stats.to_host()[:p.batch * p.heads * p.sq * 2].reshape(p.batch, p.heads, p.sq, 2)
    for b, n in enumerate(p.live()):
        if n == 0:
            assert np.all(stats[b] == 0)
        else:  # 2^max * sum is what does not depend on the order of the keys
            lse = stats[b, ..., 0] + np.log2(stats[b, ..., 1].astype(np.float64))
            value, bound = ref["stats"]
            compare(lse, value[b, ..., 0] + np.log2(value[b, ..., 1]), bound[b], "log of the sum")
    rng = np.random.default_rng(99)
    old_q = rng.standard_normal((p.batch * p.sq, p.ld_q)).astype(np.float32)
    old_k = [rng.standard_normal((p.batch * p.sk, p.ld_kv)).astype(np.float32) for _ in range(2)]
    start_q, start_k = old_q.copy(), [x.copy() for x in old_k]
    if beta_q == 0.0:
        start_q[:, :hd] = np.nan  # never read
    if beta_kv == 0.0:
        for x in start_k:
            x[:, :kd] = np.nan
    dq, dk, dv = (hip.DeviceBuffer.from_host(x) for x in [start_q] + start_k)
    dev.backward(dq, dk, dv, beta_q, beta_kv)
    for buf, name, old, beta, n in ((dq, "dq", old_q, beta_q, hd), (dk, "dk", old_k[0], beta_kv, kd),
                                    (dv, "dv", old_k[1], beta_kv, kd)):
        got = buf.to_host(old.shape)
        value, bound = ref[name]
        was = beta * old[:, :n].astype(np.float64)
        compare(got[:, :n], value + was, bound + 2.0 ** -23 * (np.abs(value) + np.abs(was)), name)
        assert np.array_equal(got[:, n:], old[:, n:])


SHAPES = [
    # batch, heads, kv_heads, seq_q, seq_k, d_head, lens
    (1, 1, 1, 1, 1, 1, None),
    (2, 3, 3, 5, 7, 16, None),
    (1, 1, 1, 16, 16, 32, None),
    (2, 4, 2, 17, 33, 32, [33, 1]),
    (3, 2, 1, 31, 64, 64, [0, 64, 63]),
    (2, 2, 2, 64, 65, 128, [65, 17]),
    (1, 7, 1, 9, 100, 24, [99]),
    (2, 6, 3, 33, 129, 40, [-5, 1000]),
    (1, 2, 1, 70, 257, 80, None),
    (2, 4, 2, 90, 300, 72, [300, 201]),
    (2, 2, 1, 13, 96, 96, [96, 95]),
    (1, 3, 3, 20, 40, 127, None),
    (1, 2, 2, 10, 50, 3, [49]),
    (4, 8, 8, 128, 200, 32, [200, 150, 0, 31]),
    (1, 4, 4, 300, 515, 64, None),
    (2, 4, 1, 150, 700, 128, [700, 333]),
    (1, 1, 1, 600, 20, 64, None),
    (2, 2, 2, 259, 130, 16, [130, 128]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_shapes(hip, shape):
    check(hip, Problem(*shape[:6], lens=shape[6], seed=sum(shape[:6])))


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[3] <= 70],
                         ids=lambda s: "x".join(map(str, s[:6])))
def test_strides_and_accumulation(hip, shape):
    """Rows with padding, keys and values as halves of one tensor, gradients
    added to what is there."""
    pad = 1 if shape[5] % 2 else 5
    check(hip, Problem(*shape[:6], lens=shape[6], pad_q=pad, pad_kv=3, packed=True, seed=7),
          1.0, 0.5)


@pytest.mark.parametrize("batch,heads,kv,seq_k,d,lens", [
    (1, 1, 1, 1, 64, None), (3, 8, 8, 150, 64, [150, 1, 77]), (2, 8, 2, 1000, 128, [1000, 0]),
    (1, 12, 4, 4097, 32, None), (1, 2, 1, 16384, 16, [16300]), (5, 7, 1, 511, 40, [511, 3, 0, 64, 65]),
    (64, 4, 4, 300, 64, list(range(0, 64 * 5, 5))),
])
def test_single_tokens(hip, batch, heads, kv, seq_k, d, lens):
    check(hip, Problem(batch, heads, kv, 1, seq_k, d, lens=lens, seed=seq_k))


@pytest.mark.parametrize("seq_q,seq_k", [(2, 5000), (40, 9), (3000, 5), (1, 3000)])
def test_lopsided_lengths(hip, seq_q, seq_k):
    check(hip, Problem(1, 2, 1, seq_q, seq_k, 64, seed=seq_q))


@pytest.mark.parametrize("d,heads", [(20, 86), (64, 43), (80, 29), (128, 22)])
def test_much_work(hip, d, heads):
    """Enough for every compute unit to take 256 rows at a time."""
    check(hip, Problem(2, heads, heads, 130, 1500, d, lens=[1500, 1211], seed=d))


@pytest.mark.parametrize("batch,heads,kv,seq_q,seq_k,d,lens", [
    (2, 12, 4, 700, 6, 40, [6, 2]), (3, 4, 2, 2100, 32, 98, [17, 0, 32]),
    (2, 6, 2, 5, 3000, 98, [3000, 1501]), (1, 32, 1, 1, 2047, 128, None),
    (40, 8, 8, 3, 140, 16, list(range(0, 160, 4))), (2, 3, 1, 10, 31, 17, [31, 16]),
    (1, 2, 2, 4000, 1, 80, None), (2, 4, 1, 13, 1500, 128, [1490, 0]), (2, 1, 1, 500, 48, 128, [33, 48]),
    (1, 2, 2, 48, 3000, 32, None), (3, 4, 2, 130, 16, 100, [16, 1, 0]), (2, 4, 4, 37, 17, 33, [17, 4]), (3, 2, 1, 2500, 47, 16, [0, 47, 5]), (2, 1, 1, 49, 90, 8, [90, 6]), (2, 1, 1, 90, 49, 8, [49, 6]),
])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_short_sides(hip, batch, heads, kv, seq_q, seq_k, d, lens, beta):
    """Up to 48 rows or keys of an item (and just above), the other side short and
    long."""
    check(hip, Problem(batch, heads, kv, seq_q, seq_k, d, lens=lens, pad_q=2, seed=d), beta, beta)


def test_large_scores(hip):
    """Scores in the hundreds: only the differences to the maximum count."""
    check(hip, Problem(1, 2, 2, 40, 90, 32, seed=3, magnitude=8.0))


@pytest.mark.parametrize("seq_q", [1, 200])
@pytest.mark.parametrize("step", [0.05, 2.0, -2.0])
def test_scores_that_climb(hip, seq_q, step):
    """Every key's score is above (or below) the one before: the running
    maximum moves at each tile, or never after the first, to scores in the
    thousands, whose powers of two no float holds."""
    p = Problem(1, 2, 1, seq_q, 1000, 64, seed=11)
    p.q[:] = np.abs(p.q) + np.float32(0.5)
    p.k[:] = np.abs(p.k) * np.float32(0.01) + (np.arange(1000) * step / 30).astype(np.float32)[:, None]
    check(hip, p)


def test_zero_lengths(hip):
    for sq, sk in ((0, 5), (4, 0), (0, 0)):
        check(hip, Problem(2, 2, 2, sq, sk, 16))
    check(hip, Problem(0, 2, 2, 4, 4, 16))
    # the last case has keys and no rows: their gradients are zeros (or as they were)
    p = Problem(2, 2, 2, 0, 5, 16)
    dev = Device(hip, p)
    old = np.arange(10 * 32, dtype=np.float32).reshape(10, 32)
    for beta, want in ((0.0, np.zeros_like(old)), (1.0, old)):
        dk, dv = hip.DeviceBuffer.from_host(old), hip.DeviceBuffer.from_host(old)
        dev.backward(None, dk, dv, beta_kv=beta)
        assert np.array_equal(dk.to_host(old.shape), want)
        assert np.array_equal(dv.to_host(old.shape), want)


def test_parts_and_optional_outputs_have_the_same_bits(hip):
    p = Problem(2, 4, 2, 50, 140, 64, lens=[140, 81], seed=5)
    dev = Device(hip, p)
    dev.forward(stats=False)
    alone = dev.out.to_host()
    assert np.all(dev.stats.to_host() == MARK)
    dev.forward()
    assert np.array_equal(dev.out.to_host(), alone)
    shapes = [p.q.shape, p.k.shape, p.v.shape]
    full = [hip.DeviceBuffer.from_host(np.full(s, MARK)) for s in shapes]
    dev.backward(*full)
    for _ in range(2):
        q = hip.DeviceBuffer.from_host(np.full(shapes[0], MARK))
        dev.backward(q, None, None)
        assert np.array_equal(q.to_host(), full[0].to_host())
        k, v = (hip.DeviceBuffer.from_host(np.full(s, MARK)) for s in shapes[1:])
        dev.backward(None, k, v)
        assert np.array_equal(k.to_host(), full[1].to_host())
        assert np.array_equal(v.to_host(), full[2].to_host())


@pytest.mark.parametrize("shape,lens", [((2, 4, 2, 11, 2500, 64), [2500, 700]),
                                        ((2, 4, 2, 900, 40, 64), [40, 17]),
                                        ((1, 2, 2, 1, 130, 128), None), ((2, 2, 1, 60, 5, 16), [5, 0])])
def test_gradients_of_short_sides_alone_have_the_same_bits(hip, shape, lens):
    p = Problem(*shape, lens=lens, seed=12)
    dev = Device(hip, p)
    dev.forward()
    shapes = [p.q.shape, p.k.shape, p.v.shape]
    full, q, k, v = ([hip.DeviceBuffer.from_host(np.full(s, MARK)) for s in shapes]
                     for _ in range(4))
    dev.backward(*full)
    dev.backward(q[0], None, None)
    dev.backward(None, k[1], v[2])
    for i, got in enumerate((q[0], k[1], v[2])):
        assert np.array_equal(got.to_host(), full[i].to_host())


def test_an_item_does_not_depend_on_its_batch(hip):
    """NaN in one item's live keys stays in that item."""
    p = Problem(3, 2, 2, 40, 70, 32, lens=[70, 60, 50], seed=6)
    dev = Device(hip, p)
    dev.forward()
    want = dev.out.to_host((3, 40, p.ld_out))
    p.k[70 + 5, 3] = np.nan
    p.v[70 + 9, 40] = np.inf
    dev = Device(hip, p)
    dev.forward()
    got = dev.out.to_host((3, 40, p.ld_out))
    assert np.array_equal(got[[0, 2]], want[[0, 2]])
    assert np.isnan(got[1, :, :32]).all()


def test_gradients_against_differences(hip):
    """Along random directions of q, k and v: the difference quotient of the
    kernel's own outputs, off by its outputs' bounds over the step and by the
    quotient's own error, which 64 bits give."""
    p = Problem(1, 4, 2, 20, 45, 32, lens=[45], seed=8)
    dev = Device(hip, p)
    dev.forward()
    grads = [hip.DeviceBuffer(x.size) for x in (p.q, p.k, p.v)]
    dev.backward(*grads)
    rng = np.random.default_rng(4)
    h = 2.0 ** -6
    ref = p.reference()
    for name, buf in zip(("q", "k", "v"), grads):
        x = getattr(p, name)
        step = (rng.integers(0, 2, x.shape) * 2 - 1).astype(np.float32)
        loss, loss64, slack = [], [], 0.0
        for sign in (1, -1):
            q = Problem(1, 4, 2, 20, 45, 32, lens=[45], seed=8)
            setattr(q, name, (x + np.float32(sign * h) * step).astype(np.float32))
            d = Device(hip, q)
            d.forward()
            value, bound = q.reference(False)["out"]
            w = p.dout.astype(np.float64)
            loss.append((d.out.to_host(value.shape) * w).sum())
            loss64.append((value * w).sum())
            slack += (np.abs(w) * (bound + 2.0 ** -24 * np.abs(value))).sum() / (2 * h)
        # the perturbed inputs round: half a step of |x| + h each
        slack += (np.abs(ref["d" + name][0]) * 2.0 ** -24 * (np.abs(x) + h)).sum() / h
        quotient, quotient64 = (loss[0] - loss[1]) / (2 * h), (loss64[0] - loss64[1]) / (2 * h)
        exact = (ref["d" + name][0] * step).sum()
        got = (buf.to_host(x.shape).astype(np.float64) * step).sum()
        slack += abs(quotient64 - exact) + (ref["d" + name][1]).sum()
        print(name, quotient, got, slack, flush=True)
        assert abs(quotient - got) <= slack


def test_own_scratch_gives_the_same_bits(hip):
    for shape in ((1, 2, 1, 1, 5000, 64), (2, 2, 2, 200, 600, 128), (1, 1, 1, 1000, 40, 32)):
        p = Problem(*shape, seed=9)
        dev = Device(hip, p)
        dev.forward()
        want = dev.out.to_host()
        need = hip.cross_attention_workspace(*shape)
        work = hip.DeviceBuffer(max(4, (need + 3) // 4 + 64))
        fill = np.full(work.n, MARK)
        work = hip.DeviceBuffer.from_host(fill)
        dev.forward(work=work)
        assert np.array_equal(dev.out.to_host(), want)
        assert np.array_equal(work.to_host()[(need + 3) // 4:], fill[(need + 3) // 4:])
        grads = [[hip.DeviceBuffer(x.size) for x in (p.q, p.k, p.v)] for _ in range(2)]
        dev.backward(*grads[0])
        need = hip.cross_attention_workspace(*shape, backward=True)
        fill = np.full((need + 3) // 4 + 64, MARK)
        work = hip.DeviceBuffer.from_host(fill)
        dev.backward(*grads[1], work=work)
        for a, b in zip(*grads):
            assert np.array_equal(a.to_host(), b.to_host())
        assert np.array_equal(work.to_host()[(need + 3) // 4:], fill[(need + 3) // 4:])
