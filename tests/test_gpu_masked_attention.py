"""nrs_masked_attention_forward / _backward against the same algebra in 64 bits
(tests/masked_ref.py, which also derives how far f32 may be off). Keys that no row
sees hold NaN, every output buffer starts as a marker that shows what was written, and
the scratch holds NaN."""
import numpy as np
import pytest

from masked_ref import Problem

pytestmark = pytest.mark.gpu

MARK = np.float32(-12345.0)


class Device:
    """A problem's tensors on the device."""

    def __init__(self, hip, p, work=True):
        self.hip, self.p = hip, p
        up = hip.DeviceBuffer.from_host

        def ints(x):
            return None if x is None else up(x, np.int32)

        self.q, self.dout, self.kbuf = up(p.q), up(p.dout), up(p.k)
        self.vbuf = self.kbuf if p.packed else up(p.v)
        self.k, self.v = self.kbuf.ptr, self.vbuf.ptr + 4 * p.v_at
        self.mask = hip.attention_mask(
            p.causal, ints(p.q_start), ints(p.key_len), ints(p.prefix_len), ints(p.key_begin),
            ints(p.key_end), None if p.slopes is None else up(p.slopes), p.cap)
        self.out = up(np.full((p.batch * p.sq, p.ld_out), MARK))
        self.stats = up(np.full(max(1, p.batch * p.heads * p.sq * 2), MARK))
        self.work = [None, None]
        if work:
            for back in (0, 1):
                n = hip.masked_attention_workspace(*p.shape()[:6], backward=back)
                self.work[back] = up(np.full(max(4, n // 4), np.nan))

    def forward(self, stats=True):
        self.hip.masked_attention_forward(self.out, self.stats if stats else None, self.q, self.k,
                                          self.v, self.mask, *self.p.shape(), self.p.scale,
                                          self.work[0])

    def backward(self, dq, dk, dv, beta_q=0.0, beta_kv=0.0):
        self.hip.masked_attention_backward(dq, dk, dv, self.dout, self.out, self.q, self.k, self.v,
                                           self.stats, self.mask, *self.p.shape(), self.p.scale,
                                           beta_q, beta_kv, self.work[1])


def compare(got, value, bound, what):
    """Within the bound (plus what a float of the value's size rounds)."""
    tol = bound + 2.0 ** -24 * np.abs(value) + 2.0 ** -126
    bad = ~(np.abs(got - value) <= tol)
    assert not bad.any(), (
        f"{what}: {bad.sum()} of {bad.size} off; worst {np.nanmax(np.abs(got - value) / tol):.3g} of "
        f"its bound, first at {np.argwhere(bad)[0]}: {got[tuple(np.argwhere(bad)[0])]} for "
        f"{value[tuple(np.argwhere(bad)[0])]}")


def check(hip, p, beta_q=0.0, beta_kv=0.0, gradients=True, work=True):
    print(f"masked attention {p.shape()} beta {beta_q} {beta_kv}", flush=True)
    ref = p.reference(gradients)
    dev = Device(hip, p, work)
    dev.forward(stats=gradients)
    hd, kd = p.heads * p.d, p.kv * p.d
    out = dev.out.to_host((p.batch * p.sq, p.ld_out))
    compare(out[:, :hd], *ref["out"], "out")
    assert np.all(out[:, hd:] == MARK)
    if not gradients:
        return
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


def documents(seq, firsts):
    """key_begin and key_end of packed documents that begin at `firsts`."""
    firsts = sorted(firsts)
    begin = [max(f for f in firsts if f <= i) for i in range(seq)]
    end = [min([f for f in firsts if f > i] + [seq]) for i in range(seq)]
    return begin, end


CAUSAL = [
    # batch, heads, kv_heads, seq, d_head
    (1, 1, 1, 1, 1), (2, 3, 3, 7, 16), (1, 2, 2, 32, 32), (2, 4, 2, 33, 24), (1, 2, 1, 64, 64),
    (2, 2, 2, 65, 128), (1, 7, 1, 31, 40), (1, 2, 1, 130, 80), (2, 2, 1, 129, 96), (1, 3, 3, 200, 127),
    (1, 4, 4, 300, 64), (1, 4, 1, 259, 128), (3, 8, 8, 128, 32), (1, 2, 2, 515, 3), (1, 8, 2, 40, 32),
]


@pytest.mark.parametrize("shape", CAUSAL, ids=lambda s: "x".join(map(str, s)))
def test_causal(hip, shape):
    b, h, kv, n, d = shape
    check(hip, Problem(b, h, kv, n, n, d, seed=sum(shape)))


MASKS = {
    "padded": dict(key_len=[150, 37]),
    "nothing_live": dict(key_len=[0, -4]),
    "prefix": dict(prefix_len=[60, 149]),
    "prefix_past_the_keys": dict(prefix_len=[1000, 0], key_len=[140, 150]),
    "documents": dict(key_begin=documents(150, [0, 1, 40, 96, 128])[0]),
    "documents_both_ways": dict(causal=False, key_begin=documents(150, [0, 31, 33, 100])[0],
                                key_end=documents(150, [0, 31, 33, 100])[1]),
    "any_ranges": dict(causal=False,
                       key_begin=np.random.default_rng(1).integers(-20, 170, (2, 150)),
                       key_end=np.random.default_rng(2).integers(-20, 170, (2, 150))),
    "empty_ranges": dict(key_begin=np.where(np.arange(150) % 3 == 0, 200, 0)),
    "first_rows_before_the_keys": dict(q_start=[-60, -149]),
    "rows_behind_the_keys": dict(q_start=[10, 1000]),
    "a_key_each": dict(causal=False, key_begin=np.arange(150)[::-1], key_end=np.arange(150)[::-1] + 1),
    "no_mask": dict(causal=False),
}


@pytest.mark.parametrize("extra", [dict(), dict(slopes=True), dict(cap=2.0), dict(cap=30.0, slopes=True)],
                         ids=["plain", "slopes", "cap", "cap_slopes"])
@pytest.mark.parametrize("name", MASKS)
def test_masks(hip, name, extra):
    check(hip, Problem(2, 4, 2, 150, 150, 32, seed=7, **MASKS[name], **extra))


@pytest.mark.parametrize("d", [64, 72, 96, 128])
@pytest.mark.parametrize("name", ["padded", "prefix", "documents", "any_ranges", "empty_ranges"])
def test_masks_of_wider_heads(hip, name, d):
    check(hip, Problem(2, 3, 1, 150, 150, d, seed=8, slopes=d == 64, cap=20.0 if d == 96 else 0.0,
                       **MASKS[name]))


@pytest.mark.parametrize("sq,sk,d,kw", [
    (1, 1, 16, dict()), (1, 300, 64, dict(q_start=[299, 17], key_len=[300, 18])),
    (1, 1000, 128, dict(slopes=True)), (4, 333, 40, dict(cap=5.0, q_start=[100, 329])),
    (3, 50, 32, dict(slopes=True, cap=3.0, key_begin=[[0, 30, 47], [5, 49, 60]])),
    (16, 200, 32, dict(q_start=[0, 184])), (1, 257, 128, dict(key_len=[0, 257])),
    (2, 2000, 64, dict(causal=False, key_begin=[[0, 1990], [7, 8]], key_end=[[3, 2000], [1999, 8]])),
    (7, 100, 96, dict(prefix_len=[100, 3], q_start=[0, 50])),
], ids=str)
@pytest.mark.parametrize("group", [1, 4])
def test_tokens(hip, sq, sk, d, kw, group):
    """Few rows over a cache, without and with what a backward needs."""
    p = Problem(2, 2 * group, 2, sq, sk, d, seed=sq + sk, **kw)
    check(hip, p, gradients=False)
    check(hip, p)


@pytest.mark.parametrize("sq,sk", [(50, 200), (200, 50), (33, 1000), (300, 5), (1, 5)])
def test_prompts(hip, sq, sk):
    """Queries that continue a cache, or that stand before their keys."""
    check(hip, Problem(2, 4, 2, sq, sk, 64, seed=sq, slopes=True))


@pytest.mark.parametrize("beta_q,beta_kv", [(1.0, 1.0), (0.0, 1.0), (0.5, -2.0)])
@pytest.mark.parametrize("d", [32, 64])
def test_accumulates(hip, d, beta_q, beta_kv):
    check(hip, Problem(2, 2, 1, 90, 90, d, key_len=[90, 40], seed=4), beta_q, beta_kv)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d", [32, 37, 128])
def test_strides(hip, packed, d):
    check(hip, Problem(2, 2, 2, 70, 70, d, pad_q=5, pad_kv=3, packed=packed, seed=9, slopes=True))


def test_library_scratch(hip):
    check(hip, Problem(1, 2, 1, 300, 300, 64, seed=2), work=False)
    check(hip, Problem(2, 2, 1, 1, 3000, 64, seed=2), work=False)


@pytest.mark.parametrize("missing", ["dq", "dkv"])
@pytest.mark.parametrize("d", [32, 64])
def test_one_gradient_has_the_bits_of_both(hip, missing, d):
    p = Problem(2, 4, 2, 140, 140, d, seed=11, cap=4.0)
    dev = Device(hip, p)
    dev.forward()
    zeros = hip.DeviceBuffer.zeros
    sizes = [p.q.size, p.k.size, p.v.size]
    both = [zeros(n) for n in sizes]
    dev.backward(*both)
    one = [zeros(n) for n in sizes]
    dev.backward(*([None] + one[1:] if missing == "dq" else [one[0], None, None]))
    for i in ((1, 2) if missing == "dq" else (0,)):
        assert np.array_equal(both[i].to_host(), one[i].to_host())


def test_the_same_call_has_the_same_bits(hip):
    p = Problem(2, 4, 1, 200, 200, 64, seed=12, slopes=True)
    seen = []
    for _ in range(3):
        dev = Device(hip, p)
        dev.forward()
        grads = [hip.DeviceBuffer.zeros(n) for n in (p.q.size, p.k.size, p.v.size)]
        dev.backward(*grads)
        seen.append([x.to_host() for x in [dev.out, dev.stats] + grads])
    for other in seen[1:]:
        for x, y in zip(seen[0], other):
            assert np.array_equal(x, y)


def run(hip, p):
    """out, dq, dk, dv as the library gives them."""
    dev = Device(hip, p)
    dev.forward()
    grads = [hip.DeviceBuffer.zeros(n) for n in (p.q.size, p.k.size, p.v.size)]
    dev.backward(*grads)
    return [x.to_host(s) for x, s in zip([dev.out] + grads, [(-1, p.ld_out), p.q.shape, p.k.shape, p.v.shape])]


BAD = [np.nan, np.inf, -np.inf]


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("sq,sk,d", [(150, 150, 32), (150, 150, 128), (6, 90, 64)])
def test_a_bad_key_stays_with_the_rows_that_see_it(hip, sq, sk, d, which, bad):
    """Key `at` of item 0 goes bad in one column. Rows that see it lose
    their results; the others keep their bits, and so do the gradients that only they
    have a part in."""
    p = Problem(2, 2, 1, sq, sk, d, seed=13)
    at = sk - sq // 2 - 1
    clean = run(hip, p)
    getattr(p, which)[at, d // 3] = bad
    out, dq, dk, dv = run(hip, p)
    sees = p.visible(0)[:, at]
    assert sees.any() and not sees.all()
    hidden = np.concatenate([~sees, np.ones(sq, bool)])
    for got, was in ((out, clean[0]), (dq, clean[1])):
        assert np.array_equal(got[hidden], was[hidden])
    if which == "v" or np.isnan(bad):  # a score of minus infinity is no weight
        assert not np.isfinite(out[:sq][sees]).all(axis=1).any()
    # keys that no row with a bad result sees keep their gradients
    touched = np.concatenate([p.visible(0)[sees].any(axis=0), np.zeros(sk, bool)])
    for got, was in ((dk, clean[2]), (dv, clean[3])):
        assert np.array_equal(got[~touched], was[~touched])


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("which", ["q", "dout"])
@pytest.mark.parametrize("d", [32, 128])
def test_a_bad_row_stays_with_the_keys_that_it_sees(hip, d, which, bad):
    p = Problem(2, 2, 2, 150, 150, d, causal=False, seed=14,
                key_begin=documents(150, [0, 70])[0], key_end=documents(150, [0, 70])[1])
    clean = run(hip, p)
    getattr(p, which)[80, d // 2] = bad  # head 0 of a row of the second document
    got = run(hip, p)
    other = np.ones((300, 2 * d), bool)
    other[80, :d] = False
    for i in (0, 1):
        assert np.array_equal(got[i][other], clean[i][other])
    other = np.ones((300, 2 * d), bool)
    other[70:150, :d] = False
    for i in (2, 3):
        assert np.array_equal(got[i][other], clean[i][other])
    assert not np.isfinite(got[2][70:150, :d]).all(axis=1).any()


def test_masked_scores_of_the_lowest_value(hip):
    """Rows whose visible scores are all far below those of hidden keys."""
    p = Problem(1, 1, 1, 64, 64, 32, causal=False, key_begin=np.full((1, 64), 40), seed=15)
    p.q[:] = 3.0
    p.k[:40] = 1e30   # hidden from all
    p.k[40:] = -1e3 * np.arange(1, 25, dtype=np.float32)[:, None]
    check(hip, p)


def test_far_rows_keep_their_scores(hip):
    """A token far past its keys: the bias is taken relative to the nearest."""
    p = Problem(1, 2, 1, 3, 40, 16, q_start=[10 ** 6], slopes=True, seed=16)
    check(hip, p)


def test_positions_at_the_ends_of_int32(hip):
    p = Problem(2, 2, 1, 5, 20, 16, q_start=[2 ** 31 - 1, -2 ** 31], key_len=[2 ** 31 - 1, 20], seed=17)
    check(hip, p)


def test_nothing_to_do(hip):
    dev = Device(hip, Problem(1, 1, 1, 4, 1, 8, key_len=[0], seed=1))
    dev.forward()
    assert np.all(dev.out.to_host() == 0) and np.all(dev.stats.to_host() == 0)
    mark = hip.DeviceBuffer.from_host(np.full(32, MARK))
    hip.masked_attention_forward(mark, None, mark, None, None, None, 2, 1, 1, 2, 0, 8, 8, 8, 8, 1.0)
    assert np.all(mark.to_host() == 0)


@pytest.mark.parametrize("shape", [(2, 4, 2, 100, 0, 32), (2, 4, 2, 0, 100, 32), (2, 4, 2, 0, 100, 128),
                                   (1, 2, 1, 0, 0, 64)], ids=str)
def test_no_rows_or_no_keys(hip, shape):
    check(hip, Problem(*shape, seed=18), beta_kv=0.5)
    check(hip, Problem(*shape, seed=18), beta_q=1.0, beta_kv=1.0)


def test_many_items_of_a_token(hip):
    """More items than share one line of tiles."""
    check(hip, Problem(1500, 2, 1, 1, 60, 16, q_start=np.arange(1500) % 60, seed=19), gradients=False)


def test_many_short_items(hip):
    check(hip, Problem(300, 2, 2, 7, 7, 8, key_len=np.arange(300) % 8, seed=20))


@pytest.mark.parametrize("d", [32, 64, 128])
def test_long_walks_in_parts(hip, d):
    """Few units over long ranges: forward and backward walks in several parts, of which
    some rows (and keys) have one."""
    p = Problem(1, 1, 1, 2100, 2100, d, seed=21, key_begin=np.where(np.arange(2100) % 700 < 650, 0, 1900))
    check(hip, p)
    check(hip, Problem(1, 2, 1, 600, 4000, d, seed=22, slopes=True, prefix_len=[3800]))


@pytest.mark.parametrize("magnitude", [1e-12, 1e-3, 30.0])
def test_magnitudes(hip, magnitude):
    check(hip, Problem(1, 2, 2, 60, 60, 32, seed=23, magnitude=magnitude, cap=5.0))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(hip, scale):
    p = Problem(1, 2, 2, 60, 60, 32, seed=24, slopes=True)
    p.scale = np.float32(scale)
    check(hip, p)
    p = Problem(1, 2, 2, 3, 60, 32, seed=24, cap=1.0)
    p.scale = np.float32(scale)
    check(hip, p, gradients=False)


def test_a_group_of_many_heads(hip):
    check(hip, Problem(1, 112, 1, 9, 40, 24, seed=25, cap=3.0))
    check(hip, Problem(2, 33, 1, 1, 200, 24, seed=26, slopes=True))


@pytest.mark.parametrize("extra", [dict(), dict(cap=2.0), dict(cap=2.0, slopes=True), dict(slopes=True)],
                         ids=str)
@pytest.mark.parametrize("sq,d", [(150, 32), (150, 96), (150, 128), (600, 64), (9, 64)])
def test_hidden_magnitudes(hip, sq, d, extra):
    """Finite values whose products overflow, in a document of their own: the other
    document's results and gradients keep their bits."""
    sk, firsts = 150 if sq < 150 else sq, [0, sq // 2]
    begin, end = (np.array(x) for x in documents(sq, firsts))
    cut = sk - sq + firsts[1]  # the second document's first key
    p = Problem(1, 2, 1, sq, sk, d, causal=False, seed=27, key_begin=np.where(begin > 0, cut, 0),
                key_end=np.where(begin > 0, sk, cut), **extra)
    clean = run(hip, p)
    rng = np.random.default_rng(5)
    for x, at in ((p.q, firsts[1]), (p.dout, firsts[1]), (p.k, cut), (p.v, cut)):
        x[at:] = rng.choice([-1.6e38, 1.6e38], x[at:].shape)
    got = run(hip, p)
    for i, at in ((0, firsts[1]), (1, firsts[1]), (2, cut), (3, cut)):
        assert np.array_equal(got[i][:at], clean[i][:at]), ["out", "dq", "dk", "dv"][i]


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("d", [32, 128])
def test_a_row_that_sees_nothing_has_no_gradient(hip, d, bad):
    """Whatever its own numbers are."""
    p = Problem(1, 2, 2, 150, 150, d, key_begin=np.where(np.arange(150) % 3 == 0, 200, 0), seed=28)
    clean = run(hip, p)
    p.q[::3] = p.dout[::3] = bad
    got = run(hip, p)
    for x, was in zip(got, clean):
        assert np.array_equal(x, was)
    assert np.all(got[0][::3] == 0) and np.all(got[1][::3] == 0)
