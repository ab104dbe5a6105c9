"""Cross attention on every kernel that its planner can choose (cross_plan.py lists the
calls, test_cross_plan.py holds them to their kernels), against the algebra of
attention_ref.py in 64 bits on the device, with its bounds."""
import math

import pytest
import torch

import cross_plan
from attention_ref import TINY, U, gamma

pytestmark = pytest.mark.gpu

MARK = -12345.0


def mm(a, b):
    return torch.mm(a.contiguous(), b.contiguous())


def reference(q, k, v, g, scale, lost=0.0):
    """(value, bound) of out, the log2 of the rows' sums, dq, dk and dv: as
    attention_ref.forward and backward, one item and key head. Every operand of a
    product, and every term of a sum, may be off by `lost` besides."""
    n, d, rows = len(k), q.shape[1], len(q)
    if n == 0:
        zero = [torch.zeros_like(x) for x in (q, q, k, v)]
        none = torch.zeros(rows, dtype=torch.float64, device=q.device)
        return [(x, x) for x in [zero[0], none] + zero[1:]]
    s = mm(q, k.t()) * scale
    m = s.amax(dim=1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(dim=1, keepdim=True)
    p = p / total
    size = lambda x: x.abs().sum(dim=1, keepdim=True)
    es = (gamma(d) + 4 * U) * (mm(q.abs(), k.abs().t()) * abs(scale)).amax(dim=1, keepdim=True)
    es = es + lost * abs(scale) * (size(q) + size(k).max() + d)
    ep = 2 * es + gamma(n) + 8 * U
    out = mm(p, v)
    out_bound = (ep + gamma(n)) * mm(p, v.abs()) + (TINY + lost) * v.abs().sum(dim=0) + lost * (n + 1)
    lse = m / math.log(2.0) + torch.log2(total)
    lse_bound = 1.45 * ep + 4 * U * m.abs() / math.log(2.0)
    dp = mm(g, v.t())
    delta = (g * out).sum(dim=1, keepdim=True)
    ds = p * (dp - delta) * scale
    e_delta = (gamma(d) * g.abs() * out.abs() + g.abs() * out_bound).sum(dim=1, keepdim=True)
    e_dp = gamma(d) * mm(g.abs(), v.abs().t()) + lost * (size(g) + size(v).t() + d)
    e_ds = abs(scale) * p * ((ep + 4 * U) * (dp - delta).abs() + e_dp + e_delta)
    e_ds = e_ds + (TINY + lost) * (1 + abs(scale)) * (1 + (dp - delta).abs())
    e_p = ep * p + TINY + lost
    return [(out, out_bound), (lse[:, 0], lse_bound[:, 0]),
            (mm(ds, k), mm(e_ds + gamma(n) * ds.abs(), k.abs()) + lost * (size(ds) + n)),
            (mm(ds.t(), q), mm((e_ds + gamma(rows) * ds.abs()).t(), q.abs()) + lost * (size(ds.t()) + rows)),
            (mm(p.t(), g), mm((e_p + gamma(rows) * p).t(), g.abs()) + lost * (size(p.t()) + rows))]


def within(got, value, bound, what):
    tol = bound + 2.0 ** -24 * value.abs() + 2.0 ** -126
    error = (got.double() - value).abs()
    assert (error <= tol).all(), f"{what}: worst {(error / tol).nan_to_num(math.inf).max().item():.3g} of its bound"


def check(hip, shape, number, lens=None, scale=None, ld=None):
    """One call and its backward. Every second has padded rows and K and V in one
    tensor; where there are several items their lengths differ and one is empty,
    unless given. The gradients are written, added to the old ones, or added to half
    of them. The scratch holds NaN: nothing is read that the call did not write."""
    batch, heads, kv, seq_q, seq_k, d = shape
    print(f"cross attention {shape}", flush=True)
    packed, beta = number % 2 == 1, (0.0, 1.0, 0.5)[number % 3]
    gen = torch.Generator(device="cuda").manual_seed(number)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    hd, kd, group = heads * d, kv * d, heads // kv
    ld_q, ld_out, ld_kv = hd + 3 * packed, hd + 5 * packed, kd * (1 + packed) + packed
    if ld:
        ld_q = ld_out = ld_kv = ld
    given = lens is not None
    if not given:
        lens = [max(1, seq_k - i * seq_k // (2 * batch)) for i in range(batch)]
        if batch > 1:
            lens[batch // 2] = 0
    key_len = torch.tensor(lens, dtype=torch.int32, device="cuda") if given or batch > 1 else None
    q, dout, old_q = new(batch * seq_q, ld_q), new(batch * seq_q, ld_out), new(batch * seq_q, ld_q)
    kb, old_k = new(batch * seq_k, ld_kv), new(batch * seq_k, ld_kv)
    vb, old_v = (kb, old_k) if packed else (new(batch * seq_k, ld_kv), new(batch * seq_k, ld_kv))
    for b, n in enumerate(lens):  # never looked at
        kb[b * seq_k + n:(b + 1) * seq_k] = math.nan
        vb[b * seq_k + n:(b + 1) * seq_k] = math.nan
    at = kd if packed else 0
    k, v = kb[:, :kd], vb[:, at:at + kd]
    dq, dkb = old_q.clone(), old_k.clone()
    dvb = dkb if packed else old_v.clone()
    dk, dv = dkb[:, :kd], dvb[:, at:at + kd]
    if beta == 0.0:  # the old gradients are never read
        dq[:, :hd] = math.nan
        dk.fill_(math.nan)
        dv.fill_(math.nan)
    out = torch.full((batch * seq_q, ld_out), MARK, device="cuda")
    stats = torch.full((batch, heads, seq_q, 2), MARK, device="cuda")
    scale = torch.tensor(1 / math.sqrt(d) if scale is None else scale).item()
    args = (*shape, ld_q, ld_kv, ld_out, scale)
    work = [torch.full((hip.cross_attention_workspace(*shape, backward=b) // 4 + 1,), math.nan, device="cuda")
            for b in (False, True)]
    hip.cross_attention_forward(out, stats, q, k, v, key_len, *args, work[0])
    hip.cross_attention_backward(dq, dk, dv, dout, out, q, k, v, stats, key_len, *args, beta, beta, work[1])
    torch.cuda.synchronize()
    assert (out[:, hd:] == MARK).all()
    assert torch.equal(dq[:, hd:], old_q[:, hd:]) and torch.equal(dkb[:, at + kd:], old_k[:, at + kd:])
    for b, n in enumerate(lens):
        rows, keys = slice(b * seq_q, (b + 1) * seq_q), slice(b * seq_k, (b + 1) * seq_k)
        for j in range(kv):
            qc, kc = slice(j * group * d, (j + 1) * group * d), slice(j * d, (j + 1) * d)
            as_rows = lambda x: x[rows, qc].double().reshape(seq_q * group, d)
            live = lambda x: x[keys, kc][:n].double()
            ref = reference(as_rows(q), live(k), live(v), as_rows(dout), scale)
            what = f"item {b}, key head {j}: "
            within(as_rows(out), *ref[0], what + "out")
            st = stats[b, j * group:(j + 1) * group].double().transpose(0, 1).reshape(-1, 2)
            if n:
                within(st[:, 0] + torch.log2(st[:, 1]), *ref[1], what + "log of the sum")
            else:
                assert (st == 0).all()
            was = beta * as_rows(old_q)
            within(as_rows(dq), ref[2][0] + was, ref[2][1] + 2 * U * (ref[2][0].abs() + was.abs()), what + "dq")
            for got, old, (value, bound), name in ((dk, old_k[:, :kd], ref[3], "dk"),
                                                   (dv, old_v[:, at:at + kd], ref[4], "dv")):
                was = beta * live(old)
                within(live(got), value + was, bound + 2 * U * (value.abs() + was.abs()), what + name)
                dead = beta * old[keys, kc][n:]  # (exact: a half of a float, or all of it)
                assert torch.equal(got[keys, kc][n:], dead), what + name + " of dead keys"


@pytest.mark.parametrize("number", range(len(cross_plan.SHAPES)),
                         ids=lambda i: "x".join(map(str, cross_plan.SHAPES[i])))
def test_every_kernel(hip, number):
    check(hip, cross_plan.SHAPES[number], number)


# More items than a workgroup has threads, which look for its part of the line of
# key tiles, up to the 1024 of a shared launch and past them; empty items about the
# parts' ends, or nothing but empty ones.
@pytest.mark.parametrize("shape,live", [
    ((300, 2, 1, 1, 200, 32), lambda i: 200 - i % 150), ((1000, 1, 1, 1, 250, 16), lambda i: 250 if i % 3 else 0),
    ((1024, 1, 1, 3, 130, 24), lambda i: 130 if i in (0, 511, 1023) else 0),
    ((1025, 1, 1, 1, 60, 40), lambda i: i % 61), ((700, 1, 1, 2, 100, 64), lambda i: 100 if i == 699 else 0),
    ((520, 1, 1, 60, 3000, 32), lambda i: 3000 - i % 7 * 429),
    ((513, 1, 1, 250, 2000, 24), lambda i: 2000 if i % 5 else 0), ((600, 1, 1, 33, 300, 16), lambda i: 300 * (i % 2)),
    ((4, 8, 8, 1, 3000, 64), lambda i: 0), ((2, 8, 8, 700, 900, 64), lambda i: 0),
    ((3, 8, 2, 500, 700, 128), lambda i: 700 if i == 1 else 0)],
    ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else "")
def test_many_items_and_empty_ones(hip, shape, live):
    check(hip, shape, 2, lens=[live(i) for i in range(shape[0])])


@pytest.mark.parametrize("shape", [(3, 4, 2, 9, 700, 64), (3, 4, 2, 90, 300, 40), (3, 4, 2, 300, 400, 128),
                                   (3, 4, 2, 100, 9, 24), (2, 2, 2, 130, 40, 16), (2, 4, 2, 1, 90, 100)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_is_not_finite_stays_where_it_is(hip, shape, where, value):
    """A query row's NaN or infinity changes its own row and what its key head
    gathers, a key's all of its item's key head; nothing else changes a bit."""
    batch, heads, kv, seq_q, seq_k, d = shape
    print(f"cross attention {shape}, {value} in {where}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(3)
    hd, kd, group = heads * d, kv * d, heads // kv
    t = {n: torch.randn(*size, generator=gen, device="cuda")
         for n, size in (("q", (batch, seq_q, hd)), ("k", (batch, seq_k, kd)), ("v", (batch, seq_k, kd)),
                         ("dout", (batch, seq_q, hd)))}
    lens = torch.tensor([seq_k, seq_k - seq_k // 3, seq_k][:batch], dtype=torch.int32, device="cuda")
    args = (*shape, hd, kd, hd, 0.25)

    def run():
        out, stats = torch.empty_like(t["q"]), torch.empty(batch * heads * seq_q * 2, device="cuda")
        dq, dk, dv = (torch.empty_like(t[n]) for n in ("q", "k", "v"))
        hip.cross_attention_forward(out, stats, t["q"], t["k"], t["v"], lens, *args)
        hip.cross_attention_backward(dq, dk, dv, t["dout"], out, t["q"], t["k"], t["v"], stats, lens, *args)
        return [x.reshape(batch, -1, n, d) for x, n in ((out, heads), (dq, heads), (dk, kv), (dv, kv))]

    want = run()
    head = heads - 1 if where in ("q", "dout") else kv - 1
    row = (seq_q if where in ("q", "dout") else lens[1].item()) // 2
    t[where][1, row, head * d + d // 2] = value
    got = run()
    key_head = head // group if where in ("q", "dout") else head
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        same = a == b
        if name in ("dk", "dv"):
            same[1, :, key_head] = True
        elif where in ("q", "dout"):
            same[1, row, head] = True
        else:
            same[1, :, key_head * group:(key_head + 1) * group] = True
        assert same.all(), (name, torch.argwhere(~same)[:3].tolist())
    if where != "dout":
        assert not torch.isfinite(got[0][1, row if where == "q" else 0, head if where == "q" else key_head * group]).all()


@pytest.mark.parametrize("shape", [
    (32, 8, 8, 1, 1500, 64), (2, 32, 8, 1, 16384, 128), (9, 4, 2, 8, 3000, 32), (8, 4, 4, 60, 4000, 64),
    (4, 16, 16, 512, 1500, 64), (3, 2, 1, 300, 9000, 128), (5, 6, 2, 400, 5000, 24), (2, 8, 8, 300, 7000, 96),
    (3, 2, 2, 1000, 40000, 16)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("most", [40, 200])
def test_short_lengths_in_a_long_cache(hip, shape, most):
    """Fewer key tiles are live than there are workgroups to share those of a full
    call."""
    check(hip, shape, 0, lens=[1 + (i + 1) * 7919 % most for i in range(shape[0])])


@pytest.mark.parametrize("shape", [(2, 4, 2, 3, 90, 32), (2, 4, 2, 90, 150, 64), (1, 2, 2, 150, 9, 40),
                                   (1, 3, 1, 70, 200, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("scale", [0.0, -0.25, 1.0])
def test_any_scale(hip, shape, scale):
    """Zero gives every live key the same weight, a negative one the most to the
    least product."""
    check(hip, shape, 0, scale=scale)


@pytest.mark.parametrize("shape", [(1, 2, 1, 200, 300, 64), (2, 4, 4, 1, 500, 128), (1, 2, 2, 150, 10, 24),
                                   (1, 3, 3, 20, 200, 96)], ids=lambda s: "x".join(map(str, s)))
def test_the_longest_strides(hip, shape):
    check(hip, shape, 0, ld=1 << 20)


@pytest.mark.parametrize("shape", [(1, 32768, 1, 2, 40, 32), (2, 8192, 2, 1, 20, 128), (1, 16384, 1, 1, 700, 64),
                                   (1, 1500, 1500, 1, 3, 8), (1, 600, 600, 50, 60, 16)],
                         ids=lambda s: "x".join(map(str, s)))
def test_many_heads(hip, shape):
    """Up to 32768, and as many to a key head: rows of up to 2^20 floats."""
    check(hip, shape, 0)


@pytest.mark.parametrize("seq_k,d", [(10, 64), (60, 64), (60, 24), (40, 100)])
def test_rows_past_32_bits(hip, seq_k, d):
    """Queries, outputs and their gradients whose offsets pass 2^31 floats. Sums of n
    rows get six times the deviation of n roundings without a common sign, 6 sqrt(n)
    half steps, as n half steps would be an eighth of them."""
    n, ld = (1 << 21) + 37, 1056
    print(f"{n} rows of stride {ld}, {seq_k} keys of {d}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(seq_k + d)
    new = lambda rows: torch.randn(rows, d, generator=gen, device="cuda")
    wide = [torch.empty(n, ld, device="cuda") for _ in range(4)]
    q, dout, out, dq = (x[:, :d] for x in wide)
    q.copy_(new(n))
    dout.copy_(new(n))
    dout[-5:] *= 1e5  # the last rows' share of the keys' gradients shows
    k, v = new(seq_k), new(seq_k)
    dk, dv, stats = torch.empty_like(k), torch.empty_like(v), torch.empty(2 * n, device="cuda")
    scale = torch.tensor(1 / math.sqrt(d)).item()
    args = (1, 1, 1, n, seq_k, d, ld, d, ld, scale)
    hip.cross_attention_forward(out, stats, q, k, v, None, *args)
    hip.cross_attention_backward(dq, dk, dv, dout, out, q, k, v, stats, None, *args)
    torch.cuda.synchronize()
    total, size, parts = [0.0, 0.0], [0.0, 0.0], 16
    for i in range(parts):
        rows = slice(n * i // parts, n * (i + 1) // parts)
        ref = reference(q[rows].double(), k.double(), v.double(), dout[rows].double(), scale)
        within(out[rows], *ref[0], "out")
        within(dq[rows], *ref[2], "dq")
        s = torch.softmax(mm(q[rows].double(), k.double().t()) * scale, dim=1)
        ds = s * (mm(dout[rows].double(), v.double().t()) - (dout[rows] * ref[0][0]).sum(1, keepdim=True)) * scale
        for at, (x, y) in enumerate(((ds, q), (s, dout))):
            total[at] = total[at] + mm(x.t(), y[rows].double())
            size[at] = size[at] + mm(x.abs().t(), y[rows].double().abs())
    for got, value, most in zip((dk, dv), total, size):
        # (each row's own error, gamma(...) in reference's bound, has no common sign either)
        assert ((got.double() - value).abs() <= (6 * math.sqrt(n) + 100) * U * most).all()
    last = mm(s[-5:].t(), y[-5:].double()).abs().max()
    assert last > 100 * ((6 * math.sqrt(n) + 100) * U * size[1]).min()
    del wide, q, dout, out, dq
    torch.cuda.empty_cache()


def test_the_most_rows(hip):
    """2^26 rows of one key: each takes its value, and the key gathers them all."""
    n = 1 << 26
    print(f"{n} rows", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(n, 1, generator=gen, device="cuda")
    dout = torch.empty(n, 1, device="cuda").random_(-3, 4, generator=gen)
    k, v = torch.ones(1, 1, device="cuda"), torch.full((1, 1), 2.0, device="cuda")
    out, dq, stats = torch.empty_like(q), torch.empty_like(q), torch.empty(2 * n, device="cuda")
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    args = (1, 1, 1, n, 1, 1, 1, 1, 1, 1.0)
    hip.cross_attention_forward(out, stats, q, k, v, None, *args)
    hip.cross_attention_backward(dq, dk, dv, dout, out, q, k, v, stats, None, *args)
    assert torch.all(out == 2.0) and torch.all(dq == 0.0) and dk.item() == 0.0
    # (whole numbers of at most 3 x 2^20 in a share's sum, and few shares)
    assert dv.item() == dout.double().sum().item()


@pytest.mark.parametrize("d", [1, 4])
def test_the_most_keys(hip, d):
    """2^26 keys of one row. A sum of n terms without a common sign of its roundings
    is off by 6 sqrt(n) half steps of the sum of magnitudes at most."""
    n = 1 << 26
    print(f"{n} keys of {d}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, dout = (torch.randn(1, d, generator=gen, device="cuda") for _ in range(2))
    k, v = (torch.randn(n, d, generator=gen, device="cuda") for _ in range(2))
    v[-3:] = 1e6  # the last keys' part shows
    out, dq, stats = torch.empty_like(q), torch.empty_like(q), torch.empty(2, device="cuda")
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    args = (1, 1, 1, 1, n, d, d, d, d, 1.0)
    hip.cross_attention_forward(out, stats, q, k, v, None, *args)
    hip.cross_attention_backward(dq, dk, dv, dout, out, q, k, v, stats, None, *args)
    # (sums by elements: the library's products refuse as many rows)
    along = lambda x, row: (x.double() * row.double()).sum(dim=1)
    down = lambda weight, x: (weight[:, None] * x.double()).sum(dim=0)
    p = torch.softmax(along(k, q), dim=0)
    some = 6 * math.sqrt(n) * U
    want, size = down(p, v), down(p, v.abs())
    ep = 2 * (gamma(d) + 4 * U) * along(k.abs(), q.abs()).max().item() + some + 8 * U
    assert ((out[0] - want).abs() <= (ep + some) * size).all()
    assert (down(p[-3:], v[-3:]).abs() > 3 * (ep + some) * size).all()
    assert ((dv - p[:, None] * dout.double()).abs() <= (ep + 4 * U) * p[:, None] * dout.double().abs() + TINY).all()
    del dv
    dp = along(v, dout)
    ds = p * (dp - (p * dp).sum())
    # dp - dout . out: d products' roundings, and those of out, whose bound is above
    e_ds = (ep + 4 * U) * ds.abs() + p * (gamma(d) * along(v.abs(), dout.abs())
                                          + ((ep + some + gamma(d)) * size * dout[0].double().abs()).sum())
    assert ((dk - ds[:, None] * q.double()).abs() <= (e_ds + 2 * U * ds.abs())[:, None] * q.double().abs() + TINY).all()
    assert ((dq[0] - down(ds, k)).abs() <= down(e_ds + some * ds.abs(), k.abs())).all()
    del k, v, dk, p, dp, ds, e_ds
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(1, 2, 2, 20, 90, 64), (1, 2, 2, 90, 30, 32), (1, 2, 2, 70, 90, 32),
                                   (1, 2, 2, 200, 150, 64), (1, 2, 2, 70, 90, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("small", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("power", [-90, -115, -130])
def test_small_magnitudes(hip, shape, small, power):
    """An operand of a product may be off by 2^-125, whichever kernel takes the
    call: with it, the bounds hold where a tensor, and what is made of it, is near
    the smallest floats or among the subnormal ones."""
    batch, heads, kv, seq_q, seq_k, d = shape
    print(f"cross attention {shape}, {small} about 2^{power}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(power + 1000)
    t = {n: torch.randn(rows, heads * d, generator=gen, device="cuda")
         for n, rows in (("q", seq_q), ("k", seq_k), ("v", seq_k), ("dout", seq_q))}
    t[small] = (t[small].double() * 2.0 ** power).float()
    out, stats = torch.empty_like(t["q"]), torch.empty(heads * seq_q * 2, device="cuda")
    dq, dk, dv = (torch.empty_like(t[n]) for n in ("q", "k", "v"))
    scale = torch.tensor(1 / math.sqrt(d)).item()
    args = (*shape, heads * d, heads * d, heads * d, scale)
    hip.cross_attention_forward(out, stats, t["q"], t["k"], t["v"], None, *args)
    hip.cross_attention_backward(dq, dk, dv, t["dout"], out, t["q"], t["k"], t["v"], stats, None, *args)
    for j in range(heads):
        c = slice(j * d, (j + 1) * d)
        ref = reference(*(t[n][:, c].double() for n in ("q", "k", "v", "dout")), scale, 2.0 ** -125)
        for got, (value, bound), name in zip((out, dq, dk, dv), ref[:1] + ref[2:], ("out", "dq", "dk", "dv")):
            within(got[:, c], value, bound, f"head {j}: {name}")
        if power == -90:  # (far above the smallest floats that adds next to nothing)
            plain = reference(*(t[n][:, c].double() for n in ("q", "k", "v", "dout")), scale)
            for (_, bound), (_, without) in zip(ref, plain):
                assert (bound - without).max() < 1e-3 * without.max()
