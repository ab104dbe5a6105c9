"""Cross attention, embedding and dropout under HIP graph capture, on another
stream than the null stream, and on tensors past 2^31 floats."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def side(hip):
    """A stream of torch's that is the library's, too, until the test ends."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    hip.call("nrs_set_stream", s.cuda_stream)
    yield s
    torch.cuda.synchronize()
    hip.call("nrs_set_stream", None)


class Step:
    """A training step's calls on one set of buffers: tokens through the
    embedding, dropout, attention over given states, and all gradients."""

    B, H, KV, SQ, SK, D, V, P = 2, 4, 2, 70, 300, 32, 50, 0.3

    def __init__(self, hip, seed, own=True, seq_q=None):
        self.hip = hip
        if seq_q:
            self.SQ = seq_q
        g = torch.Generator(device="cuda").manual_seed(seed)
        n, w, kw = self.B * self.SQ, self.H * self.D, self.KV * self.D
        self.n, self.w = n, w
        self.ids = torch.randint(-1, self.V, (n,), generator=g, device="cuda", dtype=torch.int32)
        self.lens = torch.tensor([self.SK, self.SK // 2], dtype=torch.int32, device="cuda")
        self.step = torch.zeros(1, dtype=torch.int64, device="cuda")
        new = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.table, self.dout = new(self.V, w), new(n, w)
        self.k, self.v = new(self.B * self.SK, kw), new(self.B * self.SK, kw)
        self.x, self.q, self.out, self.dq, self.dx = (torch.empty(n, w, device="cuda") for _ in range(5))
        self.stats = torch.empty(self.B * self.H * self.SQ * 2, device="cuda")
        self.dk, self.dv, self.dtable = (torch.empty_like(t) for t in (self.k, self.v, self.table))
        self.shape = (self.B, self.H, self.KV, self.SQ, self.SK, self.D, w, kw, w)
        size = lambda b: torch.empty(max(16, b) // 4, device="cuda")
        self.work = [None] * 3
        if own:
            self.work = [size(hip.cross_attention_workspace(*self.shape[:6])),
                         size(hip.cross_attention_workspace(*self.shape[:6], backward=True)),
                         size(hip.embedding_workspace(n, self.V, w))]

    def run(self):
        hip, n, w, scale = self.hip, self.n, self.w, 1 / math.sqrt(self.D)
        hip.embedding_forward(self.x, self.table, self.ids, n, self.V, w, 1.5)
        hip.dropout_forward(self.q, self.x, None, n * w, self.P, 7, 3, self.step)
        hip.cross_attention_forward(self.out, self.stats, self.q, self.k, self.v, self.lens,
                                    *self.shape, scale, self.work[0])
        hip.cross_attention_backward(self.dq, self.dk, self.dv, self.dout, self.out, self.q, self.k,
                                     self.v, self.stats, self.lens, *self.shape, scale,
                                     work=self.work[1])
        hip.dropout_backward(self.dx, self.dq, n * w, self.P, 7, 3, self.step)
        hip.embedding_backward(self.dtable, self.dx, self.ids, n, self.V, w, 1.5, work=self.work[2])

    def results(self):
        return [t.clone() for t in (self.x, self.q, self.out, self.dk, self.dv, self.dx, self.dtable)]

    def change(self, i):
        g = torch.Generator(device="cuda").manual_seed(1000 + i)
        self.ids.copy_(torch.randint(-1, self.V, self.ids.shape, generator=g, device="cuda"))
        self.k.copy_(torch.randn(self.k.shape, generator=g, device="cuda"))
        self.lens.copy_(torch.tensor([self.SK - i, 17 * i], device="cuda"))
        self.step.fill_(i)


@pytest.mark.parametrize("seq_q", [70, 1, 300])
def test_replays_equal_eager_calls(hip, side, seq_q):
    """Every replay, with inputs, lengths and the dropout's step changed in
    between and eager calls of the same operators in between, too."""
    print(f"graph replays, seq_q {seq_q}", flush=True)
    with torch.cuda.stream(side):
        step, other = Step(hip, 1, seq_q=seq_q), Step(hip, 2, own=False)
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.run()
        for i in range(1, 5):
            step.change(i)
            for t in (step.out, step.dk, step.dtable, step.work[0], step.work[1], step.work[2]):
                t.fill_(float("nan"))
            graph.replay()
            got = step.results()
            other.change(i)
            other.run()  # uses and grows the library's own scratch
            torch.cuda.synchronize()
            step.run()
            for a, b in zip(got, step.results()):
                assert torch.equal(a, b)
        assert not torch.equal(step.results()[1], got[1] * 0)


def test_two_graphs_with_their_own_scratch(hip, side):
    with torch.cuda.stream(side):
        steps = [Step(hip, 3), Step(hip, 4, seq_q=1)]
        graphs = []
        for s in steps:
            s.run()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                s.run()
            graphs.append(g)
        for i in range(1, 4):
            for s in steps:
                s.change(i)
            for g in graphs + graphs:
                g.replay()
            got = [s.results() for s in steps]
            torch.cuda.synchronize()
            for s, r in zip(steps, got):
                s.run()
                for a, b in zip(r, s.results()):
                    assert torch.equal(a, b)


def test_capture_without_scratch_is_refused(hip, side):
    with torch.cuda.stream(side):
        step = Step(hip, 5, own=False)
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.x.fill_(1.0)
            with pytest.raises(hip.NrsError, match="its own work buffer"):
                hip.cross_attention_backward(step.dq, step.dk, step.dv, step.dout, step.out, step.q,
                                             step.k, step.v, step.stats, step.lens, *step.shape, 1.0)
            with pytest.raises(hip.NrsError, match="its own work buffer"):
                hip.embedding_backward(step.dtable, step.dx, step.ids, step.n, step.V, step.w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.all(step.x == 1.0)


def test_small_or_unaligned_scratch_is_refused(hip):
    step = Step(hip, 6)
    for bad, why in ((step.work[1][:-4], "needs"), (step.work[1][1:], "aligned")):
        with pytest.raises(hip.NrsError, match=why):
            hip.cross_attention_backward(step.dq, step.dk, step.dv, step.dout, step.out, step.q, step.k,
                                         step.v, step.stats, step.lens, *step.shape, 1.0, work=bad)
    with pytest.raises(hip.NrsError, match="needs"):
        hip.embedding_backward(step.dtable, step.dx, step.ids, step.n, step.V, step.w,
                               work=step.work[2][:4])


@pytest.mark.parametrize("seq_q", [1, 50])
def test_keys_past_32_bits(hip, seq_q):
    """Keys and values whose offsets pass 2^31 floats. The reference is in 64
    bits on the device; the bound is attention_ref's, for these sizes: scores
    of 64 products, sums of n keys."""
    n, d, ld = (1 << 21) + 37, 64, 1056
    print(f"{n} keys of stride {ld}, {seq_q} rows", flush=True)
    g = torch.Generator(device="cuda").manual_seed(7)
    kv = torch.empty(n, ld, device="cuda")
    k, v = kv[:, :d], kv[:, d:2 * d]
    for t in (k, v):
        t.copy_(torch.randn(n, d, generator=g, device="cuda"))
    q, dout = (torch.randn(seq_q, d, generator=g, device="cuda") for _ in range(2))
    # the last keys weigh most
    k[-5:] = q[:1] * 2
    out, stats = torch.empty_like(q), torch.empty(2 * seq_q, device="cuda")
    shape = (1, 1, 1, seq_q, n, d, d, ld, d)
    scale = 1 / math.sqrt(d)
    hip.cross_attention_forward(out, stats, q, k, v, None, *shape, scale)
    dkv, dq = torch.empty_like(kv), torch.empty_like(q)
    hip.cross_attention_backward(dq, dkv[:, :d], dkv[:, d:2 * d], dout, out, q, k, v, stats, None,
                                 *shape, scale)
    q64, k64, v64, g64 = (t.double() for t in (q, k, v, dout))
    s = torch.mm(q64, k64.t().contiguous()) * scale
    p = torch.softmax(s, dim=1)
    want = torch.mm(p, v64)
    u = 2.0 ** -24
    es = (64 + 12) * u * (torch.mm(q64.abs(), k64.abs().t().contiguous()) * scale).amax(dim=1, keepdim=True)
    # A sum of n floats is off by at most n half steps, 1/8 of its size here; the
    # roundings have no common sign, so the bound is six times the deviation of
    # that many, 6 sqrt(n) half steps, which the sums of n keys get.
    n_keys, n_d = 6 * math.sqrt(n) * u, (d + 8) * u
    ep = 2 * es + n_keys
    size = torch.mm(p, v64.abs())
    out_bound = (ep + n_keys) * size
    assert torch.all((out - want).abs() <= out_bound)
    dp = torch.mm(g64, v64.t().contiguous())
    delta = (g64 * want).sum(dim=1, keepdim=True)
    ds = p * (dp - delta) * scale
    e_ds = scale * p * ((ep + 4 * u) * (dp - delta).abs()
                        + n_d * torch.mm(g64.abs(), v64.abs().t().contiguous())
                        + (n_d * g64.abs() * want.abs() + g64.abs() * out_bound).sum(dim=1, keepdim=True))
    rows = (seq_q + 8) * u
    for got, value, bound in (
            (dq, torch.mm(ds, k64), torch.mm(e_ds + n_keys * ds.abs(), k64.abs())),
            (dkv[:, :d], torch.mm(ds.t().contiguous(), q64),
             torch.mm((e_ds + rows * ds.abs()).t().contiguous(), q64.abs())),
            (dkv[:, d:2 * d], torch.mm(p.t().contiguous(), g64),
             torch.mm((ep * p + rows * p).t().contiguous(), g64.abs()))):
        assert torch.all((got - value).abs() <= bound + 2.0 ** -24 * value.abs() + 2.0 ** -126)
    # (and the rows behind the 32nd bit hold more than rounding can)
    assert value[-5:].abs().max() > 100 * bound[-5:].max()


def test_an_embedding_gradient_of_few_positions_takes_no_scratch(hip):
    """The one launch of up to 256 positions writes to none: without a work buffer
    the library's own scratch does not grow (by a place for each of 2^28 tokens)."""
    count, vocab = 200, 1 << 28
    hip.call("nrs_shutdown")  # gives the scratch of earlier calls back
    table = torch.zeros(vocab, device="cuda")
    grad = torch.ones(count, device="cuda")
    ids = torch.arange(count, device="cuda", dtype=torch.int32) * (vocab // count)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    print(f"embedding, {count} of {vocab}", flush=True)
    for beta in (0.0, 1.0):
        hip.embedding_backward(table, grad, ids, count, vocab, 1, 1.0, beta)
    hip.sync()
    taken = before - torch.cuda.mem_get_info()[0]
    assert taken < 1 << 28
    assert torch.count_nonzero(table) == count and torch.all(table[ids.long()] == 2.0)
    del table
    torch.cuda.empty_cache()


@pytest.mark.parametrize("advance,again", [(3, False), (1, True)])
def test_masks_of_replays_with_several_dropouts(hip, side, advance, again):
    """Three dropouts of calls 0, 1 and 2 under one seed: no mask of a replay comes
    again in another when the program adds at least 3 to *step, and the next
    dropout's mask is this one's when it adds 1."""
    n = 4096
    print(f"dropouts, step + {advance}", flush=True)
    with torch.cuda.stream(side):
        x, step = torch.ones(n, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
        outs = [torch.empty(n, device="cuda") for _ in range(3)]

        def run():
            for call, out in enumerate(outs):
                hip.dropout_forward(out, x, None, n, 0.5, 9, call, step)

        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        masks = []
        for i in range(4):
            step.fill_(advance * i)
            graph.replay()
            masks += [out.clone() for out in outs]
            torch.cuda.synchronize()
            run()
            for out, mask in zip(outs, masks[-3:]):
                assert torch.equal(out, mask)
    same = [(i, j) for i in range(len(masks)) for j in range(i) if torch.equal(masks[i], masks[j])]
    assert bool(same) == again
    if again:  # call 0 of the next replay is call 1 of this one
        assert (3, 1) in same
