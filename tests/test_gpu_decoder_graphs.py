"""Rotary positions, masked attention and distillation as a decoder uses them: in place
on the rows of one projection, token by token over a cache, under HIP graph capture, on
another stream than the null stream, and over caches past 2^31 floats."""
import math

import numpy as np
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
    """A training step's calls on one set of buffers: the queries and keys of one
    projection turned in place, attention, its gradients into the projection's, turned
    back in place, and the loss of some logits."""

    B, H, KV, D, V, K = 2, 4, 2, 32, 301, 7

    def __init__(self, hip, seed, seq=70, own=True):
        self.hip, self.S = hip, seq
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = self.n = self.B * seq
        self.ld = (self.H + 2 * self.KV) * self.D
        self.source = torch.randn(n, self.ld, generator=g, device="cuda")
        self.qkv, self.dqkv = torch.empty_like(self.source), torch.empty_like(self.source)
        w = self.H * self.D
        self.dout, self.out = torch.randn(n, w, generator=g, device="cuda"), torch.empty(n, w, device="cuda")
        self.stats = torch.empty(self.B * self.H * seq * 2, device="cuda")
        self.positions = torch.arange(seq, device="cuda", dtype=torch.int32).repeat(self.B)
        self.freq = torch.exp2(-torch.arange(self.D // 2, device="cuda").float())
        self.begin = torch.zeros(n, device="cuda", dtype=torch.int32)
        self.lens = torch.tensor([seq, seq // 2], device="cuda", dtype=torch.int32)
        self.slopes = torch.tensor([0.5, 0.25, 0.1, 0.0], device="cuda")
        self.mask = hip.attention_mask(True, key_len=self.lens, key_begin=self.begin,
                                       slopes=self.slopes, cap=10.0)
        self.logits = torch.randn(n, self.V, generator=g, device="cuda")
        self.top = torch.randn(n, self.K, generator=g, device="cuda")
        self.ids = torch.randint(-1, self.V, (n, self.K), generator=g, device="cuda", dtype=torch.int32)
        self.labels = torch.randint(-1, self.V, (n,), generator=g, device="cuda", dtype=torch.int32)
        self.loss, self.dlogits = torch.empty(n, device="cuda"), torch.empty_like(self.logits)
        self.shape = (self.B, self.H, self.KV, seq, seq, self.D, self.ld, self.ld, w)
        self.work = [None, None]
        if own:
            self.work = [torch.empty(max(16, hip.masked_attention_workspace(*self.shape[:6], backward=b)) // 4,
                                     device="cuda") for b in (False, True)]

    def parts(self, t):
        q, k = self.H * self.D, (self.H + self.KV) * self.D
        return t[:, :q], t[:, q:k], t[:, k:]

    def run(self):
        hip = self.hip
        self.qkv.copy_(self.source)
        turn = (self.n, self.H + self.KV, self.D, self.D // 2, 1, self.ld, self.ld)
        hip.rotary_forward(self.qkv, self.qkv, self.positions, self.freq, None, *turn)
        q, k, v = self.parts(self.qkv)
        dq, dk, dv = self.parts(self.dqkv)
        scale = 1 / math.sqrt(self.D)
        hip.masked_attention_forward(self.out, self.stats, q, k, v, self.mask, *self.shape, scale,
                                     self.work[0])
        hip.masked_attention_backward(dq, dk, dv, self.dout, self.out, q, k, v, self.stats, self.mask,
                                      *self.shape, scale, work=self.work[1])
        hip.rotary_backward(self.dqkv, self.dqkv, self.positions, self.freq, None, *turn)
        hip.distill_backward(self.dlogits, self.loss, None, self.logits, self.top, self.ids,
                             self.labels, self.n, self.V, self.K, self.V, temperature=2.0, hard=0.3)

    def results(self):
        return [t.clone() for t in (self.qkv, self.out, self.dqkv, self.loss, self.dlogits)]

    def change(self, i):
        g = torch.Generator(device="cuda").manual_seed(1000 + i)
        self.source.copy_(torch.randn(self.source.shape, generator=g, device="cuda"))
        self.lens.copy_(torch.tensor([self.S - i, i], device="cuda"))
        self.begin.copy_((torch.arange(self.S, device="cuda") // (10 * i) * (10 * i)).repeat(self.B))
        self.positions.add_(i)
        self.logits.copy_(torch.randn(self.logits.shape, generator=g, device="cuda"))
        self.ids.copy_(torch.randint(-1, 5 * i, self.ids.shape, generator=g, device="cuda"))


@pytest.mark.parametrize("seq", [70, 5, 700])
def test_replays_equal_eager_calls(hip, side, seq):
    """Every replay, with inputs, masks and positions changed in between, and eager calls
    of the same operators in between, too."""
    print(f"graph replays, seq {seq}", flush=True)
    with torch.cuda.stream(side):
        step, other = Step(hip, 1, seq), Step(hip, 2, seq, own=False)
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.run()
        for i in range(1, 5):
            step.change(i)
            for t in (step.out, step.dqkv, step.dlogits, step.work[0], step.work[1]):
                t.fill_(float("nan"))
            graph.replay()
            got = step.results()
            other.change(i)
            other.run()  # uses and grows the library's own scratch
            torch.cuda.synchronize()
            step.run()
            for a, b in zip(got, step.results()):
                assert torch.equal(a, b)
                assert torch.isfinite(a).all()


def test_two_graphs_with_their_own_scratch(hip, side):
    with torch.cuda.stream(side):
        steps = [Step(hip, 3, 300), Step(hip, 4, 6)]
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
        q, k, v = step.parts(step.qkv)
        dq, dk, dv = step.parts(step.dqkv)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.loss.fill_(1.0)
            with pytest.raises(hip.NrsError, match="its own work buffer"):
                hip.masked_attention_backward(dq, dk, dv, step.dout, step.out, q, k, v, step.stats,
                                              step.mask, *step.shape, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.all(step.loss == 1.0)


def test_small_or_unaligned_scratch_is_refused(hip):
    step = Step(hip, 6)
    q, k, v = step.parts(step.qkv)
    dq, dk, dv = step.parts(step.dqkv)
    for bad, why in ((step.work[1][:-4], "needs"), (step.work[1][1:], "aligned")):
        with pytest.raises(hip.NrsError, match=why):
            hip.masked_attention_backward(dq, dk, dv, step.dout, step.out, q, k, v, step.stats,
                                          step.mask, *step.shape, 1.0, work=bad)


@pytest.mark.parametrize("draft", [1, 3])
def test_token_by_token_is_the_whole(hip, draft):
    """A cache filled `draft` tokens at a time (a place of three items, of which the
    second begins later, and rows behind the last token hold NaN), against one causal call
    over all. Both are within their f32 bound of the same sums: of values of size 1, 2 *
    (D + S + 32) * 2^-24 of them, times 4 for the scores' share."""
    B, H, KV, D, S = 3, 4, 2, 32, 45
    g = torch.Generator(device="cuda").manual_seed(9)
    ld = (H + 2 * KV) * D
    rows = torch.randn(B * S, ld, generator=g, device="cuda")
    at = torch.arange(S, device="cuda", dtype=torch.int32)
    freq = torch.exp2(-torch.arange(D // 2, device="cuda").float())
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    scale, q_end, k_end = 1 / math.sqrt(D), H * D, (H + KV) * D
    whole = rows.clone()
    hip.rotary_forward(whole, whole, at.repeat(B), freq, None, B * S, H + KV, D, D // 2, 1, ld, ld)
    want = torch.empty(B * S, H * D, device="cuda")
    hip.masked_attention_forward(want, None, whole[:, :q_end], whole[:, q_end:k_end], whole[:, k_end:],
                                 hip.attention_mask(True, slopes=slopes), B, H, KV, S, S, D, ld, ld,
                                 H * D, scale)
    room = S + 20
    cache = torch.full((B, room, 2 * KV * D), float("nan"), device="cuda")
    got = torch.full((B, S, H * D), float("nan"), device="cuda")
    late = torch.tensor([0, 9, 3], device="cuda", dtype=torch.int32)  # steps that an item waits
    for first in range(0, S + 9, draft):
        start = (first - late).clamp(min=0, max=S - draft)
        new = torch.empty(B * draft, ld, device="cuda")
        place = (start[:, None] + torch.arange(draft, device="cuda")).int()
        for b in range(B):
            new[b * draft:(b + 1) * draft] = rows.view(B, S, ld)[b, place[b].long()]
        hip.rotary_forward(new, new, place.reshape(-1).contiguous(), freq, None, B * draft, H + KV, D,
                           D // 2, 1, ld, ld)
        for b in range(B):
            cache[b, place[b].long()] = new[b * draft:(b + 1) * draft, q_end:]
        lens = (start + draft).int()
        out = torch.empty(B * draft, H * D, device="cuda")
        mask = hip.attention_mask(True, q_start=start.int(), key_len=lens, slopes=slopes)
        hip.masked_attention_forward(out, None, new[:, :q_end], cache[:, :, :KV * D], cache[:, :, KV * D:],
                                     mask, B, H, KV, draft, room, D, ld, 2 * KV * D, H * D, scale)
        for b in range(B):
            got[b, place[b].long()] = out.view(B, draft, -1)[b]
    assert torch.isfinite(got).all()
    bound = 4 * 2 * (D + S + 32) * 2.0 ** -24 * float(rows.abs().max())
    assert float((got.reshape(B * S, -1) - want).abs().max()) <= bound


@pytest.mark.parametrize("seq_q", [2, 40])
def test_caches_past_2_31_floats(hip, seq_q):
    """An item's keys reach past 2^32 floats; rows see the last few of them."""
    sk, ld, d = 2 ** 23 + 77, 520, 64
    kv = torch.empty(sk * ld, device="cuda")  # 17 GB; only the tail is set
    kv[:1].fill_(0)
    tail = 100
    g = torch.Generator(device="cuda").manual_seed(3)
    block = torch.randn(tail, ld, generator=g, device="cuda")
    kv[(sk - tail) * ld:] = block.reshape(-1)
    q, dout = (torch.randn(seq_q, d, generator=g, device="cuda") for _ in range(2))
    begin = torch.full((seq_q,), sk - 60, dtype=torch.int32, device="cuda")
    out, stats = torch.empty_like(q), torch.empty(2 * seq_q, device="cuda")
    mask = hip.attention_mask(True, key_begin=begin)
    # a small call with the same keys alone
    small_mask = hip.attention_mask(True, key_begin=torch.full_like(begin, tail - 60))
    small, small_stats = torch.empty_like(out), torch.empty_like(stats)
    shape = (1, 1, 1, seq_q, sk, d, d, ld, d)
    hip.masked_attention_forward(out, stats, q, kv, kv.data_ptr() + 4 * 256, mask, *shape, 0.125)
    tiny = (1, 1, 1, seq_q, tail, d, d, ld, d)
    hip.masked_attention_forward(small, small_stats, q, block, block.data_ptr() + 4 * 256, small_mask,
                                 *tiny, 0.125)
    # the same 60 keys: values of size 4 at most, sums of 60 and products of 64
    tol = 4 * 4 * (64 + 60 + 16) * 2.0 ** -24
    assert float((out - small).abs().max()) <= tol
    if seq_q == 2:
        return
    dq, small_dq = torch.empty_like(q), torch.empty_like(q)
    dkv = torch.empty_like(kv)
    small_dkv = torch.empty_like(block)
    hip.masked_attention_backward(dq, dkv, dkv.data_ptr() + 4 * 256, dout, out, q, kv,
                                  kv.data_ptr() + 4 * 256, stats, mask, *shape, 0.125)
    hip.masked_attention_backward(small_dq, small_dkv, small_dkv.data_ptr() + 4 * 256, dout, small, q,
                                  block, block.data_ptr() + 4 * 256, small_stats, small_mask, *tiny, 0.125)
    tol *= 64  # of dout . v and the sums over rows
    assert float((dq - small_dq).abs().max()) <= tol
    last = dkv[(sk - tail) * ld:].reshape(tail, ld)
    for c in (0, 256):
        assert float((last[:, c:c + d] - small_dkv[:, c:c + d]).abs().max()) <= tol
        assert torch.all(last[:tail - 60, c:c + d] == 0)
        assert torch.all(dkv[(sk // 2) * ld + c:(sk // 2) * ld + c + d] == 0)


def test_another_device_is_refused_or_absent(hip):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    step = Step(hip, 7)
    q, k, v = step.parts(step.qkv)
    with torch.cuda.device(1):
        with pytest.raises(hip.NrsError, match="is current"):
            hip.masked_attention_forward(step.out, step.stats, q, k, v, step.mask, *step.shape, 1.0)
        with pytest.raises(hip.NrsError, match="is current"):
            hip.rotary_forward(step.qkv, step.qkv, step.positions, step.freq, None, step.n, 6, 32, 16,
                               1, step.ld, step.ld)
        with pytest.raises(hip.NrsError, match="is current"):
            hip.distill_forward(step.loss, step.logits, step.top, step.ids, None, step.n, step.V,
                                step.K, step.V)


def test_distillation_of_rows_past_2_31_floats(hip):
    """65536 rows of a stride of 40000: only the last rows' values matter."""
    rows, vocab, ld = 65541, 333, 40000
    z = torch.zeros(rows * ld, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    last = torch.randn(3, vocab, generator=g, device="cuda")
    for i in range(3):
        z[(rows - 3 + i) * ld:(rows - 3 + i) * ld + vocab] = last[i]
    top = torch.randn(rows, 4, generator=g, device="cuda")
    ids = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda", dtype=torch.int32)
    loss, small = torch.empty(rows, device="cuda"), torch.empty(3, device="cuda")
    ones, few = torch.ones(rows, device="cuda"), torch.empty(3, vocab, device="cuda")
    hip.distill_backward(z, loss, ones, z, top, ids, None, rows, vocab, 4, ld)
    hip.distill_backward(few, small, ones, last, top[-3:].contiguous(), ids[-3:].contiguous(), None, 3,
                         vocab, 4, vocab)
    assert torch.equal(loss[-3:], small)
    for i in range(3):
        assert torch.equal(z[(rows - 3 + i) * ld:(rows - 3 + i) * ld + vocab], few[i])
    assert np.isclose(float(loss[0]), float(np.log(vocab) - _entropy(top[0], ids[0])), atol=1e-4)


def _entropy(top, ids):
    """Minus sum p log p of the places (a repeated token's are places of their own)."""
    p = torch.softmax(top.double(), 0)
    return -(p * p.log()).sum().item()
