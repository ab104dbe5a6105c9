"""Calls that reach every kernel that masked attention's planner can choose
(tests/masked_plan.py), with each way to make scores, against the algebra in 64 bits on
the GPU, head by head (of the larger calls, some of them). The bounds are those of
masked_ref.py, whose derivation stands there."""
import math

import pytest
import torch

import masked_plan
from attention_ref import TINY, U, gamma

pytestmark = pytest.mark.gpu

MODES = ("plain", "slopes", "cap")


class Call:
    """A call's tensors, with masks of every kind: causal, documents of odd lengths, a
    length for each item, and keys that no row sees, which hold NaN."""

    def __init__(self, hip, shape, mode, causal=True):
        self.hip, self.shape6 = hip, shape
        self.B, self.H, self.KV, self.SQ, self.SK, self.D = shape
        g = torch.Generator(device="cuda").manual_seed(sum(shape))
        new = lambda *s: torch.randn(*s, generator=g, device="cuda")
        B, H, KV, SQ, SK, D = shape
        self.q, self.dout = new(B * SQ, H * D), new(B * SQ, H * D)
        self.k, self.v = new(B * SK, KV * D), new(B * SK, KV * D)
        self.lens = torch.tensor([SK - b * (SK // (2 * B)) for b in range(B)], dtype=torch.int32,
                                 device="cuda")
        # a document in five begins within the last eighth: the others see far back
        at = torch.arange(SQ, device="cuda")
        self.begin = torch.where(at % 5 == 0, (at - 1 - at % 77) * max(1, SK // max(SQ, 1)) * 7 // 8, 0)
        self.begin = self.begin.clamp(min=0).repeat(B).int()
        self.slopes = None
        if mode == "slopes":
            self.slopes = torch.exp2(-4.0 - 4.0 * torch.arange(H, device="cuda") / H)
        self.cap = 3.0 if mode == "cap" else 0.0
        self.scale = 1.0 / math.sqrt(D)
        self.mask = hip.attention_mask(causal, key_len=self.lens, key_begin=self.begin,
                                       slopes=self.slopes, cap=self.cap)
        for b in range(B):
            rows = slice(b * SK, (b + 1) * SK)
            dead = ~self.visible(b).any(dim=0)
            self.k[rows][dead] = math.nan
            self.v[rows][dead] = math.nan
        self.out, self.dq = torch.empty_like(self.q), torch.full_like(self.q, math.nan)
        self.dk, self.dv = torch.full_like(self.k, math.nan), torch.full_like(self.v, math.nan)
        self.stats = torch.empty(B * H * SQ * 2, device="cuda")

    def visible(self, b):
        t = torch.arange(self.SK, device="cuda")[None, :]
        i = (self.SK - self.SQ + torch.arange(self.SQ, device="cuda"))[:, None]
        begin = self.begin[b * self.SQ:(b + 1) * self.SQ, None]
        see = (t < self.lens[b]) & (t >= begin)
        return see & (t <= i) if self.mask.causal else see

    def run(self, backward):
        shape = (*self.shape6, self.H * self.D, self.KV * self.D, self.H * self.D)
        work = [torch.full((max(16, self.hip.masked_attention_workspace(*self.shape6, backward=b)) // 4,),
                           math.nan, device="cuda") for b in (False, True)]
        self.hip.masked_attention_forward(self.out, self.stats if backward else None, self.q, self.k,
                                          self.v, self.mask, *shape, self.scale, work[0])
        if backward:
            self.hip.masked_attention_backward(self.dq, self.dk, self.dv, self.dout, self.out, self.q,
                                               self.k, self.v, self.stats, self.mask, *shape,
                                               self.scale, work=work[1])

    def check(self, b, j, backward):
        """Key head j of item b: all its query heads."""
        D, SQ, SK, group = self.D, self.SQ, self.SK, self.H // self.KV
        rows, keys = slice(b * SQ, (b + 1) * SQ), slice(b * SK, (b + 1) * SK)
        kc = slice(j * D, (j + 1) * D)
        see = self.visible(b)
        dead = ~see.any(dim=0)
        k, v = self.k[keys, kc].double(), self.v[keys, kc].double()
        k[dead] = 0.0
        v[dead] = 0.0
        sums = [torch.zeros(SK, D, dtype=torch.float64, device="cuda") for _ in range(4)]
        i = (SK - SQ + torch.arange(SQ, device="cuda"))[:, None]
        t = torch.arange(SK, device="cuda")[None, :]
        scale = float(torch.tensor(self.scale, dtype=torch.float32))
        for h in range(j * group, (j + 1) * group):
            cols = slice(h * D, (h + 1) * D)
            q, g = self.q[rows, cols].double(), self.dout[rows, cols].double()
            x = q @ k.t() * scale
            e_u = gamma(D) * scale * (q.abs() @ k.abs().t())
            inner, e_inner = 1.0, 0.0
            if self.cap:
                th = torch.tanh(x / self.cap)
                inner = 1.0 - th * th
                e_inner = 2 * th.abs() * (e_u / self.cap * inner + 4 * U * th.abs()) + 2 * U
                x = self.cap * th
                e_u = e_u * inner + 6 * U * x.abs()
            if self.slopes is not None:
                far = (i - t).abs()
                near = torch.where(see, far, 2 ** 62).amin(dim=1, keepdim=True)
                bias = float(self.slopes[h]) * torch.where(see, far - near, 0)
                x = x - bias
                e_u = e_u + 3 * U * bias
            any_seen = see.any(dim=1, keepdim=True)
            m = torch.where(any_seen, x.masked_fill(~see, -math.inf).amax(dim=1, keepdim=True), 0.0)
            e = torch.exp((x - m).masked_fill(~see, -math.inf))
            total = torch.where(any_seen, e.sum(dim=1, keepdim=True), 1.0)
            p = e / total
            es = torch.where(see, e_u + 4 * U * (x.abs() + (m + torch.log(total)).abs()), 0.0)
            ep = es + (p * es).sum(dim=1, keepdim=True) + gamma(SK) + 8 * U
            out = p @ v
            b_out = (p * (ep + gamma(SK))) @ v.abs() + TINY * (see.double() @ v.abs())
            self.compare(self.out[rows, cols], out, b_out, f"out {b} {h}")
            if not backward:
                continue
            dp = g @ v.t()
            delta = (g * out).sum(dim=1, keepdim=True)
            diff = (dp - delta).abs()
            ds = p * (dp - delta) * inner * scale
            e_dp = gamma(D) * (g.abs() @ v.abs().t())
            e_delta = (gamma(D) * (g.abs() * out.abs()) + g.abs() * b_out).sum(dim=1, keepdim=True)
            e_ds = scale * p * (((ep + 4 * U) * diff + e_dp + e_delta) * inner + diff * e_inner)
            e_ds = torch.where(see, e_ds + TINY * (1 + scale * diff), 0.0)
            e_p = torch.where(see, ep * p + TINY, 0.0)
            n = SQ * group
            self.compare(self.dq[rows, cols], ds @ k,
                         e_ds @ k.abs() + gamma(SK) * (ds.abs() @ k.abs()), f"dq {b} {h}")
            for at, part in enumerate((ds.t().contiguous() @ q,
                                       e_ds.t().contiguous() @ q.abs() + gamma(n) * (ds.abs().t().contiguous() @ q.abs()),
                                       p.t().contiguous() @ g,
                                       e_p.t().contiguous() @ g.abs() + gamma(n) * (p.t().contiguous() @ g.abs()))):
                sums[at] += part
        if backward:
            self.compare(self.dk[keys, kc], sums[0], sums[1], f"dk {b} {j}")
            self.compare(self.dv[keys, kc], sums[2], sums[3], f"dv {b} {j}")

    @staticmethod
    def compare(got, value, bound, what):
        tol = bound + U * value.abs() + 2.0 ** -126
        bad = ~((got - value).abs() <= tol)
        assert not bool(bad.any()), (what, int(bad.sum()), float(((got - value).abs() / tol).max()))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("shape", masked_plan.SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_every_kernel(hip, shape, mode):
    print(f"masked attention {shape} {mode}", flush=True)
    call = Call(hip, shape, mode)
    backward = shape[3] > 3
    call.run(backward)
    work = shape[3] * shape[4]
    picked = {(0, 0), (shape[0] - 1, shape[2] - 1)}
    if work < 10 ** 6:
        picked |= {(b, j) for b in range(shape[0]) for j in range(shape[2])}
    for b, j in sorted(picked)[:6 if work < 10 ** 6 else 2]:
        call.check(b, j, backward)


@pytest.mark.parametrize("shape", [(2, 4, 2, 500, 500, 64), (4, 16, 16, 1800, 2000, 128)], ids=str)
def test_not_causal(hip, shape):
    call = Call(hip, shape, "slopes", causal=False)
    call.run(True)
    call.check(0, 0, True)
    call.check(shape[0] - 1, shape[2] - 1, True)
