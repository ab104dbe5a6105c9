"""Masked attention in 64 bits, with bounds on what f32 arithmetic may differ.

The bounds are first-order worst cases, as in attention_ref.py: u = 2^-24 is half a
step of f32, gamma(n) = (n + 8) u. Per score x = scale q.k, taken as a sum of d
products, off by e_x = gamma(d) sum |q||k| scale. The cap: y = x / cap (a rounding),
t = tanh(y), computed to 4 u of itself and 1-Lipschitz, cap t (a rounding): e_u =
e_x + 6 u |cap t|. The bias is slope times a whole distance (exact as a float),
relative to the row's nearest key: 3 u of it for the factor log2 e, the product and
the sum. Changing to base 2 and the subtraction of the row's reference (or of its log
sum) round to u of each of them: 4 u (|score| + |log sum|). The error of an exponent
is a relative one of its probability; the row's sum has the average of them.
"""
import numpy as np

from attention_ref import TINY, U, gamma


class Problem:
    """Inputs of one call in the library's layout, and its reference."""

    def __init__(self, batch, heads, kv_heads, seq_q, seq_k, d, causal=True, q_start=None,
                 key_len=None, prefix_len=None, key_begin=None, key_end=None, slopes=False, cap=0.0,
                 pad_q=0, pad_kv=0, packed=False, seed=0, magnitude=1.0):
        self.batch, self.heads, self.kv, self.sq, self.sk, self.d = batch, heads, kv_heads, seq_q, seq_k, d
        self.group = heads // kv_heads
        self.ld_q = heads * d + pad_q
        self.ld_out = heads * d + (pad_q and pad_q + 3)
        self.ld_kv = kv_heads * d * (2 if packed else 1) + pad_kv
        self.v_at = kv_heads * d if packed else 0
        self.packed = packed
        self.scale = np.float32(1.0 / np.sqrt(d))
        self.causal, self.cap = causal, float(np.float32(cap))

        def ints(x, shape):
            return None if x is None else np.broadcast_to(np.asarray(x, np.int32), shape).copy()

        self.q_start, self.key_len = ints(q_start, (batch,)), ints(key_len, (batch,))
        self.prefix_len = ints(prefix_len, (batch,))
        self.key_begin, self.key_end = ints(key_begin, (batch, seq_q)), ints(key_end, (batch, seq_q))
        rng = np.random.default_rng(seed)
        self.slopes = (2.0 ** -rng.uniform(0.5, 8.0, heads)).astype(np.float32) if slopes else None

        def rows(n, ld):
            return (rng.standard_normal((n, ld)) * magnitude).astype(np.float32)

        self.q, self.dout = rows(batch * seq_q, self.ld_q), rows(batch * seq_q, self.ld_out)
        self.k = rows(batch * seq_k, self.ld_kv)
        self.v = self.k if packed else rows(batch * seq_k, self.ld_kv)
        # keys that no row of their item sees must not change anything
        for b in range(batch):
            dead = ~self.visible(b).any(axis=0)
            self.k[b * seq_k:(b + 1) * seq_k][dead] = np.nan
            self.v[b * seq_k:(b + 1) * seq_k][dead] = np.nan

    def positions(self, b):
        start = self.sk - self.sq if self.q_start is None else int(self.q_start[b])
        return start + np.arange(self.sq, dtype=np.int64)

    def visible(self, b):
        """[seq_q, seq_k]: the definition, key by key."""
        t = np.arange(self.sk)[None, :]
        see = np.ones((self.sq, self.sk), bool)
        if self.key_len is not None:
            see &= t < self.key_len[b]
        if self.causal:
            prefix = 0 if self.prefix_len is None else self.prefix_len[b]
            see &= (t <= self.positions(b)[:, None]) | (t < prefix)
        if self.key_begin is not None:
            see &= t >= self.key_begin[b][:, None]
        if self.key_end is not None:
            see &= t < self.key_end[b][:, None]
        return see

    def shape(self):
        return (self.batch, self.heads, self.kv, self.sq, self.sk, self.d, self.ld_q, self.ld_kv,
                self.ld_out)

    def one(self, b, h, gradients=True):
        """out, dq, dk, dv of a head and their bounds; dk and dv are this head's part."""
        d, L = self.d, self.sk
        rows, cols = slice(b * self.sq, (b + 1) * self.sq), slice(h * d, (h + 1) * d)
        j = h // self.group
        q, g = (x[rows, cols].astype(np.float64) for x in (self.q, self.dout))
        k = self.k[b * L:(b + 1) * L, j * d:(j + 1) * d].astype(np.float64)
        v = self.v[b * L:(b + 1) * L, self.v_at + j * d:self.v_at + (j + 1) * d].astype(np.float64)
        see = self.visible(b)
        dead = ~see.any(axis=0)
        k[dead] = v[dead] = 0.0
        scale = float(self.scale)
        x = q @ k.T * scale
        e_u = gamma(d) * (np.abs(q) @ np.abs(k).T * abs(scale))
        t, inner, e_inner = np.zeros_like(x), np.ones_like(x), np.zeros_like(x)
        if self.cap:
            t = np.tanh(x / self.cap)
            inner = 1.0 - t * t
            # 1 - t t: two roundings, and t's own error twice
            e_inner = 2 * np.abs(t) * (e_u / self.cap * inner + 4 * U * np.abs(t)) + 2 * U
            x = self.cap * t
            e_u = e_u * inner + 6 * U * np.abs(x)
        if self.slopes is not None:
            far = np.abs(self.positions(b)[:, None] - np.arange(L)[None, :])
            near = np.where(see, far, np.iinfo(np.int64).max).min(axis=1, keepdims=True)
            bias = float(self.slopes[h]) * np.where(see, far - near, 0)
            x = x - bias
            e_u = e_u + 3 * U * bias
        any_seen = see.any(axis=1, keepdims=True)
        x = np.where(see, x, -np.inf)
        m = np.where(any_seen, x.max(axis=1, keepdims=True, initial=-np.inf), 0.0)
        e = np.exp(x - m)
        total = np.where(any_seen, e.sum(axis=1, keepdims=True), 1.0)
        p = e / total
        lse = np.abs(m + np.log(total))
        es = np.where(see, e_u + 4 * U * (np.abs(np.where(see, x, 0.0)) + lse), 0.0)
        ep = es + (p * es).sum(axis=1, keepdims=True) + gamma(L) + 8 * U
        out = p @ v
        b_out = (p * (ep + gamma(L))) @ np.abs(v) + TINY * (see @ np.abs(v))
        if not gradients:
            return (out, b_out), None, None, None
        dp = g @ v.T
        delta = (g * out).sum(axis=1, keepdims=True)
        ds = p * (dp - delta) * inner * scale
        e_dp = gamma(d) * (np.abs(g) @ np.abs(v).T)
        e_delta = (gamma(d) * (np.abs(g) * np.abs(out)) + np.abs(g) * b_out).sum(axis=1, keepdims=True)
        diff = np.abs(dp - delta)
        e_ds = abs(scale) * p * (((ep + 4 * U) * diff + e_dp + e_delta) * np.abs(inner) + diff * e_inner)
        e_ds = np.where(see, e_ds + TINY * (1 + abs(scale) * diff), 0.0)
        e_p = np.where(see, ep * p + TINY, 0.0)
        R = self.sq * self.group
        dq = (ds @ k, e_ds @ np.abs(k) + gamma(L) * (np.abs(ds) @ np.abs(k)))
        dk = (ds.T @ q, e_ds.T @ np.abs(q) + gamma(R) * (np.abs(ds).T @ np.abs(q)))
        dv = (p.T @ g, e_p.T @ np.abs(g) + gamma(R) * (p.T @ np.abs(g)))
        return (out, b_out), dq, dk, dv

    def reference(self, gradients=True):
        """out and the gradients, each as (value, bound) arrays of the tensors' own
        layout without the padding columns."""
        zq = (self.batch * self.sq, self.heads * self.d)
        zk = (self.batch * self.sk, self.kv * self.d)
        r = {n: (np.zeros(zq), np.zeros(zq)) for n in ("out", "dq")}
        r.update({n: (np.zeros(zk), np.zeros(zk)) for n in ("dk", "dv")})
        for b in range(self.batch):
            for h in range(self.heads):
                rows, cols = slice(b * self.sq, (b + 1) * self.sq), slice(h * self.d, (h + 1) * self.d)
                j = h // self.group
                kr, kc = slice(b * self.sk, (b + 1) * self.sk), slice(j * self.d, (j + 1) * self.d)
                for name, got, at in zip(("out", "dq", "dk", "dv"), self.one(b, h, gradients),
                                         ((rows, cols), (rows, cols), (kr, kc), (kr, kc))):
                    if got is not None:
                        r[name][0][at] += got[0]
                        r[name][1][at] += got[1]
        return r
