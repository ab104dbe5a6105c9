"""Cross attention in 64 bits, with bounds on what f32 arithmetic may differ.

One (item, key head) at a time: q [R, d] the rows of all its query heads,
k, v [L, d] its live keys.

The bounds are first-order worst cases. u = 2^-24 is half a step of f32; a
sum of n products taken in any order is off by at most (n + c) u times the sum
of the products' magnitudes, c = 8 counting the rounding of the operands'
scale, of the products (2 u when they are made of bf16 pieces) and of the
result. The error of an exponent is an absolute one and becomes a relative one
of its probability (e = the score's error, twice: the row's sum has it too).
"""
import numpy as np

U = 2.0 ** -24
# What a weight (p or ds) may lose absolutely: an exponential under 2^-126, the
# smallest normal float, may come out as zero, and so may the weight's product
# or the pieces of it that are under that: 2^-126 each.
TINY = 2 * 2.0 ** -126


def gamma(n):
    return (n + 8) * U


def forward(q, k, v, scale):
    """out, (max, sum) in base 2, and the bound of out."""
    if len(k) == 0:
        zero = np.zeros((len(q), v.shape[1]))
        return zero, np.zeros((len(q), 2)), zero, np.zeros((len(q), 0)), np.zeros((len(q), 1))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    s = q @ k.T * scale
    m = s.max(axis=1, keepdims=True)
    e = np.exp(s - m)
    total = e.sum(axis=1, keepdims=True)
    p = e / total
    # scores: the products, and log2 e folded into the scale of the operand;
    # the exponential's own error (2 u) and the subtraction of the maximum
    # (u times the score) are in the 4 of the next line
    es = (gamma(q.shape[1]) + 4 * U) * (np.abs(q) @ np.abs(k).T * abs(scale)).max(axis=1, keepdims=True)
    ep = 2 * es + gamma(len(k)) + 8 * U  # relative error of p
    bound = (ep + gamma(len(k))) * (p @ np.abs(v)) + TINY * np.abs(v).sum(axis=0)
    return p @ v, np.concatenate([m * np.log2(np.e), total], axis=1), bound, p, ep


def backward(q, k, v, g, scale):
    """(dq, dk, dv) and their bounds."""
    out, _, out_bound, p, ep = forward(q, k, v, scale)
    q, k, v, g = (x.astype(np.float64) for x in (q, k, v, g))
    if len(k) == 0:
        z = [np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)]
        return z, z
    d, L, R = q.shape[1], len(k), len(q)
    dp = g @ v.T
    delta = (g * out).sum(axis=1, keepdims=True)
    ds = p * (dp - delta) * scale
    e_dp = gamma(d) * (np.abs(g) @ np.abs(v).T)
    e_delta = (gamma(d) * (np.abs(g) * np.abs(out)) + np.abs(g) * out_bound).sum(axis=1, keepdims=True)
    e_ds = abs(scale) * p * ((ep + 4 * U) * np.abs(dp - delta) + e_dp + e_delta)
    e_ds += TINY * (1 + abs(scale) * np.abs(dp - delta))
    e_p = ep * p + TINY
    dq, dk, dv = ds @ k, ds.T @ q, p.T @ g
    bounds = [e_ds @ np.abs(k) + gamma(L) * (np.abs(ds) @ np.abs(k)),
              e_ds.T @ np.abs(q) + gamma(R) * (np.abs(ds).T @ np.abs(q)),
              e_p.T @ np.abs(g) + gamma(R) * (p.T @ np.abs(g))]
    return [dq, dk, dv], bounds


class Problem:
    """Inputs of one call in the library's layout, and its reference."""

    def __init__(self, batch, heads, kv_heads, seq_q, seq_k, d, lens=None, pad_q=0, pad_kv=0,
                 packed=False, seed=0, magnitude=1.0):
        self.batch, self.heads, self.kv, self.sq, self.sk, self.d = batch, heads, kv_heads, seq_q, seq_k, d
        self.group = heads // kv_heads
        self.ld_q = heads * d + pad_q
        self.ld_out = heads * d + (pad_q and pad_q + 3)
        self.ld_kv = kv_heads * d * (2 if packed else 1) + pad_kv
        self.v_at = kv_heads * d if packed else 0
        self.packed = packed
        self.scale = np.float32(1.0 / np.sqrt(d))
        self.lens = None if lens is None else np.asarray(lens, np.int32)
        rng = np.random.default_rng(seed)

        def rows(n, ld):
            return (rng.standard_normal((n, ld)) * magnitude).astype(np.float32)

        self.q, self.dout = rows(batch * seq_q, self.ld_q), rows(batch * seq_q, self.ld_out)
        self.k = rows(batch * seq_k, self.ld_kv)
        self.v = self.k if packed else rows(batch * seq_k, self.ld_kv)
        # what lies past the live keys must never be looked at
        for b, n in enumerate(self.live()):
            self.k[b * seq_k + n:(b + 1) * seq_k] = np.nan
            self.v[b * seq_k + n:(b + 1) * seq_k] = np.nan

    def live(self):
        if self.lens is None:
            return [self.sk] * self.batch
        return [int(n) for n in np.clip(self.lens, 0, self.sk)]

    def shape(self):
        return (self.batch, self.heads, self.kv, self.sq, self.sk, self.d, self.ld_q, self.ld_kv,
                self.ld_out)

    def _queries(self, x, b, j):
        """[rows of the group's heads, d] of item b, key head j: query major."""
        x = x[b * self.sq:(b + 1) * self.sq, j * self.group * self.d:(j + 1) * self.group * self.d]
        return x.reshape(self.sq * self.group, self.d)

    def _keys(self, x, b, j, n, at=0):
        return x[b * self.sk:b * self.sk + n, at + j * self.d:at + (j + 1) * self.d]

    def reference(self, gradients=True):
        """out, stats and the gradients, each as (value, bound) arrays of the
        tensors' own layout without the padding columns."""
        hd, kd = self.heads * self.d, self.kv * self.d
        zq, zk = (self.batch * self.sq, hd), (self.batch * self.sk, kd)
        r = {n: (np.zeros(zq), np.zeros(zq)) for n in ("out", "dq")}
        r.update({n: (np.zeros(zk), np.zeros(zk)) for n in ("dk", "dv")})
        stats = np.zeros((self.batch, self.heads, self.sq, 2))
        stats_bound = np.zeros((self.batch, self.heads, self.sq))
        for b, n in enumerate(self.live()):
            for j in range(self.kv):
                q = self._queries(self.q, b, j)
                k, v = self._keys(self.k, b, j, n), self._keys(self.v, b, j, n, self.v_at)
                out, st, bound, _, ep = forward(q, k, v, float(self.scale))
                cols = slice(j * self.group * self.d, (j + 1) * self.group * self.d)
                rows = slice(b * self.sq, (b + 1) * self.sq)
                r["out"][0][rows, cols] = out.reshape(self.sq, self.group * self.d)
                r["out"][1][rows, cols] = bound.reshape(self.sq, self.group * self.d)
                stats[b, j * self.group:(j + 1) * self.group] = st.reshape(
                    self.sq, self.group, 2).transpose(1, 0, 2)
                # of log2 of the sum of exponentials: the scores' error and the
                # sum's, in base 2, both in ep; the maximum is rounded once
                stats_bound[b, j * self.group:(j + 1) * self.group] = (
                    1.45 * ep + 4 * U * np.abs(st[:, :1])).reshape(self.sq, self.group).T
                if not gradients:
                    continue
                g = self._queries(self.dout, b, j)
                (dq, dk, dv), (bq, bk, bv) = backward(q, k, v, g, float(self.scale))
                r["dq"][0][rows, cols], r["dq"][1][rows, cols] = dq.reshape(self.sq, self.group * self.d), bq.reshape(self.sq, self.group * self.d)
                kr, kc = slice(b * self.sk, b * self.sk + n), slice(j * self.d, (j + 1) * self.d)
                r["dk"][0][kr, kc], r["dk"][1][kr, kc] = dk, bk
                r["dv"][0][kr, kc], r["dv"][1][kr, kc] = dv, bv
        r["stats"] = (stats, stats_bound)
        return r
