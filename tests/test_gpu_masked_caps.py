"""Masked attention's caps: far above the scores, far below the operands, and scores
near the cap, whose gradients are small but have all their bits.

The derivative of cap tanh(x / cap) is 1 / cosh(y)^2, y = x / cap, and the bound here
is relative to it, where masked_ref.py's allows two steps of 1. With u = 2^-24: y is
off by e_x / cap and by 2 u of itself (the factor 1 / cap and the product), which
the derivative takes 2 |tanh y| <= 2 times, relative. It is computed as
4 e / (1 + e)^2 from e = e^(-2 |y|): the exponent in base 2 is rounded twice (the
constant, the product), 2 u of 2 |y|, the exponential has 2 u of itself, 1 + e one, the
reciprocal two, squared with it 6, the products 3: (4 |y| + 11) u; and as 1 - t^2 up to
|y| = 0.6, where it is 0.71 and more: t is off by 4 u of itself at most, the rest by a
step each: (8 t^2 + 2) u / 0.71 < 7 u. Together 2 e_x / cap + (8 |y| + 16) u.
"""
import numpy as np
import pytest

from attention_ref import TINY, U, gamma
from masked_ref import Problem
from test_gpu_masked_attention import check, compare, run

pytestmark = pytest.mark.gpu

SIZES = [(3, 300, 64), (16, 700, 128), (150, 150, 32), (150, 150, 64), (150, 150, 80), (150, 150, 128)]


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("cap", [1e10, 1e30, 1e36, 1.6e38])
@pytest.mark.parametrize("sq,sk,d", SIZES, ids=str)
def test_caps_far_above_the_scores(hip, sq, sk, d, cap, slopes):
    check(hip, Problem(1, 2, 1, sq, sk, d, seed=29, cap=cap, slopes=slopes))


@pytest.mark.parametrize("sq,sk,d", SIZES, ids=str)
def test_caps_far_below_the_operands(hip, sq, sk, d):
    """Scores of 10^17 caps: every weight is that of a score of plus or minus a cap."""
    p = Problem(1, 2, 1, sq, sk, d, seed=30, cap=1e-30, key_len=[sk])
    p.scale = np.float32(1.0)
    p.q *= np.float32(1e-25)
    p.k *= np.float32(1e12)
    check(hip, p)


@pytest.mark.parametrize("cap", [2.0 ** -126, 1e-37, 1e-3])
@pytest.mark.parametrize("sq,sk,d", SIZES, ids=str)
def test_the_smallest_caps(hip, sq, sk, d, cap):
    p = Problem(1, 2, 1, sq, sk, d, seed=31, cap=cap)
    p.scale = np.float32(cap)
    check(hip, p)


def gradients(p, h):
    """dq of head h and its part of dk, with their bounds; one item, no bias."""
    d, j = p.d, h // p.group
    cols, kc = slice(h * d, (h + 1) * d), slice(j * d, (j + 1) * d)
    q, g = p.q[:, cols].astype(np.float64), p.dout[:, cols].astype(np.float64)
    k, v = p.k[:, kc].astype(np.float64), p.v[:, kc].astype(np.float64)
    see, scale = p.visible(0), float(p.scale)
    assert see.any(axis=0).all() and see.any(axis=1).all()
    x = q @ k.T * scale
    e_x = gamma(d) * (np.abs(q) @ np.abs(k).T * scale)
    y = x / p.cap
    inner = 1.0 / np.cosh(y) ** 2
    e_inner = inner * (2 * e_x / p.cap + (8 * np.abs(y) + 16) * U)
    u = p.cap * np.tanh(y)
    e_u = e_x * inner + 6 * U * np.abs(u)
    u = np.where(see, u, -np.inf)
    m = u.max(axis=1, keepdims=True)
    e = np.exp(u - m)
    total = e.sum(axis=1, keepdims=True)
    w = e / total
    es = np.where(see, e_u + 4 * U * (np.abs(np.where(see, u, 0.0)) + np.abs(m + np.log(total))), 0.0)
    ew = es + (w * es).sum(axis=1, keepdims=True) + gamma(p.sk) + 8 * U
    out = w @ v
    b_out = (w * (ew + gamma(p.sk))) @ np.abs(v)
    dp, delta = g @ v.T, (g * out).sum(axis=1, keepdims=True)
    diff = np.abs(dp - delta)
    e_diff = gamma(d) * (np.abs(g) @ np.abs(v).T) + (
        gamma(d) * (np.abs(g) * np.abs(out)) + np.abs(g) * b_out).sum(axis=1, keepdims=True)
    ds = w * (dp - delta) * inner * scale
    e_ds = scale * w * (((ew + 4 * U) * diff + e_diff) * inner + diff * e_inner)
    e_ds = np.where(see, e_ds + TINY * (1 + scale * diff), 0.0)
    R = p.sq * p.group
    return ((ds @ k, e_ds @ np.abs(k) + gamma(p.sk) * (np.abs(ds) @ np.abs(k))),
            (ds.T @ q, e_ds.T @ np.abs(q) + gamma(R) * (np.abs(ds).T @ np.abs(q))))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("far", [0.3, 1.0, 6.0, 9.0, 20.0])
@pytest.mark.parametrize("d", [32, 24, 64, 96, 128])
def test_gradients_of_scores_near_the_cap(hip, d, far, causal):
    """Scores of 0.7 to 1.3 times `far` caps, of either sign, each key with its own."""
    p = Problem(1, 2, 1, 150, 150, d, causal=causal, seed=32, cap=1.5)
    rng = np.random.default_rng(d)
    size = far * p.cap / np.sqrt(d) * rng.uniform(0.75, 1.25, 150) * rng.choice([-1.0, 1.0], 150)
    p.q = (1.0 + 0.02 * p.q).astype(np.float32)
    p.k = (size[:, None] * (1.0 + 0.02 * p.k)).astype(np.float32)
    got = run(hip, p)
    dk, b_dk = np.zeros((150, d)), np.zeros((150, d))
    for h in range(2):
        dq, part = gradients(p, h)
        compare(got[1][:, h * d:(h + 1) * d], *dq, f"dq {h}")
        dk += part[0]
        b_dk += part[1]
    compare(got[2], dk, b_dk, "dk")


def test_the_formula_against_differences():
    """The reference's own gradients, where a third of the scores are near the cap."""
    p = Problem(1, 2, 1, 6, 6, 4, seed=33, cap=0.5)
    p.q, p.k, p.v = (x.astype(np.float64) for x in (p.q, p.k, p.v))

    def loss():
        total = 0.0
        for h in range(2):
            (out, _), _, _, _ = p.one(0, h, gradients=False)
            total += float((out * p.dout[:, 4 * h:4 * h + 4].astype(np.float64)).sum())
        return total

    (dq0, dk0), (dq1, dk1) = gradients(p, 0), gradients(p, 1)
    want = {"q": np.concatenate([dq0[0], dq1[0]], axis=1), "k": dk0[0] + dk1[0]}
    for name, grad in want.items():
        x = getattr(p, name)
        for at in np.ndindex(*x.shape):
            was = x[at]
            x[at] = was + 1e-5
            up = loss()
            x[at] = was - 1e-5
            down = loss()
            x[at] = was
            # h^2 f''' / 6 with f''' some (1 / cap)^3, and 1e-16 / h
            assert abs((up - down) / 2e-5 - grad[at]) < 1e-8, (name, at)
