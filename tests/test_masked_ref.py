"""The reference of masked attention (masked_ref.py) against differences of its own
forward, and against cross attention's where nothing is masked."""
import numpy as np
import pytest

import attention_ref
from masked_ref import Problem


def loss(p, b, h):
    (out, _), _, _, _ = p.one(b, h, gradients=False)
    g = p.dout[b * p.sq:(b + 1) * p.sq, h * p.d:(h + 1) * p.d].astype(np.float64)
    return float((out * g).sum())


@pytest.mark.parametrize("kw", [
    dict(), dict(cap=1.5), dict(slopes=True), dict(causal=False, key_len=[5]),
    dict(prefix_len=[4], cap=2.0, slopes=True), dict(key_begin=[[0, 0, 0, 3, 3, 3, 6]]),
    dict(causal=False, key_begin=[[0, 0, 2, 2, 4, 6, 7]], key_end=[[3, 0, 9, 2, 5, 7, 7]], slopes=True),
], ids=str)
def test_gradients_are_differences(kw):
    p = Problem(1, 2, 1, 7, 7, 4, seed=3, **kw)
    for x in (p.q, p.k, p.v):
        x[:] = np.nan_to_num(x, nan=0.5)
    p.q, p.k, p.v = (x.astype(np.float64) for x in (p.q, p.k, p.v))
    dk, dv = np.zeros((7, 4)), np.zeros((7, 4))
    for h in range(2):
        _, dq, k_part, v_part = p.one(0, h)
        dk += k_part[0]
        dv += v_part[0]
        for i, j in np.ndindex(7, 4):
            at = (i, h * 4 + j)
            assert abs(difference(p, p.q, at, lambda: loss(p, 0, h)) - dq[0][i, j]) < 1e-7
    both = lambda: loss(p, 0, 0) + loss(p, 0, 1)
    for i, j in np.ndindex(7, 4):
        assert abs(difference(p, p.k, (i, j), both) - dk[i, j]) < 1e-7
        assert abs(difference(p, p.v, (i, j), both) - dv[i, j]) < 1e-7


def difference(p, x, at, f, step=1e-5):
    """(f(x + h) - f(x - h)) / 2h: off by h^2 f''' / 6, some 1e-10, and by f's rounding
    over h, some 1e-11."""
    was = x[at]
    x[at] = was + step
    up = f()
    x[at] = was - step
    down = f()
    x[at] = was
    return (up - down) / (2 * step)


def test_unmasked_is_cross_attention():
    p = Problem(2, 4, 2, 5, 9, 8, causal=False, key_len=[9, 4], seed=5)
    c = attention_ref.Problem(2, 4, 2, 5, 9, 8, lens=[9, 4], seed=5)
    for n in ("q", "k", "v", "dout"):
        setattr(c, n, getattr(p, n))
    mine, theirs = p.reference(), c.reference()
    for n in ("out", "dq", "dk", "dv"):
        assert np.allclose(mine[n][0], theirs[n][0], rtol=1e-12, atol=1e-12)


def test_ranges():
    p = Problem(1, 1, 1, 3, 6, 4, q_start=[2], prefix_len=[4], key_begin=[[1, 0, 5]], key_len=[5])
    want = np.array([[0, 1, 1, 1, 0, 0], [1, 1, 1, 1, 0, 0], [0, 0, 0, 0, 0, 0]], bool)
    assert np.array_equal(p.visible(0), want)
