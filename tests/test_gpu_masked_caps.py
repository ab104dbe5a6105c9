"""Masked attention's caps far above the scores and far below the operands. The bounds are
those of masked_ref.py, whose derivation stands there."""
import numpy as np
import pytest

from masked_ref import Problem
from test_gpu_masked_attention import check

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
