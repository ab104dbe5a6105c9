"""What masked attention, rotary positions and distillation refuse, before anything
touches a GPU: the checks of arguments come first, so these run anywhere. The
pointers are placeholders that no refused call looks at."""
import math
import os

import pytest

from neuralrs_amd import _abi
from test_operator_refusals import BAD, GOOD

P = 4096  # stands for a device pointer


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libnrs_hip.so not built")
    _abi.load()


@pytest.mark.parametrize("change,why", BAD, ids=lambda x: str(x))
def test_masked_attention_shapes(change, why):
    s = {**GOOD, **change}
    m = _abi.attention_mask(causal=True)
    assert _abi.load().nrs_masked_attention_supported(*s.values()) == 0
    with pytest.raises(_abi.NrsError, match=why):
        _abi.masked_attention_forward(P, P, P, P, P, m, *s.values(), 1.0)
    with pytest.raises(_abi.NrsError, match=why):
        _abi.masked_attention_backward(P, P, P, P, P, P, P, P, P, m, *s.values(), 1.0)


def test_masked_attention_supported():
    assert _abi.load().nrs_masked_attention_supported(*GOOD.values()) == 1


@pytest.mark.parametrize("mask,why", [
    (dict(cap=-1.0), "cap"), (dict(cap=math.nan), "cap"), (dict(cap=math.inf), "cap"),
    (dict(prefix_len=P), "prefix"),
], ids=str)
def test_masks(mask, why):
    m = _abi.attention_mask(**mask)
    with pytest.raises(_abi.NrsError, match=why):
        _abi.masked_attention_forward(P, P, P, P, P, m, *GOOD.values(), 1.0)
    with pytest.raises(_abi.NrsError, match=why):
        _abi.masked_attention_backward(*[P] * 9, m, *GOOD.values(), 1.0)


@pytest.mark.parametrize("cap,scale", [(3e38, 1.0), (1e-39, 1.0), (1.0, math.inf), (1.0, math.nan),
                                       (1e-30, 1e10)])
def test_caps_that_floats_do_not_hold(cap, scale):
    m = _abi.attention_mask(cap=cap)
    with pytest.raises(_abi.NrsError, match="cap"):
        _abi.masked_attention_forward(P, P, P, P, P, m, *GOOD.values(), scale)
    with pytest.raises(_abi.NrsError, match="cap"):
        _abi.masked_attention_backward(*[P] * 9, m, *GOOD.values(), scale)


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1.17e-38])
def test_caps_without_a_reciprocal(cap):
    """Below 2^-126, whatever the scale."""
    m = _abi.attention_mask(cap=cap)
    with pytest.raises(_abi.NrsError, match="2\\^-126"):
        _abi.masked_attention_forward(P, P, P, P, P, m, *GOOD.values(), 1e-10)
    with pytest.raises(_abi.NrsError, match="2\\^-126"):
        _abi.masked_attention_backward(*[P] * 9, m, *GOOD.values(), 1e-10)


@pytest.mark.parametrize("null", [0, 2, 3, 4])
def test_masked_attention_forward_nulls(null):
    args = [P, P, P, P, P, None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.masked_attention_forward(*args, *GOOD.values(), 1.0)


@pytest.mark.parametrize("null", [3, 4, 5, 6, 7, 8])
def test_masked_attention_backward_nulls(null):
    args = [P] * 9 + [None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.masked_attention_backward(*args, *GOOD.values(), 1.0)


@pytest.mark.parametrize("null", [1, 2])
def test_key_and_value_gradients_go_together(null):
    args = [P] * 9 + [None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="go together"):
        _abi.masked_attention_backward(*args, *GOOD.values(), 1.0)


def test_empty_calls_need_nothing():
    s = {**GOOD, "batch": 0}
    _abi.masked_attention_forward(*[None] * 6, *s.values(), 1.0)
    _abi.masked_attention_backward(*[None] * 10, *s.values(), 1.0)
    _abi.rotary_forward(*[None] * 5, 0, 4, 32, 16, 1, 128, 128)
    _abi.rotary_backward(*[None] * 5, 0, 4, 32, 16, 1, 128, 128)
    _abi.distill_forward(*[None] * 5, 0, 100, 3, 100)
    _abi.distill_backward(*[None] * 7, 0, 100, 3, 100)


ROTARY = dict(rows=3, heads=2, d_head=16, pairs=8, axes=2, ld_x=32, ld_out=40)
BAD_ROTARY = [
    (dict(rows=-1), "negative"), (dict(heads=0), "no heads"), (dict(d_head=0), "negative"),
    (dict(pairs=-1), "negative"), (dict(axes=0), "axes"), (dict(pairs=9), "half"),
    (dict(ld_x=31), "stride"), (dict(ld_out=31), "stride"), (dict(ld_x=2 ** 20 + 1), "2\\^20"),
    (dict(rows=2 ** 31), "2\\^30"), (dict(axes=2 ** 40), "2\\^30"), (dict(heads=2 ** 62), "stride"),
    (dict(rows=2 ** 30, heads=2 ** 15, ld_x=2 ** 20, ld_out=2 ** 20), "2\\^31"),
    (dict(d_head=2 ** 40, pairs=1), "stride"),
]


@pytest.mark.parametrize("change,why", BAD_ROTARY, ids=lambda x: str(x))
def test_rotary_shapes(change, why):
    s = {**ROTARY, **change}
    with pytest.raises(_abi.NrsError, match=why):
        _abi.rotary_forward(P, 2 * P, P, P, P, *s.values())
    with pytest.raises(_abi.NrsError, match=why):
        _abi.rotary_backward(P, 2 * P, P, P, P, *s.values())


@pytest.mark.parametrize("null", [0, 1, 2, 3])
def test_rotary_nulls(null):
    args = [P, 2 * P, P, P, None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.rotary_forward(*args, *ROTARY.values())
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.rotary_backward(*args, *ROTARY.values())


def test_rotary_in_place():
    with pytest.raises(_abi.NrsError, match="two row strides"):
        _abi.rotary_forward(P, P, P, P, P, *ROTARY.values())
    s = {**ROTARY, "ld_out": 32}
    with pytest.raises(_abi.NrsError, match="beta"):
        _abi.rotary_backward(P, P, P, P, P, *s.values(), beta=1.0)


DISTILL = dict(rows=3, vocab=100, k=4, ld=100)
BAD_DISTILL = [
    (dict(rows=-1), {}, "negative"), (dict(vocab=0), {}, "vocabulary"), (dict(k=-1), {}, "negative"),
    (dict(k=1025), {}, "1024"), (dict(ld=99), {}, "stride"), (dict(rows=2 ** 23), {}, "2\\^23"),
    (dict(vocab=2 ** 31, ld=2 ** 31), {}, "2\\^31"), ({}, dict(temperature=0.0), "temperature"),
    ({}, dict(temperature=-1.0), "temperature"), ({}, dict(temperature=math.nan), "temperature"),
    ({}, dict(temperature=math.inf), "temperature"), ({}, dict(hard=-0.1), "hard"),
    ({}, dict(hard=1.1), "hard"), ({}, dict(hard=math.nan), "hard"),
]


@pytest.mark.parametrize("change,more,why", BAD_DISTILL, ids=lambda x: str(x))
def test_distill_arguments(change, more, why):
    s = {**DISTILL, **change}
    with pytest.raises(_abi.NrsError, match=why):
        _abi.distill_forward(P, P, P, P, P, *s.values(), **more)
    with pytest.raises(_abi.NrsError, match=why):
        _abi.distill_backward(P, P, P, P, P, P, P, *s.values(), **more)


@pytest.mark.parametrize("null", [0, 1, 2, 3])
def test_distill_nulls(null):
    args = [P, P, P, P, P]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.distill_forward(*args, *DISTILL.values())
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.distill_backward(args[0], None, None, *args[1:], *DISTILL.values())


def test_distill_needs_labels():
    with pytest.raises(_abi.NrsError, match="labels"):
        _abi.distill_forward(P, P, P, P, None, *DISTILL.values(), hard=0.5)
