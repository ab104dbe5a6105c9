"""What cross attention, embedding and dropout refuse, before anything
touches a GPU: the checks of arguments come first, so these run anywhere. The
pointers are placeholders that no refused call looks at."""
import os

import pytest

from neuralrs_amd import _abi

P = 4096  # stands for a device pointer


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libnrs_hip.so not built")
    _abi.load()


GOOD = dict(batch=2, heads=4, kv_heads=2, seq_q=3, seq_k=5, d_head=32, ld_q=128, ld_kv=64, ld_out=128)
BAD = [
    (dict(batch=-1), "negative"), (dict(seq_q=-1), "negative"), (dict(seq_k=-2), "negative"),
    (dict(heads=0), "no heads"), (dict(kv_heads=0), "no heads"), (dict(kv_heads=3), "multiple"),
    (dict(d_head=0), "d_head"), (dict(d_head=129, ld_q=1024, ld_kv=1024, ld_out=1024), "d_head"),
    (dict(ld_q=127), "stride"), (dict(ld_kv=63), "stride"), (dict(ld_out=100), "stride"),
    (dict(ld_q=2 ** 20 + 1), "2\\^20"), (dict(ld_kv=2 ** 33), "2\\^20"), (dict(seq_k=2 ** 40), "2\\^26"),
    (dict(seq_q=2 ** 27), "2\\^26"), (dict(batch=2 ** 40), "2\\^26"),
    (dict(batch=2 ** 20, seq_q=2 ** 20), "2\\^26"), (dict(batch=2 ** 12, seq_k=2 ** 16), "2\\^26"),
    (dict(seq_q=2 ** 26, heads=2 ** 14, kv_heads=1, ld_q=2 ** 19, ld_out=2 ** 19), "2\\^26"),
    (dict(heads=2 ** 62, kv_heads=1), "stride"),
    # products of the sizes that 64 bits do not hold
    (dict(batch=2 ** 22, heads=2 ** 15, kv_heads=2 ** 15, seq_q=2 ** 26, seq_k=2 ** 26, ld_q=2 ** 20,
          ld_kv=2 ** 20, ld_out=2 ** 20), "2\\^26"),
    (dict(batch=2 ** 62, heads=1, kv_heads=1), "2\\^26"),
    (dict(batch=2 ** 22, heads=2 ** 15, kv_heads=1, seq_q=2 ** 26, ld_q=2 ** 20, ld_out=2 ** 20), "2\\^26"),
]


@pytest.mark.parametrize("change,why", BAD, ids=lambda x: str(x))
def test_cross_attention_shapes(change, why):
    s = {**GOOD, **change}
    assert _abi.load().nrs_cross_attention_supported(*s.values()) == 0
    with pytest.raises(_abi.NrsError, match=why):
        _abi.cross_attention_forward(P, P, P, P, P, None, *s.values(), 1.0)
    with pytest.raises(_abi.NrsError, match=why):
        _abi.cross_attention_backward(P, P, P, P, P, P, P, P, P, None, *s.values(), 1.0)


def test_cross_attention_supported():
    assert _abi.load().nrs_cross_attention_supported(*GOOD.values()) == 1


@pytest.mark.parametrize("null", [0, 2, 3, 4])
def test_cross_attention_forward_nulls(null):
    args = [P, P, P, P, P, None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.cross_attention_forward(*args, *GOOD.values(), 1.0)


@pytest.mark.parametrize("null", [3, 4, 5, 6, 7, 8])
def test_cross_attention_backward_nulls(null):
    args = [P] * 9 + [None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.cross_attention_backward(*args, *GOOD.values(), 1.0)


@pytest.mark.parametrize("null", [1, 2])
def test_key_and_value_gradients_go_together(null):
    args = [P] * 9 + [None]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="go together"):
        _abi.cross_attention_backward(*args, *GOOD.values(), 1.0)


def test_empty_calls_need_nothing():
    s = {**GOOD, "batch": 0}
    _abi.cross_attention_forward(None, None, None, None, None, None, *s.values(), 1.0)
    _abi.cross_attention_backward(*[None] * 10, *s.values(), 1.0)
    _abi.cross_attention_forward(None, None, None, None, None, None, *{**GOOD, "seq_q": 0}.values(), 1.0)
    _abi.embedding_forward(None, None, None, 0, 5, 4)
    _abi.dropout_forward(None, None, None, 0, 0.5, 1, 1)
    _abi.dropout_backward(None, None, 0, 0.5, 1, 1)


@pytest.mark.parametrize("sizes", [(-1, 5, 4), (3, 0, 4), (3, -5, 4), (3, 5, 0), (3, 5, 2 ** 20 + 1),
                                   (2 ** 30 + 1, 5, 4), (3, 2 ** 31 - 1, 4)])
def test_embedding_sizes(sizes):
    for call in (lambda: _abi.embedding_forward(P, P, P, *sizes),
                 lambda: _abi.embedding_backward(P, P, P, *sizes),
                 lambda: _abi.embedding_workspace(*sizes)):
        with pytest.raises(_abi.NrsError, match="unsupported sizes"):
            call()


@pytest.mark.parametrize("null", [0, 1, 2])
def test_embedding_nulls(null):
    args = [P, P, P]
    args[null] = None
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.embedding_forward(*args, 3, 5, 4)
    with pytest.raises(_abi.NrsError, match="null pointer"):
        _abi.embedding_backward(*args, 3, 5, 4)


@pytest.mark.parametrize("p", [-0.1, 1.0001, float("nan"), float("inf")])
def test_dropout_probability(p):
    with pytest.raises(_abi.NrsError, match="p must be in"):
        _abi.dropout_forward(P, P, None, 8, p, 1, 1)
    with pytest.raises(_abi.NrsError, match="p must be in"):
        _abi.dropout_backward(P, P, 8, p, 1, 1)


def test_dropout_sizes_and_nulls():
    with pytest.raises(_abi.NrsError, match="negative size"):
        _abi.dropout_forward(P, P, None, -1, 0.5, 1, 1)
    with pytest.raises(_abi.NrsError, match="negative size"):
        _abi.dropout_backward(P, P, -4, 0.5, 1, 1)
    for args in ((None, P), (P, None)):
        with pytest.raises(_abi.NrsError, match="null pointer"):
            _abi.dropout_forward(*args, None, 8, 0.5, 1, 1)
        with pytest.raises(_abi.NrsError, match="null pointer"):
            _abi.dropout_backward(*args, 8, 0.5, 1, 1)


def test_workspace_of_a_backward_without_keys_or_rows():
    """The rows' statistics are written even where there is nothing to attend
    to: two floats a row, in whole 16 bytes."""
    assert _abi.cross_attention_workspace(2, 4, 2, 3, 0, 32, backward=True) >= 2 * 4 * 3 * 8
    assert _abi.cross_attention_workspace(2, 4, 2, 0, 5, 32, backward=True) == 0
    assert _abi.cross_attention_workspace(2, 4, 2, 0, 5, 32) == 0
    assert _abi.cross_attention_workspace(0, 4, 2, 3, 5, 32) == 0


def test_a_line_of_key_tiles_past_32_bits_is_not_shared():
    """2049 units of 256 rows with 2^20 tiles of keys each: their places on one
    line would pass 2^31. (257 units of 2^14 tiles are shared, with scratch.)"""
    assert _abi.cross_attention_workspace(1, 1, 1, 256 * 257, 2 ** 20, 64) > 0
    assert _abi.cross_attention_workspace(1, 1, 1, 256 * 2049, 2 ** 26, 64) == 0


@pytest.mark.parametrize("sizes", [(2, 4, 3, 3, 5, 32), (2, 2 ** 62, 1, 3, 5, 128), (2, 4, 2, 3, 5, 0),
                                   (-1, 4, 2, 3, 5, 32), (2 ** 40, 4, 2, 3, 5, 32)])
def test_workspace_refuses_what_the_calls_refuse(sizes):
    for backward in (False, True):
        with pytest.raises(_abi.NrsError):
            _abi.cross_attention_workspace(*sizes, backward=backward)


def test_workspace_queries():
    assert _abi.cross_attention_workspace(2, 4, 2, 3, 5, 32) >= 0
    assert _abi.cross_attention_workspace(2, 4, 2, 3, 5, 32, backward=True) >= 0
    assert _abi.embedding_workspace(100, 50, 8) >= 0


@pytest.mark.parametrize("sizes", [(16, 32, 8, 4100, 2000, 128), (2, 33, 33, 9000, 700, 64),
                                   (3, 40, 40, 5000, 1000, 96), (2, 40, 40, 9000, 3001, 20)])
def test_scratch_of_a_shared_forward_does_not_grow_with_its_rows(sizes):
    """A workgroup leaves the sums of two units at most, the one that its part
    begins in and the one that it ends in: of 256 rows with a workgroup to each
    of 256 compute units, or of 128 with two. A unit has its first and last
    workgroup on record."""
    batch, heads, _, seq_q, _, d = sizes
    units = batch * heads * seq_q // 128 + batch * heads
    need = _abi.cross_attention_workspace(*sizes)
    assert 0 < need <= 2 * 256 * 256 * (d + 2) * 4 + 8 * units
