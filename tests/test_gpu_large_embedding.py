"""Embedding and dropout on tensors past 2^31 floats, and past 2^32 bytes in a row's
offset, with numbers whose sums never round."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def integers(gen, *shape):
    return torch.empty(*shape, device="cuda").random_(-8, 9, generator=gen)


@pytest.mark.parametrize("count", [5, 256, 4097, (1 << 21) + 5])
def test_embedding(hip, count):
    """A table of more than 2^31 floats; the last count, as many positions."""
    vocab, dim = (1 << 21) + 5, 1030
    print(f"embedding {count} of {vocab} x {dim}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(count)
    table = integers(gen, vocab, dim)
    ids = torch.randint(-1, vocab, (count,), generator=gen, device="cuda", dtype=torch.int32)
    ids[-3:] = vocab - 1  # (places that only 64-bit offsets reach)
    ids[0] = vocab - 2
    if count > 4000:
        ids[1000:2000] = vocab - 3
    out = torch.full((count, dim), float("nan"), device="cuda")
    hip.embedding_forward(out, table, ids, count, vocab, dim, 2.0)
    part = 1 << 18
    for i in range(0, count, part):
        some = ids[i:i + part].long()
        want = torch.where((some >= 0)[:, None], 2.0 * table[some.clamp(min=0)], 0.0)
        assert torch.equal(out[i:i + part], want)
    del table
    grad = integers(gen, count, dim)
    dtable = torch.full((vocab, dim), float("nan"), device="cuda")
    hip.embedding_backward(dtable, grad, ids, count, vocab, dim, 2.0)
    live = ids >= 0
    want = torch.zeros(vocab, dim, device="cuda").index_add_(0, ids[live].long(), grad[live])
    assert torch.equal(dtable, 2.0 * want)
    hip.embedding_backward(dtable, grad, ids, count, vocab, dim, 4.0, 1.0)
    assert torch.equal(dtable, 6.0 * want)
    del out, grad, dtable, want
    torch.cuda.empty_cache()


@pytest.mark.parametrize("count,vocab,dim", [(5, (1 << 31) - 2, 1), (300, (1 << 31) - 2, 1),
                                             (400, 3, 1 << 20), (100, 2, 1 << 20)])
def test_the_largest_table_and_the_widest_rows(hip, count, vocab, dim):
    print(f"embedding {count} of {vocab} x {dim}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(count)
    ids = torch.randint(0, vocab, (count,), generator=gen, device="cuda", dtype=torch.int32)
    ids[-2:] = vocab - 1
    ids[0] = -1
    grad, table = integers(gen, count, dim), torch.full((vocab, dim), 3.0, device="cuda")
    out, dtable = torch.empty_like(grad), torch.empty_like(table)
    hip.embedding_forward(out, table, ids, count, vocab, dim, 0.5)
    assert torch.all(out[1:] == 1.5) and torch.all(out[0] == 0.0)
    live = ids >= 0
    for beta in (0.0, 0.5):
        dtable.fill_(2.0)
        hip.embedding_backward(dtable, grad, ids, count, vocab, dim, 1.0, beta)
        want = torch.full_like(table, 2.0 * beta).index_add_(0, ids[live].long(), grad[live])
        assert torch.equal(dtable, want)
        del want
    del out, dtable, table, grad
    torch.cuda.empty_cache()
    hip.call("nrs_shutdown")  # (gives the scratch back)


def test_dropout_backward(hip):
    """The backward's mask is the forward's past 2^31 elements, and adds to what is
    there."""
    n = (1 << 31) + 41
    print(f"dropout {n}", flush=True)
    ones = torch.ones(n, device="cuda")
    out = torch.empty(n, device="cuda")
    hip.dropout_forward(out, ones, ones, n, 0.5, 3, 4)
    hip.dropout_backward(ones, ones, n, 0.5, 3, 4, beta=1.0)
    assert torch.equal(out, ones)
    kept = out[-(1 << 20):] == 3.0
    assert torch.all(kept | (out[-(1 << 20):] == 1.0)) and 0.49 < kept.double().mean().item() < 0.51
    del ones, out
    torch.cuda.empty_cache()
