"""nrs_distill_forward / _backward against the definition in 64 bits.

Tolerances, u = 2^-24. An exponent (z - m) log2 e / T is rounded twice and its
exponential has 2 u: e(z) = (3 |z - m| / T + 4) u relative; a sum of n has (n + 8) u at
most and the average of its terms' (gamma). log p and log q have the size of their
terms, |z - m| / T + log n, to a few u each. So a token's part p (log p - log q) is off
by p times (8 (|d_p| + |d_q| + log k + log n) + 4 gamma) u, and by the error of p,
relative, times |log p - log q|. The gradient's parts are products of those.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def softmax(z, axis=1):
    m = z.max(axis=axis, keepdims=True)
    e = np.exp(z - m)
    return e / e.sum(axis=axis, keepdims=True)


def reference(logits, vocab, top, ids, labels, temp, hard, row_grad):
    """loss, its bound, gradient, its bound; rows one by one."""
    rows = logits.shape[0]
    loss, e_loss = np.zeros(rows), np.zeros(rows)
    grad, e_grad = np.zeros((rows, vocab)), np.zeros((rows, vocab))
    temp, hard = float(np.float32(temp)), float(np.float32(hard))
    for r in range(rows):
        z = logits[r, :vocab].astype(np.float64)
        w = float(row_grad[r]) if row_grad is not None else 1.0 / rows
        parts = []
        live = (ids[r] >= 0) & (ids[r] < vocab) if top is not None else np.zeros(0, bool)
        if hard < 1.0 and live.any() and top[r][live].max() > -np.inf:
            t = top[r][live].astype(np.float64) / temp
            id_ = ids[r][live]
            p = softmax(t[None])[0]
            dist = z / temp - (z / temp).max()
            total = np.exp(dist).sum()
            logq = dist - np.log(total)
            q = np.exp(logq)
            logp = np.where(p > 0, t - t.max() - np.log(np.exp(t - t.max()).sum()), 0.0)
            on = p > 0
            loss[r] += (1 - hard) * temp ** 2 * (p[on] * (logp[on] - logq[id_][on])).sum()
            target = np.zeros(vocab)
            np.add.at(target, id_, p)
            grad[r] += w * (1 - hard) * temp * (q - target)
            far_p = np.where(on, t.max() - t, 0.0)
            far_q = np.where(np.isfinite(dist), -dist, 0.0)
            e_p = p * (3 * far_p + (p * 3 * far_p).sum() + len(p) + 16) * U
            n_sum = vocab / 64 + 64  # no sum is one chain: 64 partial ones at least
            e_q = q * (3 * far_q + (q * 3 * far_q).sum() + n_sum + 16) * U
            size = far_p[on] + far_q[id_][on] + np.log(len(p)) + np.log(total) + 4
            e_loss[r] += (1 - hard) * temp ** 2 * (
                (p[on] * (8 * size + (p * 3 * far_p).sum() + (q * 3 * far_q).sum() + n_sum + len(p)) * U).sum()
                + (e_p[on] * np.abs(logp[on] - logq[id_][on])).sum()
                + len(p) * U * (p[on] * np.abs(logp[on] - logq[id_][on])).sum())
            e_t = np.zeros(vocab)
            np.add.at(e_t, id_, e_p + 4 * U * p)
            e_grad[r] += abs(w) * (1 - hard) * temp * (e_q + e_t + 8 * U * (q + target))
        if hard > 0.0 and 0 <= labels[r] < vocab:
            dist = z - z.max()
            total = np.exp(dist).sum()
            far = np.where(np.isfinite(dist), -dist, 0.0)
            one = np.exp(dist) / total
            loss[r] -= hard * (dist[labels[r]] - np.log(total))
            n_sum = vocab / 64 + 64
            e_loss[r] += hard * (8 * (far[labels[r]] + np.log(total) + 4) + (one * 3 * far).sum() + n_sum) * U
            g = one.copy()
            g[labels[r]] -= 1.0
            grad[r] += w * hard * g
            e_grad[r] += abs(w) * hard * (one * (3 * far + (one * 3 * far).sum() + n_sum + 24) * U)
            e_grad[r][labels[r]] += abs(w) * hard * 8 * U
    return loss, e_loss + 4 * U * np.abs(loss), grad, e_grad + 2.0 ** -126


def make(rows, vocab, k, seed, pad=0, scale=2.0, labels=True, ragged=True):
    rng = np.random.default_rng(seed)
    logits = (scale * rng.standard_normal((rows, vocab + pad))).astype(np.float32)
    ids = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)]).astype(np.int32).reshape(rows, k)
    top = (scale * rng.standard_normal((rows, k)) + 3).astype(np.float32)
    if ragged and k > 1:
        ids[:, k // 2:][rng.random((rows, k - k // 2)) < 0.4] = -1
    lab = rng.integers(-1, vocab, rows).astype(np.int32) if labels else None
    return logits, top, ids, lab


def check(hip, logits, vocab, top, ids, labels, temp, hard, row_grad=None, in_place=False):
    rows, ld = logits.shape
    k = top.shape[1] if top is not None else 0
    print(f"distill rows {rows} vocab {vocab} k {k} ld {ld} T {temp} hard {hard}", flush=True)
    loss, e_loss, grad, e_grad = reference(logits, vocab, top, ids, labels, temp, hard, row_grad)
    up = hip.DeviceBuffer.from_host
    z = up(logits)
    t, i = (up(top), up(ids, np.int32)) if k else (None, None)
    lab = None if labels is None else up(labels, np.int32)
    w = None if row_grad is None else up(row_grad)
    got = up(np.full(rows + 1, 7.0))
    args = (t, i, lab, rows, vocab, k, ld)
    hip.distill_forward(got, z, *args, temperature=temp, hard=hard)
    first = got.to_host()
    assert first[rows] == 7.0
    bad = ~(np.abs(first[:rows] - loss) <= e_loss)
    assert not bad.any(), (first[:rows][bad], loss[bad], e_loss[bad])
    mark = np.full((rows, ld), 7.0, np.float32)
    g = z if in_place else up(mark)
    got = up(np.full(rows + 1, 7.0))
    hip.distill_backward(g, got, w, z, *args, temperature=temp, hard=hard)
    assert np.array_equal(got.to_host(), first)
    out = g.to_host((rows, ld))
    assert np.array_equal(out[:, vocab:], (logits if in_place else mark)[:, vocab:])
    bad = ~(np.abs(out[:, :vocab] - grad) <= e_grad)
    at = tuple(np.argwhere(bad)[0]) if bad.any() else None
    assert not bad.any(), (bad.sum(), at, out[at], grad[at], e_grad[at])
    return out


CASES = [
    # rows, vocab, k
    (1, 1, 1), (2, 2, 1), (3, 5, 5), (7, 64, 8), (5, 1000, 16), (4, 2047, 3), (3, 2048, 33),
    (2, 2049, 256), (9, 8000, 64), (2, 30001, 1000), (1, 70000, 1024), (300, 257, 20), (1, 160000, 7),
    (3, 40003, 100), (2, 131075, 12), (2, 1500, 1024), (70, 33000, 5), (1, 8193, 1),
]


@pytest.mark.parametrize("temp,hard", [(1.0, 0.0), (2.0, 0.0), (1.0, 0.3), (3.0, 0.5), (0.5, 1.0)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_sizes(hip, case, temp, hard):
    logits, top, ids, labels = make(*case, seed=sum(case))
    check(hip, logits, case[1], top, ids, labels, temp, hard)


@pytest.mark.parametrize("pad", [1, 2, 3, 4, 61])
def test_strides_weights_and_in_place(hip, pad):
    logits, top, ids, labels = make(13, 1013, 9, seed=pad, pad=pad)
    w = np.random.default_rng(2).standard_normal(13).astype(np.float32)
    w[3] = 0.0
    one = check(hip, logits, 1013, top, ids, labels, 2.0, 0.25, row_grad=w)
    two = check(hip, logits, 1013, top, ids, labels, 2.0, 0.25, row_grad=w, in_place=True)
    assert np.array_equal(one[:, :1013], two[:, :1013])


def test_in_place_of_a_wide_row(hip):
    logits, top, ids, labels = make(3, 150001, 50, seed=8)
    one = check(hip, logits, 150001, top, ids, labels, 2.0, 0.25)
    assert np.array_equal(one, check(hip, logits, 150001, top, ids, labels, 2.0, 0.25, in_place=True))


def test_no_teacher_is_cross_entropy(hip):
    logits, _, _, labels = make(20, 333, 1, seed=5)
    labels[4] = 333
    labels[5] = 2 ** 31 - 1
    check(hip, logits, 333, None, None, labels, 1.0, 1.0)
    check(hip, logits, 333, None, None, labels, 1.0, 0.5)


def test_repeated_tokens_share(hip):
    """The same token at several places, every place the same token, the label among them."""
    logits, top, ids, labels = make(40, 50, 16, seed=6)
    rng = np.random.default_rng(3)
    ids[:20] = rng.integers(-1, 5, (20, 16))
    ids[20] = 17
    labels[20] = 17
    labels[:10] = ids[:10, 0]
    check(hip, logits, 50, top, ids, labels, 2.0, 0.4)
    check(hip, logits, 50, top, ids, labels, 1.0, 0.4)


def test_many_repeated_tokens(hip):
    logits, top, ids, labels = make(3, 5000, 1024, seed=16)
    ids[0] = np.arange(1024) % 300
    ids[1] = ids[1][::-1] % 7
    ids[2, 1023] = ids[2, 0] = 4999
    check(hip, logits, 5000, top, ids, labels, 2.0, 0.4)


def test_rows_without_a_teacher(hip):
    logits, top, ids, labels = make(6, 100, 4, seed=7)
    ids[0] = -1
    ids[1] = [100, -7, 2 ** 31 - 1, -2 ** 31]
    top[2] = -np.inf
    top[3, :3] = -np.inf
    top[4, 0] = -np.inf
    labels[:] = [3, -1, -1, 5, 6, 7]
    out = check(hip, logits, 100, top, ids, labels, 2.0, 0.5)
    assert np.all(out[1] == 0) and np.all(out[2] == 0)


def test_masked_logits(hip):
    """Logits of minus infinity: no probability, no gradient but the teacher's."""
    logits, top, ids, labels = make(8, 3000, 6, seed=9, ragged=False)
    rng = np.random.default_rng(4)
    dead = rng.random((8, 3000)) < 0.7
    for r in range(8):
        dead[r, ids[r]] = False
        dead[r, max(labels[r], 0)] = False
    logits[dead] = -np.inf
    out = check(hip, logits, 3000, top, ids, labels, 2.0, 0.3)
    assert np.all(out[dead] == 0)
    # all but a token, at any place
    for keep in (0, 1, 2047, 2999):
        logits[0] = -np.inf
        logits[0, keep] = 5.0
        ids[0] = [keep, -1, -1, -1, -1, -1]
        labels[0] = keep
        check(hip, logits, 3000, top, ids, labels, 1.0, 0.3)


def test_a_dead_token_of_the_teacher_costs_everything(hip):
    logits, top, ids, _ = make(2, 64, 3, seed=10, ragged=False)
    logits[0, ids[0, 1]] = -np.inf
    up = hip.DeviceBuffer.from_host
    loss, grad = hip.DeviceBuffer(2), hip.DeviceBuffer(128)
    hip.distill_backward(grad, loss, None, up(logits), up(top), up(ids, np.int32), None, 2, 64, 3, 64)
    assert loss.to_host()[0] == np.inf and np.isfinite(loss.to_host()[1])
    assert np.isfinite(grad.to_host()).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=str)
@pytest.mark.parametrize("at", [0, 500, 2999])
def test_a_bad_row_stays_alone(hip, bad, at):
    logits, top, ids, _ = make(3, 3000, 6, seed=11, ragged=False)
    logits[1, at] = bad
    up = hip.DeviceBuffer.from_host
    loss, grad = hip.DeviceBuffer(3), hip.DeviceBuffer(9000)
    hip.distill_backward(grad, loss, None, up(logits), up(top), up(ids, np.int32), None, 3, 3000, 6, 3000)
    assert np.isnan(loss.to_host()[1]) and np.isfinite(loss.to_host()[[0, 2]]).all()
    g = grad.to_host((3, 3000))
    assert np.isnan(g[1]).any() and np.isfinite(g[[0, 2]]).all()


@pytest.mark.parametrize("scale", [1e-20, 50.0, 1e4])
def test_small_and_large_logits(hip, scale):
    logits, top, ids, labels = make(5, 700, 8, seed=12, scale=scale)
    check(hip, logits, 700, top, ids, labels, 1.0, 0.0)


def test_gradient_is_the_difference_of_losses(hip):
    """Central differences of the device's own loss. An f32 loss of about 10 rounds to
    1e-6, over 2 h = 0.125 that is 1e-5 of noise; h^2 f''' / 6 < 0.0625^2 / 6 of the
    probabilities involved, 7e-4 of them: 2e-3 covers both."""
    logits, top, ids, labels = make(4, 24, 5, seed=13, scale=1.0)
    labels[:] = [0, 3, 23, -1]
    up = hip.DeviceBuffer.from_host
    t, i, lab = up(top), up(ids, np.int32), up(labels, np.int32)

    def losses(z):
        out = hip.DeviceBuffer(4)
        hip.distill_forward(out, up(z), t, i, lab, 4, 24, 5, 24, temperature=2.0, hard=0.4)
        return out.to_host().astype(np.float64)

    grad = hip.DeviceBuffer(96)
    ones = up(np.ones(4))
    hip.distill_backward(grad, None, ones, up(logits), t, i, lab, 4, 24, 5, 24, temperature=2.0, hard=0.4)
    g = grad.to_host((4, 24))
    for v in range(24):
        step = np.zeros_like(logits)
        step[:, v] = 0.0625
        diff = (losses(logits + step) - losses(logits - step)) / 0.125
        assert np.all(np.abs(diff - g[:, v]) < 2e-3)


def test_the_same_call_has_the_same_bits(hip):
    logits, top, ids, labels = make(50, 9001, 64, seed=14)
    a = check(hip, logits, 9001, top, ids, labels, 2.0, 0.3)
    b = check(hip, logits, 9001, top, ids, labels, 2.0, 0.3)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("rows,vocab", [(4, 1003), (300, 35), (3, 140001)])
def test_rows_that_learn_from_nothing(hip, rows, vocab, bad):
    """Padding: no teacher token and no label, and anything in the logits, none finite
    among it."""
    logits, top, ids, labels = make(rows, vocab, 5, seed=13)
    ids[1], labels[1] = -1, -1
    top[2], labels[2] = -np.inf, vocab
    logits[1:3] = bad
    up = hip.DeviceBuffer.from_host
    for grad in (hip.DeviceBuffer(rows * vocab), None):
        z, loss = up(logits), hip.DeviceBuffer(rows)
        into = grad or z
        hip.distill_backward(into, loss, None, z, up(top), up(ids, np.int32), up(labels, np.int32),
                             rows, vocab, 5, vocab, temperature=2.0, hard=0.5)
        got = into.to_host((rows, vocab))
        assert np.all(loss.to_host()[1:3] == 0) and np.all(got[1:3] == 0)
        assert np.isfinite(loss.to_host()).all() and np.isfinite(got).all()
        assert np.any(got[0] != 0)


@pytest.mark.parametrize("hard", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("rows,vocab,k", [(6, 500, 7), (6, 9001, 300), (300, 2100, 2), (6, 40001, 5)])
def test_a_teacher_that_is_not_a_number(hip, rows, vocab, k, hard):
    """NaN in a teacher's logits, in all of them too, comes out in the row's loss and in
    its tokens' gradients, wherever the teacher has a weight; a NaN beside an id that is
    left out is left out with it."""
    logits, top, ids, labels = make(rows, vocab, k, seed=17, ragged=False)
    labels[:5] = [3, -1, -1, 5, vocab]
    ids[3, k // 2:] = -1
    up = hip.DeviceBuffer.from_host

    def run():
        loss, grad = hip.DeviceBuffer(rows), hip.DeviceBuffer(rows * vocab)
        args = (up(logits), up(top), up(ids, np.int32), up(labels, np.int32), rows, vocab, k, vocab)
        hip.distill_backward(grad, loss, None, *args, temperature=2.0, hard=hard)
        alone = hip.DeviceBuffer(rows)
        hip.distill_forward(alone, *args, temperature=2.0, hard=hard)
        assert np.array_equal(alone.to_host(), loss.to_host(), equal_nan=True)
        return loss.to_host(), grad.to_host((rows, vocab))

    was_loss, was = run()
    assert np.isfinite(was_loss).all() and np.isfinite(was).all()
    top[1] = np.nan
    top[2, k // 2] = np.nan
    top[3, k // 2:] = np.nan
    top[4], top[4, k - 1] = -np.inf, np.nan
    loss, grad = run()
    bad = [1, 2, 4] if hard < 1.0 else []
    assert np.isnan(loss[bad]).all()
    other = np.ones((rows, vocab), bool)
    for r in bad:
        assert np.isnan(grad[r, ids[r]]).all()
        other[r, ids[r]] = False
    assert np.array_equal(grad[other], was[other])
    rest = np.setdiff1d(np.arange(rows), bad)
    assert np.array_equal(loss[rest], was_loss[rest])
