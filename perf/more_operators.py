"""The operators of decoder models as measurable cases.

Attention under masks (causal, prefix, documents, padding) with a bias by
distance and scores capped by a tanh; rotary positions of one or several axes;
the loss against a teacher's top logits with its gradient. With ``own`` false
``run`` computes them in elementary torch operations; with ``own`` true it
calls the entry points of ``include/nrs_hip.h`` through ``neuralrs_amd._abi``
on the same tensors, with output buffers that the program keeps from call to
call. f32 is the library's only type; ids, positions and lengths are int32.

A training case of attention is the forward and the backward (beta 0, as into
gradients that were just zeroed); one of rotary positions turns the projected
queries and keys and turns their gradients back; one of the loss is the call
that gives each row's loss and the gradient of the logits.
"""
import math

import torch

own = False


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # Self-attention of a decoder in training at the block size that the repository
        # measures (batch 32, 8 heads of 32), sentences padded to one length.
        _attn("attn_train_32x128h8x32", "train", 32, 8, 8, 128, 128, 32, ragged=True),
        # Training on documents packed into rows of odd length, heads of 64: a token sees
        # its own document up to itself. A bias by distance in place of positions.
        _attn("attn_train_4x1021h16x64_docs", "train", 4, 16, 16, 1021, 1021, 64, docs=True,
              slopes=True),
        # The largest training call: long rows, four query heads to a key head, capped
        # scores, a prefix that all tokens see (a prompt, or an image's tokens).
        _attn("attn_train_2x4000h16g4x128_prefix_cap", "train", 2, 16, 4, 4000, 4000, 128,
              prefix=True, cap=50.0),
        # A long prompt when serving: forward alone, causal.
        _attn("attn_prompt_1x8192h32g8x128", "prompt", 1, 32, 8, 8192, 8192, 128),
        # One new token for each of 32 requests over caches of mixed fill.
        _attn("attn_token_32x1500h8x64", "token", 32, 8, 8, 1, 1500, 64, ragged=True,
              slopes=True),
        # One new token of four requests over long caches, capped scores.
        _attn("attn_token_4x16384h32g8x128_cap", "token", 4, 32, 8, 1, 16384, 128, ragged=True,
              cap=30.0),
        # The smallest calls: the positions of one decoding step (queries and keys of 8
        # heads of 32 side by side).
        _rope("rope_step_32h16x32", False, 32, 16, 32, 16, 1),
        # A training batch of the block size: forward and backward, pairs of neighbours.
        _rope("rope_train_4096h16x32", True, 4096, 16, 32, 16, 1, interleaved=True),
        # Video tokens at far positions (time, height, width; the last quarter of each head
        # is not turned), training.
        _rope("rope_train_16001h20x128_3d", True, 16001, 20, 128, 48, 3),
        # Evaluation on a small batch: few rows of a small vocabulary.
        _distill("distill_eval_32x8000k16", False, 32, 8000, 16, 2.0, 0.0),
        # A training batch at the block size (4096 tokens) with hard labels mixed in, some
        # of them padding, and weights of the tokens.
        _distill("distill_train_4096x32000k64", True, 4096, 32000, 64, 2.0, 0.5, weights=True),
        # Rows of a large odd vocabulary, teacher and student at temperature 1.
        _distill("distill_train_1021x128003k100", True, 1021, 128003, 100, 1.0, 0.0),
    ]


def _attn(name, use, batch, heads, kv, sq, sk, d, ragged=False, docs=False, prefix=False,
          slopes=False, cap=0.0, packed=True):
    return {"name": name, "kind": "attn", "use": use, "batch": batch, "heads": heads,
            "kv_heads": kv, "seq_q": sq, "seq_k": sk, "d_head": d, "ragged": ragged,
            "docs": docs, "prefix": prefix, "slopes": slopes, "cap": cap, "packed": packed}


def _rope(name, train, rows, heads, d, pairs, axes, interleaved=False):
    return {"name": name, "kind": "rope", "train": train, "rows": rows, "heads": heads,
            "d_head": d, "pairs": pairs, "axes": axes, "interleaved": interleaved}


def _distill(name, train, rows, vocab, k, temperature, hard, weights=False):
    return {"name": name, "kind": "distill", "train": train, "rows": rows, "vocab": vocab,
            "k": k, "temperature": temperature, "hard": hard, "weights": weights}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rope", "distill", "distill"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "attn":
            use = rng.choice(["train", "train", "prompt", "token"])
            kv = rng.choice([1, 2, 3, 4, 8, 16])
            group = rng.choice([1, 1, 1, 2, 4, 7])
            sk = _log_int(rng, 1, 16384)
            # a prompt may continue a cache; a few tokens at once are checked drafts
            sq = {"train": sk, "token": rng.choice([1, 1, 1, 4]),
                  "prompt": rng.choice([sk, _log_int(rng, 1, sk)])}[use]
            sk = max(sk, sq)
            docs = rng.random() < 0.3
            case = _attn("", use, _log_int(rng, 1, 64), kv * group, kv, sq, sk,
                         rng.choice([16, 32, 64, 128, 24, 40, 80, 96, rng.randint(8, 128)]),
                         ragged=rng.random() < 0.5, docs=docs,
                         prefix=not docs and use != "token" and rng.random() < 0.3,
                         slopes=rng.random() < 0.4, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                         packed=rng.random() < 0.5)
        elif kind == "rope":
            d = rng.choice([16, 32, 64, 128, 80, 96, 2 * rng.randint(4, 64)])
            case = _rope("", rng.random() < 0.6, _log_int(rng, 1, 40000), rng.randint(1, 48), d,
                         rng.choice([d // 2, d // 2, rng.randint(1, d // 2)]), rng.randint(1, 3),
                         rng.random() < 0.4)
        else:
            vocab = _log_int(rng, 100, 160000)
            case = _distill("", rng.random() < 0.7, _log_int(rng, 1, 8192), vocab,
                            min(vocab, _log_int(rng, 1, 256)), rng.choice([1.0, 1.5, 2.0, 4.0]),
                            rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.4)
        if _cost(case) <= most:
            del case["name"]
            return case


def _lengths(case):
    """The live keys of each item, before their order is drawn: from all of
    them down to a seventh (but no fewer than the queries when serving)."""
    b, n = case["batch"], case["seq_k"]
    if not case["ragged"]:
        return [n] * b
    least = 1 if case["use"] == "train" else case["seq_q"]
    return [max(least, n - (i * (n - n // 7)) // b) for i in range(b)]


def _doc_length(case):
    """Documents' average length: a dozen to a row, 16 tokens at least."""
    return max(16, case["seq_k"] // 12)


def _visible(case):
    """Pairs of a query and a key that it sees, of all items and one head."""
    sq, total = case["seq_q"], 0
    for n in _lengths(case):
        start = 0 if case["use"] == "train" else n - sq
        # query i sees min(n, start + i + 1) keys
        whole = max(0, min(sq, start + sq - n))  # those that see all n
        part = sq - whole
        pairs = whole * n + part * (start + 1) + part * (part - 1) // 2
        if case["docs"]:
            pairs = min(pairs, sq * (_doc_length(case) + 1) // 2)
        if case["prefix"]:
            pre = min(n, case["seq_k"] // 4)
            rows = max(0, pre - start)
            pairs += rows * (rows - 1) // 2
        total += pairs
    return total


def work(case):
    if case["kind"] == "attn":
        h, kv, d = case["heads"], case["kv_heads"], case["d_head"]
        rows, pairs = case["batch"] * case["seq_q"] * h, _visible(case) * h
        live = sum(_lengths(case))
        q, kvb, stats = 4 * rows * d, 4 * live * kv * d, 8 * rows
        if case["use"] == "token" and case["docs"]:
            kvb = min(kvb, 4 * case["batch"] * (_doc_length(case) // 2 + case["seq_q"]) * kv * d)
        if case["use"] != "train":
            return {"bytes": 2 * q + 2 * kvb, "flops": 4 * pairs * d}
        # forward: q, k, v in, out and statistics out; backward: those and
        # dout in, dq, dk, dv out (dk, dv for every row of k and v)
        all_kv = 4 * case["batch"] * case["seq_k"] * kv * d
        return {"bytes": 6 * q + 4 * kvb + 2 * stats + 2 * all_kv, "flops": 14 * pairs * d}
    if case["kind"] == "rope":
        n = case["rows"] * case["heads"] * case["d_head"]
        turned = case["rows"] * case["heads"] * case["pairs"]
        times = 2 if case["train"] else 1
        return {"bytes": times * (8 * n + 4 * case["rows"] * case["axes"]),
                "flops": times * 6 * turned}
    n, k = case["rows"] * case["vocab"], case["rows"] * case["k"]
    return {"bytes": 4 * n * (2 if case["train"] else 1) + 8 * k + 8 * case["rows"],
            "flops": (5 if case["train"] else 3) * n}


def _cost(case):
    """Work and memory of the plain form, in one figure."""
    w = work(case)
    if case["kind"] == "attn":
        pairs = case["batch"] * case["seq_q"] * case["seq_k"] * case["heads"]
        return w["flops"] / 1e14 + (w["bytes"] + 30 * pairs) / 4e12
    return w["bytes"]


# ------------------------------------------------------------------ the inputs
def _inputs(case, seed, device):
    g = torch.Generator(device=device).manual_seed(1000003 * seed + 29)
    host = torch.Generator().manual_seed(seed + 5)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    if case["kind"] == "attn":
        b, sq, sk, h = case["batch"], case["seq_q"], case["seq_k"], case["heads"]
        d = case["d_head"]
        dkv = case["kv_heads"] * d
        x = {"q": normal(b * sq, h * d), "kv": normal(b * sk, 2 * dkv)}
        if not case["packed"]:
            x["k"], x["v"] = x["kv"][:, :dkv].contiguous(), x["kv"][:, dkv:].contiguous()
            del x["kv"]
        if case["use"] == "train":
            x["dout"] = normal(b * sq, h * d)
        lens = [_lengths(case)[i] for i in torch.randperm(b, generator=host).tolist()]
        x["lens"] = ints(lens) if case["ragged"] else None
        x["start"] = None  # where an item's first query stands among its keys
        if case["use"] != "train":
            x["start"] = ints([n - sq for n in lens])
        x["prefix"] = None
        if case["prefix"]:
            most = max(1, sk // 4)
            x["prefix"] = torch.randint(0, most + 1, (b,), generator=host).int().to(device)
        x["begin"] = None  # the first token of each query's document
        if case["docs"]:
            # a token in a dozen (of a row) begins a document
            first = torch.rand(b, sk, generator=g, device=device) < 1.0 / _doc_length(case)
            first[:, 0] = True
            at = torch.arange(sk, device=device)[None, :].expand(b, sk)
            begin = torch.where(first, at, 0).cummax(dim=1).values
            if x["start"] is not None:
                begin = begin.gather(1, x["start"].long()[:, None]
                                     + torch.arange(sq, device=device)[None, :])
            x["begin"] = begin.reshape(-1).int()
        x["slopes"] = None
        if case["slopes"]:  # halved from head to head, over eight halvings in all
            x["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=device) / h)
        return x
    if case["kind"] == "rope":
        rows, axes, pairs = case["rows"], case["axes"], case["pairs"]
        n = case["heads"] * case["d_head"]
        x = {"x": normal(rows, n)}
        if case["train"]:
            x["dout"] = normal(rows, n)
        if axes == 1:  # tokens of sequences that go far
            pos = torch.randint(0, 131072, (1, rows), generator=g, device=device)
        else:  # far frames of an image of up to 64 x 64 patches
            far = [131072, 64, 64][:axes]
            pos = torch.stack([torch.randint(0, f, (rows,), generator=g, device=device)
                               for f in far])
        x["positions"] = pos.int().contiguous()
        x["freq"] = torch.exp2(-torch.arange(pairs, device=device, dtype=torch.float64)
                               * (math.log2(10000.0) / pairs)).float()
        # the axes' pairs one after the other, in equal parts
        x["axis"] = (torch.arange(pairs, device=device) * axes // pairs).int()
        return x
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    logits = 2.0 * normal(rows, vocab)
    # a teacher that agrees with the student in part; it is sure of fewer tokens
    # in some rows (places of no token have the id -1)
    teacher = torch.add(logits, normal(rows, vocab), alpha=1.5)
    top, ids = torch.topk(teacher, k, dim=1)
    del teacher
    count = torch.randint(max(1, k // 2), k + 1, (rows, 1), generator=g, device=device)
    ids = torch.where(torch.arange(k, device=device)[None, :] < count, ids, -1).int()
    x = {"logits": logits, "top": top.contiguous(), "ids": ids.contiguous(), "labels": None,
         "row_grad": None}
    if case["hard"] > 0.0:
        labels = torch.randint(0, vocab, (rows,), generator=g, device=device)
        pad = torch.rand(rows, generator=g, device=device) < 0.05
        x["labels"] = torch.where(pad, -1, labels).int()
    if case["weights"]:
        x["row_grad"] = torch.rand(rows, generator=g, device=device) / rows
    return x


def prepare(case, seed):
    device = torch.device("cuda", 0)
    x = _inputs(case, seed, device)
    s = dict(case)
    s["x"] = x
    if case["kind"] == "attn":
        dkv = case["kv_heads"] * case["d_head"]
        if case["packed"]:
            x["k"], x["v"] = x["kv"][:, :dkv], x["kv"][:, dkv:]
    if own:
        from neuralrs_amd import _abi as nrs

        nrs.load()
        nrs.init(0)
        s["nrs"] = nrs
        s["buffers"] = _buffers(case, x)
        if case["kind"] == "attn":
            s["mask"] = nrs.attention_mask(causal=True, q_start=x["start"], key_len=x["lens"],
                                           prefix_len=x["prefix"], key_begin=x["begin"],
                                           slopes=x["slopes"], cap=case["cap"])
    return s


def _buffers(case, x):
    """The outputs that a program keeps."""
    if case["kind"] == "attn":
        out = {"out": torch.empty_like(x["q"])}
        if case["use"] == "train":
            b, sq, h = case["batch"], case["seq_q"], case["heads"]
            out["stats"] = torch.empty(b * h * sq * 2, device=x["q"].device)
            out["dq"] = torch.empty_like(x["q"])
            if case["packed"]:
                dkv = case["kv_heads"] * case["d_head"]
                out["dkv"] = torch.empty_like(x["kv"])
                out["dk"], out["dv"] = out["dkv"][:, :dkv], out["dkv"][:, dkv:]
            else:
                out["dk"], out["dv"] = torch.empty_like(x["k"]), torch.empty_like(x["v"])
        return out
    if case["kind"] == "rope":
        return {"out": torch.empty_like(x["x"]), "dx": torch.empty_like(x["x"])}
    out = {"loss": torch.empty(case["rows"], device=x["logits"].device)}
    if case["train"]:
        out["grad"] = torch.empty_like(x["logits"])
    return out


# ------------------------------------------------------------------ the passes
def run(state):
    kind = state["kind"]
    if own:
        return {"attn": _own_attn, "rope": _own_rope, "distill": _own_distill}[kind](state)
    return {"attn": _plain_attn, "rope": _plain_rope, "distill": _plain_distill}[kind](state)


def _own_attn(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    d = s["d_head"]
    ld_q = s["heads"] * d
    ld_kv = s["kv_heads"] * d * (2 if s["packed"] else 1)
    shape = (s["batch"], s["heads"], s["kv_heads"], s["seq_q"], s["seq_k"], d, ld_q, ld_kv, ld_q)
    scale = 1.0 / math.sqrt(d)
    nrs.masked_attention_forward(o["out"], o.get("stats"), x["q"], x["k"], x["v"], s["mask"],
                                 *shape, scale)
    if s["use"] != "train":
        return o["out"]
    nrs.masked_attention_backward(o["dq"], o["dk"], o["dv"], x["dout"], o["out"], x["q"], x["k"],
                                  x["v"], o["stats"], s["mask"], *shape, scale)
    return [o["out"], o["dq"], o["dk"], o["dv"]]


def _own_rope(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    ld = s["heads"] * s["d_head"]
    shape = (s["rows"], s["heads"], s["d_head"], s["pairs"], s["axes"], ld, ld)
    nrs.rotary_forward(o["out"], x["x"], x["positions"], x["freq"], x["axis"], *shape,
                       interleaved=s["interleaved"])
    if not s["train"]:
        return o["out"]
    nrs.rotary_backward(o["dx"], x["dout"], x["positions"], x["freq"], x["axis"], *shape,
                        interleaved=s["interleaved"])
    return [o["out"], o["dx"]]


def _own_distill(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    shape = (s["rows"], s["vocab"], s["k"], s["vocab"])
    if not s["train"]:
        nrs.distill_forward(o["loss"], x["logits"], x["top"], x["ids"], x["labels"], *shape,
                            temperature=s["temperature"], hard=s["hard"])
        return o["loss"]
    nrs.distill_backward(o["grad"], o["loss"], x["row_grad"], x["logits"], x["top"], x["ids"],
                         x["labels"], *shape, temperature=s["temperature"], hard=s["hard"])
    return [o["loss"], o["grad"]]


def _heads(t, batch, seq, heads, d):
    """[batch*seq, heads*d] rows -> contiguous [batch*heads, seq, d]."""
    return t.reshape(batch, seq, heads, d).permute(0, 2, 1, 3).reshape(batch * heads, seq,
                                                                       d).contiguous()


def _rows(t, batch, seq, heads, d):
    return t.reshape(batch, heads, seq, d).permute(0, 2, 1, 3).reshape(batch * seq, heads * d)


def _plain_attn(s):
    x, d, b, h, kv = s["x"], s["d_head"], s["batch"], s["heads"], s["kv_heads"]
    sq, sk, group = s["seq_q"], s["seq_k"], h // kv
    device = x["q"].device
    # the group's heads as more rows of their key head
    q = _heads(x["q"], b, sq, h, d).reshape(b * kv, group * sq, d)
    k, v = _heads(x["k"], b, sk, kv, d), _heads(x["v"], b, sk, kv, d)
    scale = 1.0 / math.sqrt(d)
    start = x["start"] if x["start"] is not None else torch.zeros(b, dtype=torch.int32,
                                                                  device=device)
    i = start[:, None] + torch.arange(sq, dtype=torch.int32, device=device)[None, :]
    t = torch.arange(sk, dtype=torch.int32, device=device)
    seen = t[None, None, :] <= i[:, :, None]
    if x["prefix"] is not None:
        seen |= (t[None, :] < x["prefix"][:, None])[:, None, :]
    if x["lens"] is not None:
        seen &= (t[None, :] < x["lens"][:, None])[:, None, :]
    if x["begin"] is not None:
        seen &= t[None, None, :] >= x["begin"].reshape(b, sq)[:, :, None]
    u = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale)
    slope = None
    if s["cap"] > 0.0:
        u = torch.tanh(u.mul_(1.0 / s["cap"]))
        if s["use"] == "train":
            slope = 1.0 - u * u
        u = u.mul_(s["cap"])
    u = u.reshape(b, h, sq, sk)
    if x["slopes"] is not None:
        far = (i[:, :, None] - t[None, None, :]).abs().float()
        u = u - x["slopes"][None, :, None, None] * far[:, None]
    u = u.masked_fill_(~seen[:, None], -math.inf)
    top = u.amax(dim=-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    u = torch.exp(u.sub_(top))
    total = u.sum(dim=-1, keepdim=True)
    p = u.div_(torch.where(total > 0.0, total, 1.0)).reshape(b * kv, group * sq, sk)
    out = torch.bmm(p, v)
    rows = _rows(out.reshape(b * h, sq, d), b, sq, h, d)
    if s["use"] != "train":
        return rows
    g = _heads(x["dout"], b, sq, h, d).reshape(b * kv, group * sq, d)
    dp = torch.bmm(g, v.transpose(1, 2).contiguous())
    ds = dp.sub_((g * out).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    if slope is not None:
        ds = ds.mul_(slope)
    dq = _rows(torch.bmm(ds, k).reshape(b * h, sq, d), b, sq, h, d)
    dk = _rows(torch.bmm(ds.transpose(1, 2).contiguous(), q), b, sk, kv, d)
    dv = _rows(torch.bmm(p.transpose(1, 2).contiguous(), g), b, sk, kv, d)
    return [rows, dq, dk, dv]


def _plain_turn(s, x, sign):
    """Each pair (a, b) of a head turned by its angle: (a cos - b sin, b cos + a sin)."""
    p, d, n = s["x"], s["d_head"], s["pairs"]
    # far positions times a frequency keep their angle in 64 bits alone
    angle = p["positions"].long()[p["axis"].long()].t() * p["freq"].double()[None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], (sign * torch.sin(angle)).float()[:, None, :]
    y = x.reshape(s["rows"], s["heads"], d).clone()
    if s["interleaved"]:
        a, b = slice(0, 2 * n, 2), slice(1, 2 * n, 2)
    else:
        a, b = slice(0, n), slice(n, 2 * n)
    ya, yb = y[:, :, a] * cos - y[:, :, b] * sin, y[:, :, b] * cos + y[:, :, a] * sin
    y[:, :, a] = ya
    y[:, :, b] = yb
    return y.reshape(x.shape)


def _plain_rope(s):
    out = _plain_turn(s, s["x"]["x"], 1.0)
    return [out, _plain_turn(s, s["x"]["dout"], -1.0)] if s["train"] else out


def _log_softmax(z):
    z = z - z.amax(dim=1, keepdim=True)
    return z - torch.log(torch.exp(z).sum(dim=1, keepdim=True))


def _plain_distill(s):
    x, temp, hard = s["x"], s["temperature"], s["hard"]
    live = x["ids"] >= 0
    ids = x["ids"].long().clamp(min=0)
    logp = _log_softmax(torch.where(live, x["top"] / temp, -math.inf))
    p = torch.where(live, torch.exp(logp), 0.0)
    logq = _log_softmax(x["logits"] / temp)
    kl = torch.where(live, p * (logp - logq.gather(1, ids)), 0.0).sum(dim=1)
    loss = (1.0 - hard) * temp * temp * kl
    if hard > 0.0:
        known = x["labels"] >= 0
        label = x["labels"].long().clamp(min=0)[:, None]
        log1 = _log_softmax(x["logits"]) if temp != 1.0 else logq
        loss = loss - torch.where(known, hard * log1.gather(1, label)[:, 0], 0.0)
    if not s["train"]:
        return loss
    grad = torch.exp(logq).scatter_add_(1, ids, -p).mul_((1.0 - hard) * temp)
    if hard > 0.0:
        one = torch.exp(log1)
        one.scatter_add_(1, label, torch.full_like(label, -1.0, dtype=torch.float32))
        grad = grad + one.mul_(torch.where(known, hard, 0.0)[:, None])
    if x["row_grad"] is not None:
        return [loss, grad.mul_(x["row_grad"][:, None])]
    return [loss, grad.mul_(1.0 / s["rows"])]


# ------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    x = _inputs(case, seed, torch.device("cuda", 0))
    return {"attn": _exact_attn, "rope": _exact_rope, "distill": _exact_distill}[case["kind"]](
        case, x)


def _exact_attn(c, x):
    """Item by item, head by head, blocks of queries over the keys up to the last
    that any of them sees."""
    d, h, kv, sq, sk = c["d_head"], c["heads"], c["kv_heads"], c["seq_q"], c["seq_k"]
    k_all, v_all = (x["k"], x["v"]) if not c["packed"] else torch.split(x["kv"], kv * d, dim=1)
    train, device = c["use"] == "train", x["q"].device
    if c["batch"] * h * (-(-sq // 2048)) > 20000:
        return None  # more products than 20 seconds have
    out = torch.zeros(c["batch"] * sq, h * d, dtype=torch.float64, device=device)
    dq = torch.zeros_like(out)
    dk = torch.zeros(c["batch"] * sk, kv * d, dtype=torch.float64, device=device)
    dv = torch.zeros_like(dk)

    def whole(t, otherwise):
        return [otherwise] * c["batch"] if t is None else t.tolist()

    lens, starts, prefixes = whole(x["lens"], sk), whole(x["start"], 0), whole(x["prefix"], 0)
    for b in range(c["batch"]):
        for first in range(0, sq, 2048):
            last = min(sq, first + 2048)
            at = torch.arange(first, last, device=device) + starts[b]
            n = max(0, min(lens[b], max(starts[b] + last, prefixes[b])))
            keys = torch.arange(n, device=device)
            hidden = keys[None, :] > at[:, None]
            hidden &= keys[None, :] >= prefixes[b]
            if x["begin"] is not None:
                own_doc = x["begin"][b * sq + first:b * sq + last].long()
                hidden |= keys[None, :] < own_doc[:, None]
            empty = hidden.all(dim=1, keepdim=True)
            rows, kr = slice(b * sq + first, b * sq + last), slice(b * sk, b * sk + n)
            for i in range(h):
                qc = slice(i * d, (i + 1) * d)
                kc = slice(i // (h // kv) * d, (i // (h // kv) + 1) * d)
                q, k, v = x["q"][rows, qc].double(), k_all[kr, kc].double(), v_all[kr, kc].double()
                z = torch.mm(q, k.t()) / math.sqrt(d)
                inner = 1.0
                if c["cap"] > 0.0:
                    z = torch.tanh(z / c["cap"])
                    inner = 1.0 - z.square()
                    z = c["cap"] * z
                if x["slopes"] is not None:
                    z = z - x["slopes"][i].double() * (at[:, None] - keys[None, :]).abs()
                w = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1).masked_fill(empty, 0.0)
                out[rows, qc] = torch.mm(w, v)
                if not train:
                    continue
                g = x["dout"][rows, qc].double()
                dw = torch.mm(g, v.t())
                dz = w * (dw - (w * dw).sum(dim=1, keepdim=True)) * inner / math.sqrt(d)
                dq[rows, qc] = torch.mm(dz, k)
                dk[kr, kc] += torch.mm(dz.t(), q)
                dv[kr, kc] += torch.mm(w.t(), g)
    return [out, dq, dk, dv] if train else out


def _exact_rope(c, x):
    """The pairs as complex numbers times a unit one."""
    n, rows = c["pairs"], c["rows"]
    angle = x["positions"].double()[x["axis"].long()].t() * x["freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]

    def turned(t, by):
        t = t.double().reshape(rows, c["heads"], c["d_head"])
        head, rest = t[..., :2 * n], t[..., 2 * n:]
        head = (head.reshape(rows, -1, n, 2) if c["interleaved"]
                else head.reshape(rows, -1, 2, n).transpose(2, 3))
        y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * by)
        if not c["interleaved"]:
            y = y.transpose(2, 3)
        return torch.cat([y.reshape(rows, -1, 2 * n), rest], dim=2).reshape(rows, -1)

    out = turned(x["x"], turn)
    return [out, turned(x["dout"], turn.conj())] if c["train"] else out


def _exact_distill(c, x):
    """Some rows at a time."""
    rows, vocab, temp, hard = c["rows"], c["vocab"], c["temperature"], c["hard"]
    device = x["logits"].device
    loss = torch.zeros(rows, dtype=torch.float64, device=device)
    grad = torch.zeros(rows, vocab, dtype=torch.float64, device=device) if c["train"] else None
    step = max(1, 2 ** 27 // vocab)
    for r in range(0, rows, step):
        z = x["logits"][r:r + step].double()
        ids = x["ids"][r:r + step].long()
        none = ids < 0
        teacher = torch.softmax((x["top"][r:r + step].double() / temp).masked_fill(none, -math.inf),
                                dim=1)
        # the teacher's weights over the whole vocabulary (a column more for no token)
        target = torch.zeros(z.shape[0], vocab + 1, dtype=torch.float64, device=device)
        target.scatter_(1, torch.where(none, vocab, ids), teacher)
        target = target[:, :vocab]
        entropy = torch.special.entr(target).sum(dim=1)
        soft = torch.log_softmax(z / temp, dim=1)
        loss[r:r + step] = (1.0 - hard) * temp ** 2 * (-(target * soft).sum(dim=1) - entropy)
        g = (1.0 - hard) * temp * (soft.exp() - target)
        if hard > 0.0:
            label = x["labels"][r:r + step].long()
            at = torch.nonzero(label >= 0).flatten()
            logs = torch.log_softmax(z[at], dim=1)
            loss[r + at] -= hard * logs[torch.arange(at.numel(), device=device), label[at]]
            dense = logs.exp()
            dense[torch.arange(at.numel(), device=device), label[at]] -= 1.0
            g[at] += hard * dense
        if grad is not None:
            by = x["row_grad"][r:r + step].double() if x["row_grad"] is not None else 1.0 / rows
            grad[r:r + step] = g * (by[:, None] if torch.is_tensor(by) else by)
    return [loss, grad] if c["train"] else loss
