"""The operators of encoder-decoder models as measurable cases.

Cross attention to an encoder's states, embedding lookup with its gradient
by sorted tokens, and dropout from a counter-based generator. With ``own``
false ``run`` computes them in elementary torch operations; with ``own``
true it calls the entry points of ``include/nrs_hip.h`` through
``neuralrs_amd._abi`` on the same tensors, with output buffers that the
program keeps from call to call. f32 is the library's only type; ids and
lengths are int32.

A training case is the forward and the backward of one operator: the
backward takes the forward's output and statistics, and writes the gradients
(beta 0, as into gradients that were just zeroed).
"""
import math

import numpy as np
import torch

own = False

_LOG2E = 1.4426950408889634


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # A decoder's cross attention while training at the block size that
        # the repository measures (batch 32, 8 heads of 32), over shorter and
        # longer source sentences, one of them empty (a place of the batch not
        # in use); keys and values in one projection.
        {"name": "cross_train_32x128x200h8x32", "kind": "cross", "train": True, "batch": 32,
         "heads": 8, "kv_heads": 8, "seq_q": 128, "seq_k": 200, "d_head": 32, "packed": True,
         "ragged": True, "empty": True},
        # Training over long sources, odd lengths, heads of 64, every key live.
        {"name": "cross_train_4x1000x1500h16x64", "kind": "cross", "train": True, "batch": 4,
         "heads": 16, "kv_heads": 16, "seq_q": 1000, "seq_k": 1500, "d_head": 64,
         "packed": False, "ragged": False, "empty": False},
        # The largest call: a prompt of a few hundred tokens reads a long source, four query
        # heads to a key head, heads of 128, training.
        {"name": "cross_train_2x777x4096h16g4x128", "kind": "cross", "train": True, "batch": 2,
         "heads": 16, "kv_heads": 4, "seq_q": 777, "seq_k": 4096, "d_head": 128,
         "packed": True, "ragged": True, "empty": False},
        # The same prompt when serving: forward alone, no statistics kept.
        {"name": "cross_prompt_4x512x1500h16x64", "kind": "cross", "train": False, "batch": 4,
         "heads": 16, "kv_heads": 16, "seq_q": 512, "seq_k": 1500, "d_head": 64,
         "packed": True, "ragged": True, "empty": False},
        # One new token for each of 32 requests over sources of mixed length.
        {"name": "cross_token_32x1500h8x64", "kind": "cross", "train": False, "batch": 32,
         "heads": 8, "kv_heads": 8, "seq_q": 1, "seq_k": 1500, "d_head": 64, "packed": True,
         "ragged": True, "empty": False},
        # One token of two requests over a very long source: the key axis is
        # all there is to share out.
        {"name": "cross_token_2x16384h32g4x128", "kind": "cross", "train": False, "batch": 2,
         "heads": 32, "kv_heads": 8, "seq_q": 1, "seq_k": 16384, "d_head": 128, "packed": False,
         "ragged": False, "empty": False},
        # The smallest calls: the embeddings of one decoding step.
        {"name": "embed_step_32x256", "kind": "embed", "train": False, "count": 32,
         "vocab": 8000, "dim": 256, "pad": 0.0},
        # A training batch at the repository's block size, with padding tokens.
        {"name": "embed_train_4096x256v32000", "kind": "embed", "train": True, "count": 4096,
         "vocab": 32000, "dim": 256, "pad": 0.1},
        # A large batch of odd size over a large table, and few rows for many
        # tokens (bytes): long sums into each row.
        {"name": "embed_train_49999x1000v50021", "kind": "embed", "train": True, "count": 49999,
         "vocab": 50021, "dim": 1000, "pad": 0.02},
        {"name": "embed_train_65536x512v259", "kind": "embed", "train": True, "count": 65536,
         "vocab": 259, "dim": 512, "pad": 0.0},
        # Dropout with its residual add on the activations of one decoding-size
        # batch (latency), and of a feed-forward layer at training size.
        {"name": "dropout_32x256", "kind": "dropout", "rows": 32, "width": 256, "p": 0.1,
         "residual": True},
        {"name": "dropout_4096x4096", "kind": "dropout", "rows": 4096, "width": 4096, "p": 0.1,
         "residual": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cross", "cross", "cross", "embed", "embed", "dropout"])
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("cross", "embed",
                                                                           "dropout")}
    while True:
        if kind == "cross":
            use = rng.choice(["train", "prompt", "token"])
            kv = rng.choice([1, 2, 3, 4, 8, 16])
            group = rng.choice([1, 1, 1, 2, 4, 7])
            case = {"kind": kind, "train": use == "train", "batch": _log_int(rng, 1, 64),
                    "heads": kv * group, "kv_heads": kv,
                    "seq_q": 1 if use == "token" else _log_int(rng, 2, 2000),
                    "seq_k": _log_int(rng, 1, 16384),
                    "d_head": rng.choice([16, 32, 64, 128, 24, 40, 80, 96, rng.randint(8, 128)]),
                    "packed": rng.random() < 0.5, "ragged": rng.random() < 0.6}
            case["empty"] = case["ragged"] and case["batch"] > 1 and rng.random() < 0.4
        elif kind == "embed":
            case = {"kind": kind, "train": rng.random() < 0.7, "count": _log_int(rng, 1, 66000),
                    "vocab": _log_int(rng, 2, 130000), "dim": _log_int(rng, 16, 2048),
                    "pad": rng.choice([0.0, 0.05, 0.3])}
        else:
            case = {"kind": kind, "rows": _log_int(rng, 1, 8192), "width": _log_int(rng, 16, 4096),
                    "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "residual": rng.random() < 0.5}
        if _cost(case) <= most[kind]:
            return case


def _lengths(case):
    """The live keys of each item, before their order is drawn: from all of
    them down to a seventh, by even steps, or none for the last."""
    b, n = case["batch"], case["seq_k"]
    if not case["ragged"]:
        return [n] * b
    lens = [max(1, n - (i * (n - n // 7)) // b) for i in range(b)]
    return lens[:-1] + [0] if case["empty"] else lens


def work(case):
    if case["kind"] == "cross":
        live = sum(_lengths(case))
        h, kv, d = case["heads"], case["kv_heads"], case["d_head"]
        rows = case["batch"] * case["seq_q"] * h
        pairs = live * case["seq_q"] * h
        q, kvb, stats = 4 * rows * d, 4 * live * kv * d, 8 * rows
        lens = 4 * case["batch"] if case["ragged"] else 0
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kvb + lens, "flops": 4 * pairs * d}
        # forward: q, k, v in, out and statistics out; backward: those and
        # dout in, dq, dk, dv out (dk, dv for every row of k and v)
        all_kv = 4 * case["batch"] * case["seq_k"] * kv * d
        return {"bytes": 2 * q + 2 * kvb + stats + lens + 4 * q + 2 * kvb + stats + 2 * all_kv,
                "flops": 14 * pairs * d}
    if case["kind"] == "embed":
        n, d, v = case["count"], case["dim"], case["vocab"]
        fwd = 4 * n + 4 * min(n, v) * d + 4 * n * d
        if not case["train"]:
            return {"bytes": fwd, "flops": n * d}
        return {"bytes": fwd + 4 * n + 4 * n * d + 4 * v * d, "flops": 3 * n * d}
    n = case["rows"] * case["width"]
    return {"bytes": 4 * n * (2 + (1 if case["residual"] else 0) + 2), "flops": 5 * n}


def _cost(case):
    """Work and memory of the plain form, in one figure."""
    w = work(case)
    if case["kind"] == "cross":
        pairs = case["batch"] * case["seq_q"] * case["seq_k"] * case["heads"]
        return w["flops"] / 1e14 + (w["bytes"] + 30 * pairs) / 4e12
    return w["bytes"]


# ------------------------------------------------------------------ the inputs
def _inputs(case, seed, device):
    g = torch.Generator(device=device).manual_seed(1000003 * seed + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    if case["kind"] == "cross":
        b, sq, sk = case["batch"], case["seq_q"], case["seq_k"]
        dq, dkv = case["heads"] * case["d_head"], case["kv_heads"] * case["d_head"]
        x = {"q": normal(b * sq, dq), "kv": normal(b * sk, 2 * dkv)}
        if not case["packed"]:
            x["k"], x["v"] = x["kv"][:, :dkv].contiguous(), x["kv"][:, dkv:].contiguous()
            del x["kv"]
        if case["train"]:
            x["dout"] = normal(b * sq, dq)
        x["lens"] = None
        if case["ragged"]:
            order = torch.randperm(b, generator=torch.Generator().manual_seed(seed + 5)).tolist()
            lens = _lengths(case)
            x["lens"] = torch.tensor([lens[i] for i in order], dtype=torch.int32, device=device)
        return x
    if case["kind"] == "embed":
        n, v, d = case["count"], case["vocab"], case["dim"]
        # word frequencies fall off as one over their rank; ranks lie anywhere
        # in the table; some places are padding (id -1)
        u = torch.rand(n, generator=g, device=device, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        ids = torch.randperm(v, generator=g, device=device)[rank].to(torch.int32)
        pad = torch.rand(n, generator=g, device=device) < case["pad"]
        x = {"ids": torch.where(pad, torch.full_like(ids, -1), ids), "table": normal(v, d),
             "scale": math.sqrt(d)}
        if case["train"]:
            x["dout"] = normal(n, d)
        return x
    n = case["rows"] * case["width"]
    x = {"x": normal(n), "dout": normal(n), "residual": normal(n) if case["residual"] else None}
    # the probability as the f32 that the entry points take
    x["p"] = float(np.float32(case["p"]))
    x["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) & 0xFFFFFFFFFFFFFFFF
    x["call"] = 3 + seed
    return x


def prepare(case, seed):
    device = torch.device("cuda", 0)
    x = _inputs(case, seed, device)
    s = dict(case)
    s["x"] = x
    if case["kind"] == "cross":
        dkv = case["kv_heads"] * case["d_head"]
        if case["packed"]:
            x["k"], x["v"] = x["kv"][:, :dkv], x["kv"][:, dkv:]
    if own:
        from neuralrs_amd import _abi as nrs

        nrs.load()
        nrs.init(0)
        s["nrs"] = nrs
        s["buffers"] = _buffers(case, x)
    return s


def _buffers(case, x):
    """The outputs that a program keeps."""
    if case["kind"] == "cross":
        out = {"out": torch.empty_like(x["q"])}
        if case["train"]:
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
    if case["kind"] == "embed":
        out = {"out": torch.empty(case["count"], case["dim"], device=x["table"].device)}
        if case["train"]:
            out["dtable"] = torch.empty_like(x["table"])
        return out
    return {"out": torch.empty_like(x["x"]), "dx": torch.empty_like(x["x"])}


# ------------------------------------------------------------------ the passes
def run(state):
    kind = state["kind"]
    if own:
        return {"cross": _own_cross, "embed": _own_embed, "dropout": _own_dropout}[kind](state)
    return {"cross": _plain_cross, "embed": _plain_embed, "dropout": _plain_dropout}[kind](state)


def _own_cross(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    d = s["d_head"]
    ld_q = s["heads"] * d
    ld_kv = s["kv_heads"] * d * (2 if s["packed"] else 1)
    scale = 1.0 / math.sqrt(d)
    shape = (s["batch"], s["heads"], s["kv_heads"], s["seq_q"], s["seq_k"], d, ld_q, ld_kv, ld_q)
    nrs.cross_attention_forward(o["out"], o.get("stats"), x["q"], x["k"], x["v"], x["lens"],
                                *shape, scale)
    if not s["train"]:
        return o["out"]
    nrs.cross_attention_backward(o["dq"], o["dk"], o["dv"], x["dout"], o["out"], x["q"], x["k"],
                                 x["v"], o["stats"], x["lens"], *shape, scale)
    return [o["out"], o["dq"], o["dk"], o["dv"]]


def _own_embed(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    nrs.embedding_forward(o["out"], x["table"], x["ids"], s["count"], s["vocab"], s["dim"],
                          x["scale"])
    if not s["train"]:
        return o["out"]
    nrs.embedding_backward(o["dtable"], x["dout"], x["ids"], s["count"], s["vocab"], s["dim"],
                           x["scale"])
    return [o["out"], o["dtable"]]


def _own_dropout(s):
    nrs, x, o = s["nrs"], s["x"], s["buffers"]
    n = s["rows"] * s["width"]
    nrs.dropout_forward(o["out"], x["x"], x["residual"], n, x["p"], x["seed"], x["call"])
    nrs.dropout_backward(o["dx"], x["dout"], n, x["p"], x["seed"], x["call"])
    return [o["out"], o["dx"]]


def _heads(t, batch, seq, heads, d):
    """[batch*seq, heads*d] rows -> contiguous [batch*heads, seq, d]."""
    return t.reshape(batch, seq, heads, d).permute(0, 2, 1, 3).reshape(batch * heads, seq,
                                                                       d).contiguous()


def _rows(t, batch, seq, heads, d):
    return t.reshape(batch, heads, seq, d).permute(0, 2, 1, 3).reshape(batch * seq, heads * d)


def _plain_cross(s):
    x, d, b, h, kv = s["x"], s["d_head"], s["batch"], s["heads"], s["kv_heads"]
    sq, sk, group = s["seq_q"], s["seq_k"], h // kv
    # the group's heads as more rows of their key head
    q = _heads(x["q"], b, sq, h, d).reshape(b * kv, group * sq, d)
    k, v = _heads(x["k"], b, sk, kv, d), _heads(x["v"], b, sk, kv, d)
    scale = 1.0 / math.sqrt(d)
    u = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    if x["lens"] is not None:
        dead = torch.arange(sk, device=u.device)[None, :] >= x["lens"][:, None]
        u = u.reshape(b, kv, group * sq, sk).masked_fill_(dead[:, None, None, :], -math.inf)
        u = u.reshape(b * kv, group * sq, sk)
    top = u.amax(dim=-1, keepdim=True)
    if s["empty"]:
        top = top.clamp_(min=torch.finfo(torch.float32).min)  # rows without a live key
    u = torch.exp(u - top)
    total = u.sum(dim=-1, keepdim=True)
    p = u / (total.clamp_(min=1.0) if s["empty"] else total)
    out = torch.bmm(p, v)
    rows = _rows(out.reshape(b * h, sq, d), b, sq, h, d)
    if not s["train"]:
        return rows
    g = _heads(x["dout"], b, sq, h, d).reshape(b * kv, group * sq, d)
    dp = torch.bmm(g, v.transpose(1, 2).contiguous())
    ds = p * (dp - (g * out).sum(dim=-1, keepdim=True)) * scale
    dq = _rows(torch.bmm(ds, k).reshape(b * h, sq, d), b, sq, h, d)
    dk = _rows(torch.bmm(ds.transpose(1, 2).contiguous(), q), b, sk, kv, d)
    dv = _rows(torch.bmm(p.transpose(1, 2).contiguous(), g), b, sk, kv, d)
    return [rows, dq, dk, dv]


def _plain_embed(s):
    x = s["x"]
    ids = x["ids"].long()
    live = (ids >= 0)[:, None]
    out = torch.where(live, x["table"][ids.clamp(min=0)] * x["scale"], 0.0)
    if not s["train"]:
        return out
    grad = torch.where(live, x["dout"], 0.0)
    # sums of many rows in 64 bits
    dtable = torch.zeros(s["vocab"], s["dim"], dtype=torch.float64, device=out.device)
    dtable.index_add_(0, ids.clamp(min=0), grad.double())
    return [out, (dtable * x["scale"]).float()]


def _philox_words(n, seed, call, device):
    """Words of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
    numbers: as easy as 1, 2, 3", SC 2011), element i's being word i % 4 of
    the block with counter (i / 4, call) under the key seed. 32-bit words in
    int64: a product's wrapped bits are those of the unsigned one."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = torch.full_like(block, call & low), torch.full_like(block, (call >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1,
                          a & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


def _plain_dropout(s):
    x, n = s["x"], s["rows"] * s["width"]
    p = x["p"]
    keep = _philox_words(n, x["seed"], x["call"], x["x"].device) >= int(p * 4294967296.0 + 0.5)
    inv = 1.0 / (1.0 - p)
    out = torch.where(keep, x["x"] * inv, 0.0)
    if x["residual"] is not None:
        out = x["residual"] + out
    return [out, torch.where(keep, x["dout"] * inv, 0.0)]


# ------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    device = torch.device("cuda", 0)
    x = _inputs(case, seed, device)
    return {"cross": _exact_cross, "embed": _exact_embed, "dropout": _exact_dropout}[case["kind"]](
        case, x)


def _exact_cross(c, x):
    """Item by item and key head by key head, over the live keys alone."""
    d, h, kv, sq, sk = c["d_head"], c["heads"], c["kv_heads"], c["seq_q"], c["seq_k"]
    if not c["packed"]:
        k_all, v_all = x["k"], x["v"]
    else:
        k_all, v_all = torch.split(x["kv"], kv * d, dim=1)
    group = h // kv
    out = torch.zeros(c["batch"] * sq, h * d, dtype=torch.float64, device=x["q"].device)
    dq = torch.zeros_like(out)
    dk = torch.zeros(c["batch"] * sk, kv * d, dtype=torch.float64, device=x["q"].device)
    dv = torch.zeros_like(dk)
    lens = [sk] * c["batch"] if x["lens"] is None else x["lens"].tolist()
    for b, n in enumerate(lens):
        qr, kr = slice(b * sq, (b + 1) * sq), slice(b * sk, b * sk + n)
        for j in range(kv):
            kc = slice(j * d, (j + 1) * d)
            k, v = k_all[kr, kc].double(), v_all[kr, kc].double()
            for i in range(j * group, (j + 1) * group):
                qc = slice(i * d, (i + 1) * d)
                q = x["q"][qr, qc].double()
                weights = torch.softmax(torch.mm(q, k.t()) / math.sqrt(d), dim=1)
                out[qr, qc] = torch.mm(weights, v)
                if not c["train"]:
                    continue
                g = x["dout"][qr, qc].double()
                dw = torch.mm(g, v.t())
                dscore = weights * (dw - (weights * dw).sum(dim=1, keepdim=True)) / math.sqrt(d)
                dq[qr, qc] = torch.mm(dscore, k)
                dk[kr, kc] += torch.mm(dscore.t(), q)
                dv[kr, kc] += torch.mm(weights.t(), g)
    return [out, dq, dk, dv] if c["train"] else out


def _exact_embed(c, x):
    ids = x["ids"].long()
    live = torch.nonzero(ids >= 0).flatten()
    out = torch.zeros(c["count"], c["dim"], dtype=torch.float64, device=ids.device)
    out[live] = x["table"].double()[ids[live]] * x["scale"]
    if not c["train"]:
        return out
    order = live[torch.argsort(ids[live], stable=True)]
    sums = torch.cumsum(x["dout"].double()[order], dim=0)
    dtable = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device=ids.device)
    if order.numel():
        # the difference of running sums at the ends of each token's run
        last = torch.cat([ids[order][1:] != ids[order][:-1], torch.ones(1, dtype=torch.bool,
                                                                        device=ids.device)])
        ends = sums[last]
        dtable[ids[order][last]] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1]))
    return [out, dtable * x["scale"]]


def _exact_dropout(c, x):
    """The generator in numpy's unsigned integers, on the host."""
    n = c["rows"] * c["width"]
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    ctr = [block & low, block >> half, np.full_like(block, x["call"] & 0xFFFFFFFF),
           np.full_like(block, x["call"] >> 32)]
    for r in range(10):
        key = ((x["seed"] + r * 0x9E3779B9) & 0xFFFFFFFF,
               ((x["seed"] >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> half) ^ ctr[1] ^ np.uint64(key[0]), b & low,
               (a >> half) ^ ctr[3] ^ np.uint64(key[1]), a & low]
    words = np.stack(ctr, axis=1).reshape(-1)[:n]
    p = x["p"]
    kept = torch.from_numpy(words >= np.uint64(int(p * 4294967296.0 + 0.5))).to(x["x"].device)
    factor = kept.double() / (1.0 - p)
    out = x["x"].double() * factor
    if x["residual"] is not None:
        out = out + x["residual"].double()
    return [out, x["dout"].double() * factor]
