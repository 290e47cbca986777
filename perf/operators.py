"""What the long-context operators cost: rotary positions, attention over a prefix that a whole batch
shares, and attention over the key blocks that a cheap int8 score selects.

A case is one pass through one operator. Its plain form is elementary torch operations in 32 bits
(angles in 64), rounded once at the end; its own form is the calls of e2.c_amd/e2mi.py that a user
makes. Inputs are made on the GPU from the seed alone; lengths follow from the case alone. Rows of
queries and keys are packed: sequence b holds rows [start[b], start[b] + len[b]), key ranges start at
multiples of 8, V is transposed ([kv head][dim][row]).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
_e2mi = None

BLOCK = 64  # keys per block of the selecting attention
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
INV127 = 0.007874015718698502  # 1/127 rounded to 32 bits: the quantizer's scale is amax * this


def listed():
    return [
        # one new token of a stream: q of 3 heads and k of 1 (BASELINE heads)
        {"name": "rope_token", "op": "rope", "rows": 1, "heads": 3, "kv": 1, "d": 256, "rot": 256, "layout": "half",
         "scaling": "none", "dtype": "f16", "inverse": False, "far": 4096},
        # a batch of documents (64 x 512, U[64, 512] packed), interleaved pairs in half of each head, stretched 4x
        {"name": "rope_docs_interleaved", "op": "rope", "rows": 17264, "heads": 3, "kv": 1, "d": 256, "rot": 128,
         "layout": "interleaved", "scaling": "linear", "dtype": "bf16", "inverse": False, "far": 8192},
        # the gradient of q and k (the rotation turned back) of one long text, odd row count, base stretched
        {"name": "rope_gradient", "op": "rope", "rows": 4099, "heads": 16, "kv": 4, "d": 128, "rot": 128,
         "layout": "half", "scaling": "base", "dtype": "f16", "inverse": True, "far": 32768},
        # a very long text in f32 (the f32 copies of q and k), full-attention layers, far positions
        {"name": "rope_long_f32", "op": "rope", "rows": 65536, "heads": 4, "kv": 1, "d": 512, "rot": 512,
         "layout": "half", "scaling": "parts", "dtype": "f32", "inverse": False, "far": 1000000},
        # one short query behind a prompt: latency
        {"name": "prefix_token", "op": "prefix", "batch": 1, "q_min": 1, "q_max": 1, "k_min": 19, "k_max": 19,
         "prefix": 512, "heads": 3, "kv": 1, "d": 256, "dtype": "f16", "causal": False, "lens": 1},
        # single tokens of 64 streams behind one long document
        {"name": "prefix_tokens_batch", "op": "prefix", "batch": 64, "q_min": 1, "q_max": 1, "k_min": 0, "k_max": 512,
         "prefix": 16384, "heads": 4, "kv": 2, "d": 256, "dtype": "bf16", "causal": False, "lens": 2},
        # chunks of a document (64 x 512, U[64, 512]), each with the document's context before it
        {"name": "prefix_docs", "op": "prefix", "batch": 64, "q_min": 64, "q_max": 512, "k_min": -1, "k_max": -1,
         "prefix": 2048, "heads": 3, "kv": 1, "d": 256, "dtype": "f16", "causal": False, "lens": 3},
        # a few long continuations of an odd-sized prefix, causal, head dim of the full-attention layers
        {"name": "prefix_causal_512", "op": "prefix", "batch": 5, "q_min": 301, "q_max": 1500, "k_min": -1, "k_max": -1,
         "prefix": 4099, "heads": 4, "kv": 1, "d": 512, "dtype": "bf16", "causal": True, "lens": 4},
        # single tokens of 16 long streams whose block bounds the program keeps beside the keys
        {"name": "blocks_tokens", "op": "blocks", "batch": 16, "q_min": 1, "q_max": 1, "k_min": 9000, "k_max": 65536,
         "heads": 4, "kv": 1, "d": 256, "dtype": "f16", "causal": True, "q_block": 1, "n_sel": 32, "n_first": 1,
         "n_local": 2, "kept": True, "lens": 5},
        # one long document, bidirectional: bounds, selection and attention of a layer
        {"name": "blocks_document", "op": "blocks", "batch": 1, "q_min": -1, "q_max": -1, "k_min": 16384, "k_max": 16384,
         "heads": 3, "kv": 1, "d": 256, "dtype": "f16", "causal": False, "q_block": 32, "n_sel": 16, "n_first": 1,
         "n_local": 1, "kept": False, "lens": 6},
        # a ragged batch, causal, many small heads in groups
        {"name": "blocks_ragged", "op": "blocks", "batch": 5, "q_min": -1, "q_max": -1, "k_min": 700, "k_max": 8001,
         "heads": 16, "kv": 4, "d": 128, "dtype": "bf16", "causal": True, "q_block": 16, "n_sel": 12, "n_first": 1,
         "n_local": 2, "kept": False, "lens": 7},
        # the longest text: full-attention layers of head dim 512
        {"name": "blocks_longest", "op": "blocks", "batch": 1, "q_min": -1, "q_max": -1, "k_min": 65521, "k_max": 65521,
         "heads": 4, "kv": 1, "d": 512, "dtype": "f16", "causal": False, "q_block": 64, "n_sel": 32, "n_first": 1,
         "n_local": 1, "kept": False, "lens": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "prefix", "blocks"])
    heads, kv = rng.choice([(3, 1), (4, 2), (4, 1), (16, 4), (8, 8), (12, 2)])
    if op == "rope":
        d = rng.choice([64, 128, 256, 512])
        dtype = rng.choice(["f16", "bf16", "f32"])
        most = 650_000_000 // ((heads + kv) * d * (4 if dtype == "f32" else 2))
        return {"op": "rope", "rows": _log(rng, 1, min(100_000, most)), "heads": heads, "kv": kv, "d": d,
                "rot": rng.choice([d, d, d // 2, d // 4 + 2]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "base", "parts"]), "dtype": dtype,
                "inverse": rng.random() < 0.3, "far": _log(rng, 100, 2_000_000)}
    dtype = rng.choice(["f16", "bf16"])
    d = rng.choice([64, 128, 256, 512]) if kv < 4 else rng.choice([64, 128])
    token = rng.random() < 0.4
    causal = rng.random() < 0.5
    if op == "prefix":
        prefix = _log(rng, 1, 24_000)
        batch = _log(rng, 1, 64)
        if token:
            k_max = _log(rng, 1, 2000)
            c = {"q_min": 1, "q_max": 1, "k_min": 0, "k_max": k_max}
        else:
            top = 1.0e11 / (4 * d * heads * batch * (prefix + 300))
            q_max = _log(rng, 2, max(3, min(1500, int(top))))
            c = {"q_min": max(1, q_max // 5), "q_max": q_max, "k_min": -1, "k_max": -1}
        return {"op": "prefix", "batch": batch, **c, "prefix": prefix, "heads": heads, "kv": kv, "d": d, "dtype": dtype,
                "causal": causal, "lens": rng.randrange(1 << 30)}
    n_sel = _log(rng, 3, 32)
    if token:
        batch, q_block, q = _log(rng, 1, 24), 1, 1
        k_max = _log(rng, 100, min(65536, 120_000_000 // (batch * kv * d)))
    else:
        batch, q_block, q = _log(rng, 1, 4), rng.choice([8, 16, 24, 32, 64]), -1
        k_max = _log(rng, 100, min(20_000, 1_000_000_000 * q_block // (batch * kv * n_sel * BLOCK * d)))
    return {"op": "blocks", "batch": batch, "q_min": q, "q_max": q, "k_min": k_max // 4 + 1, "k_max": k_max, "heads": heads,
            "kv": kv, "d": d, "dtype": dtype, "causal": causal, "q_block": q_block, "n_sel": n_sel,
            "n_first": rng.choice([0, 1]), "n_local": 0 if n_sel < 6 else rng.choice([0, 1, 2]), "kept": token,
            "lens": rng.randrange(1 << 30)}


# ---- lengths and row layout: from the case alone

def _lens(c):
    rng = random.Random(c["lens"])
    k = [rng.randint(c["k_min"], c["k_max"]) for _ in range(c["batch"])] if c["k_min"] >= 0 else None
    q = [rng.randint(c["q_min"], c["q_max"]) for _ in range(c["batch"])] if c["q_min"] >= 0 else None
    if k is not None:
        k[0] = c["k_max"]
    if q is not None:
        q[0] = c["q_max"]
    return (q if q is not None else list(k)), (k if k is not None else list(q))


def _starts(lens, step):
    at, got = 0, []
    for n in lens:
        got.append(at)
        at += -(-n // step) * step
    return got, max(step, at)


def _seen(nq, nk, causal):
    """Own keys that a sequence's queries see, over all of them."""
    return sum(max(0, min(nk, i + 1 + nk - nq)) for i in range(nq)) if causal else nq * nk


def _picked(c, nq, nk):
    """Keys that a sequence's queries read with the selecting attention, over all queries (about)."""
    n = 0
    for i in range(0, nq, c["q_block"]):
        rows = min(c["q_block"], nq - i)
        top = min(nk, i + rows + nk - nq) if c["causal"] else nk
        n += rows * min(c["n_sel"] * BLOCK, max(0, top))
    return n


def work(c):
    if c["op"] == "rope":
        n = c["rows"] * (c["heads"] + c["kv"]) * c["d"]
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": 2 * n * size + 4 * c["rows"] + 4 * c["rot"],
                "flops": 3 * c["rows"] * (c["heads"] + c["kv"]) * c["rot"]}
    q, k = _lens(c)
    io = 2 * 2 * sum(q) * c["heads"] * c["d"]
    kv_row = 2 * 2 * c["kv"] * c["d"]
    if c["op"] == "prefix":
        pairs = sum(n * c["prefix"] + _seen(n, m, c["causal"]) for n, m in zip(q, k))
        return {"bytes": io + kv_row * (c["prefix"] + sum(k)), "flops": 4 * c["d"] * c["heads"] * pairs}
    nb = [-(-m // BLOCK) for m in k]
    pairs = sum(_picked(c, n, m) for n, m in zip(q, k))
    bounds = sum(nb) * c["kv"] * (2 * c["d"] + 4)
    reach = sum(min(m, _picked(c, n, m)) for n, m in zip(q, k))  # keys read at least once
    nqb = [-(-n // c["q_block"]) for n in q]
    keys = bounds + kv_row * reach if c["kept"] else kv_row // 2 * (sum(k) + reach)
    return {"bytes": io + keys + 4 * sum(nqb) * c["kv"] * c["n_sel"],
            "flops": 4 * c["d"] * c["heads"] * (pairs + sum(n * m for n, m in zip(q, nb)))}


# ---- inputs

def _freqs(c):
    """Angle per position of each rotated pair, in 64 bits, for the case's scaling (factor 4; trained on 4096)."""
    rot, theta, factor, trained = c["rot"], 10000.0, 4.0, 4096
    i = np.arange(rot // 2, dtype=np.float64)
    if c["scaling"] == "base":
        theta = theta * factor ** (rot / (rot - 2.0))
    f = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        f = f / factor
    elif c["scaling"] == "parts":  # turns over the trained length: under 1 stretched, over 32 as they are
        keep = np.clip((trained * f / (2 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    t = TYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if c["op"] == "rope":
        M, H, KV, D = c["rows"], c["heads"], c["kv"], c["d"]
        return {"c": c, "q": randn(M, H * D).to(t), "k": randn(M, KV * D).to(t),
                "pos": torch.randint(0, c["far"], (M,), generator=g, device=dev, dtype=torch.int32),
                "freqs": torch.from_numpy(_freqs(c)).to(dev)}
    H, KV, D = c["heads"], c["kv"], c["d"]
    ql, kl = _lens(c)
    qs, Mq = _starts(ql, 1 if c["q_max"] == 1 else 8)
    ks, Mk = _starts(kl, 8)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"c": c, "max_q": max(ql), "max_k": max(kl), "q_start": i32(qs), "q_len": i32(ql), "k_start": i32(ks),
         "k_len": i32(kl), "vt": randn(KV, D, Mk).to(t), "ctx": torch.zeros((Mq, H * D), dtype=t, device=dev)}
    # keys come in topics (runs of 50 rows about one direction), queries near the topic of some key: a
    # normed q.k that has something to find, as texts do
    topic = randn(Mk // 50 + 1, KV, D)
    of = torch.arange(Mk, device=dev) // 50
    s["k"] = (0.7 * topic[of] + 0.7 * randn(Mk, KV, D)).to(t).reshape(Mk, KV * D)
    near = topic[torch.randint(0, topic.shape[0], (Mq,), generator=g, device=dev)]
    s["q"] = (0.5 * near.repeat_interleave(H // KV, 1) + 0.9 * randn(Mq, H, D)).to(t).reshape(Mq, H * D)
    if c["op"] == "prefix":
        P = c["prefix"]
        s["pk"], s["pvt"] = randn(P, KV * D).to(t), randn(KV, D, P).to(t)
    elif c["kept"]:
        s["bounds"] = _bounds(s)
    return s


# ---- plain forms

def _rope(s):
    c = s["c"]
    rot, D = c["rot"], c["d"]
    turn = s["pos"].double()[:, None] * s["freqs"][None, :]
    turn = -turn if c["inverse"] else turn
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]

    def of(x):
        v = x.float().view(x.shape[0], -1, D)
        a, b = (v[..., :rot // 2], v[..., rot // 2:rot]) if c["layout"] == "half" else (v[..., 0:rot:2], v[..., 1:rot:2])
        y1, y2 = a * cos - b * sin, b * cos + a * sin
        y = torch.cat([y1, y2], -1) if c["layout"] == "half" else torch.stack([y1, y2], -1).flatten(-2)
        return torch.cat([y, v[..., rot:]], -1).to(x.dtype).view_as(x)

    return of(s["q"]), of(s["k"])


def _padded(start, n, most, rows):
    """Row index [B, most] of each sequence's rows, and which of them are rows."""
    at = torch.arange(most, device=start.device)
    ok = at[None] < n[:, None]
    return (start[:, None] + at[None]).clamp(0, rows - 1).long(), ok


def _softmax_v(logits, mask, v):
    """softmax over the last axis of the masked logits, times v; zero where nothing is seen."""
    logits = logits.masked_fill_(~mask, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _scatter(s, ctx, row, ok):
    """Padded contexts [B, rows, H * D] into the packed output."""
    out = torch.zeros_like(s["ctx"])
    out[row[ok]] = ctx[ok].to(out.dtype)
    return out


def _prefix(s):
    c = s["c"]
    H, KV, D, B, P = c["heads"], c["kv"], c["d"], c["batch"], c["prefix"]
    G, Q, K = H // KV, s["max_q"], s["max_k"]
    qrow, qok = _padded(s["q_start"], s["q_len"], Q, s["q"].shape[0])
    krow, kok = _padded(s["k_start"], s["k_len"], K, s["k"].shape[0])
    q = s["q"].float()[qrow].view(B, Q, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * Q, D) * D ** -0.5
    k = s["k"].float()[krow].view(B, K, KV, D).permute(0, 2, 3, 1)
    v = s["vt"].float()[:, :, krow].permute(2, 0, 3, 1)
    pk = s["pk"].float().view(P, KV, D).permute(1, 2, 0)[None].expand(B, KV, D, P)
    pv = s["pvt"].float().permute(0, 2, 1)[None].expand(B, KV, P, D)
    logits = torch.cat([torch.matmul(q, pk), torch.matmul(q, k)], -1)
    see = kok[:, None, :].expand(B, Q, K)
    if c["causal"]:
        last = torch.arange(Q, device=q.device)[None] + (s["k_len"] - s["q_len"])[:, None]
        see = see & (torch.arange(K, device=q.device)[None, None] <= last[..., None])
    see = torch.cat([torch.ones((B, Q, P), dtype=torch.bool, device=q.device), see], -1)
    see = see[:, None, None].expand(B, 1, G, Q, P + K).reshape(B, 1, G * Q, P + K)
    ctx = _softmax_v(logits, see, torch.cat([pv, v], 2))
    return _scatter(s, ctx.view(B, KV, G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, H * D), qrow, qok)


def _quantized(x):
    """8-bit values of the last axis (as floats) and their scale: amax / 127, ties to even."""
    amax = x.abs().amax(-1, keepdim=True)
    some = amax > 0
    inv = torch.where(some, torch.full_like(amax, 127.0) / torch.where(some, amax, torch.ones_like(amax)), torch.ones_like(amax))
    return torch.round(x * inv).clamp(-128, 127), torch.where(some, amax * INV127, torch.ones_like(amax)).squeeze(-1)


def _bounds(s):
    """Largest and smallest key value per block, kv head and dim, in 8 bits, and the scale of both."""
    c = s["c"]
    KV, D, B = c["kv"], c["d"], c["batch"]
    NB = -(-s["max_k"] // BLOCK)
    row, ok = _padded(s["k_start"], s["k_len"], NB * BLOCK, s["k"].shape[0])
    k = s["k"][row].view(B, NB, BLOCK, KV, D)
    ok = ok.view(B, NB, BLOCK, 1, 1)
    hi = torch.where(ok, k, torch.full_like(k, -math.inf)).amax(2).float()
    lo = torch.where(ok, k, torch.full_like(k, math.inf)).amin(2).float()
    some = ok.any(2)
    q, scale = _quantized(torch.where(some, torch.cat([hi, lo], -1), torch.zeros(1, device=k.device)))
    return q.to(torch.int8), scale


def _select(s, bounds):
    c = s["c"]
    H, KV, D, B, qb = c["heads"], c["kv"], c["d"], c["batch"], c["q_block"]
    G, NQ, NB = H // KV, -(-s["max_q"] // c["q_block"]), -(-s["max_k"] // BLOCK)
    dev = s["q"].device
    row, ok = _padded(s["q_start"], s["q_len"], NQ * qb, s["q"].shape[0])
    q8, qs = _quantized(s["q"].float()[row].view(B, NQ * qb, KV, G, D))
    both = torch.cat([q8.clamp(min=0), q8.clamp(max=0)], -1).permute(0, 2, 1, 3, 4).reshape(B, KV, NQ * qb * G, 2 * D)
    b8 = bounds[0].float().permute(0, 2, 3, 1)
    score = torch.matmul(both, b8).view(B, KV, NQ * qb, G, NB) * qs.permute(0, 2, 1, 3)[..., None]
    blk = torch.arange(NB, device=dev)
    off = (s["k_len"] - s["q_len"])[:, None]
    at = torch.arange(NQ * qb, device=dev)[None] + off  # each query's place among the keys
    see = ok[..., None] & (blk * BLOCK < s["k_len"][:, None, None])
    if c["causal"]:
        see = see & (blk * BLOCK <= at[..., None])
    score = score.amax(3).masked_fill_(~see[:, None], -math.inf).view(B, KV, NQ, qb, NB).amax(3)
    score = score * bounds[1].permute(0, 2, 1)[:, :, None]
    see = see.view(B, NQ, qb, NB).any(2)
    first = torch.arange(NQ, device=dev)[None] * qb
    lo = first + off
    hi = torch.minimum(first + qb, s["q_len"][:, None]) - 1 + off
    w = c["n_local"]
    near = (blk >= (lo // BLOCK - (w - 1))[..., None]) & (blk <= (hi // BLOCK + (0 if c["causal"] else w - 1))[..., None]) & (w > 0)
    must = (blk < c["n_first"]) | near
    score = torch.where(see[:, None], score.masked_fill_(must[:, None], math.inf), torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :c["n_sel"]]
    got = torch.gather(see[:, None].expand_as(score), -1, order)
    order = torch.sort(torch.where(got, order, torch.full_like(order, NB)), dim=-1).values
    sel = torch.where(order < NB, order, torch.full_like(order, -1)).permute(0, 2, 1, 3).int()
    return torch.nn.functional.pad(sel, (0, c["n_sel"] - sel.shape[-1]), value=-1)


def _blocks(s):
    c = s["c"]
    H, KV, D, B, qb = c["heads"], c["kv"], c["d"], c["batch"], c["q_block"]
    G, NQ = H // KV, -(-s["max_q"] // c["q_block"])
    dev = s["q"].device
    sel = _select(s, s["bounds"] if c["kept"] else _bounds(s))
    row, ok = _padded(s["q_start"], s["q_len"], NQ * qb, s["q"].shape[0])
    q = s["q"].float()[row].view(B, NQ, qb, KV, G, D).permute(0, 1, 3, 4, 2, 5).reshape(B, NQ, KV, G * qb, D) * D ** -0.5
    key = (sel.long()[..., None] * BLOCK + torch.arange(BLOCK, device=dev)).flatten(-2)  # [B, NQ, KV, n]
    see = (key >= 0) & (key < s["k_len"][:, None, None, None])
    at = (key + s["k_start"][:, None, None, None]).clamp(0, s["k"].shape[0] - 1)
    head = torch.arange(KV, device=dev)[None, None, :, None]
    k = s["k"].view(-1, KV, D)[at, head].float()
    v = s["vt"].permute(2, 0, 1)[at, head].float()
    see = see[:, :, :, None, :]
    if c["causal"]:
        last = torch.arange(NQ * qb, device=dev).view(1, NQ, qb) + (s["k_len"] - s["q_len"])[:, None, None]
        see = see & (key[:, :, :, None, :] <= last[:, :, None, :, None])
        see = see[:, :, :, None].expand(B, NQ, KV, G, qb, key.shape[-1]).reshape(B, NQ, KV, G * qb, key.shape[-1])
    ctx = _softmax_v(torch.matmul(q, k.transpose(-1, -2)), see, v)
    ctx = ctx.view(B, NQ, KV, G, qb, D).permute(0, 1, 4, 2, 3, 5).reshape(B, NQ * qb, H * D)
    return {"sel": sel, "ctx": _scatter(s, ctx, row, ok)}


def _lib():
    global _e2mi
    if _e2mi is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "e2.c_amd"))
        import e2mi
        _e2mi = e2mi
    return _e2mi


def run(s):
    c = s["c"]
    if not own:
        return {"rope": _rope, "prefix": _prefix, "blocks": _blocks}[c["op"]](s)
    m = _lib()
    H, KV = c["heads"], c["kv"]
    if c["op"] == "rope":
        return m.rope(s["q"], s["k"], s["pos"], s["freqs"], H, KV, layout=c["layout"], inverse=c["inverse"])
    scale = c["d"] ** -0.5
    if c["op"] == "prefix":
        return m.attention_prefix(s["q"], s["k"], s["vt"], s["pk"], s["pvt"], s["q_start"], s["q_len"], s["max_q"], H, KV,
                                  k_start=s["k_start"], k_len=s["k_len"], max_k=s["max_k"], scale=scale,
                                  causal=c["causal"], ctx=s["ctx"])
    bounds = s["bounds"] if c["kept"] else m.block_bounds(s["k"], s["k_start"], s["k_len"], s["max_k"], KV)
    sel = m.block_select(s["q"], bounds, s["q_start"], s["q_len"], s["k_len"], s["max_q"], s["max_k"], H, KV,
                         c["q_block"], c["n_sel"], n_first=c["n_first"], n_local=c["n_local"], causal=c["causal"])
    ctx = m.attention_blocks(s["q"], s["k"], s["vt"], sel, s["q_start"], s["q_len"], s["k_start"], s["k_len"],
                             s["max_q"], s["max_k"], H, KV, c["q_block"], scale=scale, causal=c["causal"], ctx=s["ctx"])
    return {"sel": sel, "ctx": ctx}


# ---- the same from the definitions, in 64 bits, a sequence and a head at a time

def _exact_rope(s):
    c = s["c"]
    rot, D = c["rot"], c["d"]
    half = rot // 2
    i = torch.arange(half, device=s["q"].device)
    lo, hi = (i, i + half) if c["layout"] == "half" else (2 * i, 2 * i + 1)
    z = torch.polar(torch.ones((), dtype=torch.float64, device=i.device),
                    (-1.0 if c["inverse"] else 1.0) * s["freqs"][None] * s["pos"][:, None].double())

    def of(x):
        y = x.double().reshape(x.shape[0], -1, D)
        for h in range(y.shape[1]):
            w = torch.complex(y[:, h, lo], y[:, h, hi]) * z
            y[:, h, lo], y[:, h, hi] = w.real, w.imag
        return y.reshape(x.shape)

    return of(s["q"]), of(s["k"])


def _exact_row_block(q, k, v, see):
    """softmax(q k^T) v over the keys that `see` leaves, in 64 bits; zero where it leaves none."""
    x = (q @ k.T).masked_fill(~see, -math.inf)
    some = see.any(-1, keepdim=True)
    w = torch.exp(x - x.max(-1, keepdim=True).values.masked_fill(~some, 0.0))
    return (w @ v) / w.sum(-1, keepdim=True).masked_fill(~some, 1.0)


def _exact_prefix(s):
    c = s["c"]
    H, KV, D, P = c["heads"], c["kv"], c["d"], c["prefix"]
    out = torch.zeros(s["ctx"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (nq, nk) in enumerate(zip(*_lens(c))):
        q0, k0 = int(s["q_start"][b]), int(s["k_start"][b])
        j = torch.arange(P + nk, device=out.device)
        last = torch.arange(nq, device=out.device) + (nk - nq if c["causal"] else nk) + P
        see = j[None] <= last[:, None]
        for h in range(H):
            a = h // (H // KV)
            k = torch.cat([s["pk"][:, a * D:(a + 1) * D], s["k"][k0:k0 + nk, a * D:(a + 1) * D]]).double()
            v = torch.cat([s["pvt"][a], s["vt"][a, :, k0:k0 + nk]], 1).double().T
            q = s["q"][q0:q0 + nq, h * D:(h + 1) * D].double() / math.sqrt(D)
            out[q0:q0 + nq, h * D:(h + 1) * D] = _exact_row_block(q, k, v, see)
    return out


def _bytes_of(x):
    """The quantizer by its definition: 32-bit scale and reciprocal, rounded to even; whole numbers in 64 bits."""
    top = x.double().abs().max(-1).values.float()
    one = torch.ones_like(top)
    inv = torch.where(top > 0, (torch.full_like(one, 127.0).double() / top.double()).float(), one)
    sc = torch.where(top > 0, (top.double() * INV127).float(), one)
    return torch.round((x.double() * inv.double()[..., None]).float()).double(), sc


def _exact_blocks(s):
    c = s["c"]
    H, KV, D, qb, n_sel = c["heads"], c["kv"], c["d"], c["q_block"], c["n_sel"]
    G = H // KV
    dev = s["q"].device
    out = torch.zeros(s["ctx"].shape, dtype=torch.float64, device=dev)
    NQ = -(-s["max_q"] // qb)
    sel = torch.full((c["batch"], NQ, KV, n_sel), -1, dtype=torch.int32)
    for b, (nq, nk) in enumerate(zip(*_lens(c))):
        q0, k0, nb = int(s["q_start"][b]), int(s["k_start"][b]), -(-nk // BLOCK)
        for a in range(KV):
            k = s["k"][k0:k0 + nk, a * D:(a + 1) * D]
            edge = torch.nn.functional.pad(k, (0, 0, 0, nb * BLOCK - nk), value=math.nan).view(nb, BLOCK, D).float()
            hi, lo = edge.nan_to_num(nan=-math.inf).amax(1), edge.nan_to_num(nan=math.inf).amin(1)
            b8, bs = _bytes_of(torch.cat([hi, lo], 1))
            q = s["q"][q0:q0 + nq].view(nq, H, D)[:, a * G:(a + 1) * G]
            q8, qs = _bytes_of(q)
            up, down = q8.clamp(min=0), q8.clamp(max=0)
            dots = (up @ b8[:, :D].T + down @ b8[:, D:].T)  # [nq, G, nb], whole numbers
            score = (dots * qs.double()[..., None]).float().amax(1)
            place = torch.arange(nq, device=dev) + nk - nq
            far = place if c["causal"] else torch.full_like(place, nk - 1)
            blk = torch.arange(nb, device=dev)
            score = score.masked_fill(blk[None] * BLOCK > far[:, None], -math.inf)
            for i in range(0, nq, qb):
                n = min(qb, nq - i)
                sc = (score[i:i + n].amax(0).double() * bs.double()).float()
                can = blk * BLOCK <= far[i + n - 1]
                must = blk < c["n_first"]
                if c["n_local"]:
                    w = c["n_local"] - 1
                    must = must | ((blk >= place[i] // BLOCK - w) & (blk <= place[i + n - 1] // BLOCK + (0 if c["causal"] else w)))
                sc = sc.masked_fill(must, math.inf)
                left = torch.nonzero(can).flatten()
                pick = left[torch.sort(sc[left], descending=True, stable=True).indices[:n_sel]].sort().values
                sel[b, i // qb, a, :pick.numel()] = pick.int().cpu()
                key = (pick[:, None] * BLOCK + torch.arange(BLOCK, device=dev)).flatten()
                key = key[key < nk]
                see = (key[None] <= far[i:i + n, None]).repeat_interleave(G, 0)
                rows = q[i:i + n].reshape(n * G, D).double() / math.sqrt(D)
                ctx = _exact_row_block(rows, k[key].double(), s["vt"][a][:, k0 + key].double().T, see)
                out[q0 + i:q0 + i + n, a * G * D:(a + 1) * G * D] = ctx.reshape(n, G * D)
    return {"sel": sel, "ctx": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "prefix": _exact_prefix, "blocks": _exact_blocks}[case["op"]](s)
