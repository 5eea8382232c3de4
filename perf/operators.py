"""The operators around a paged per-head KV cache held in TurboQuant codes: coding new tokens into its pages, attending
it, keeping it within a budget, and the attention over the prompts that fill it.

A case names one operator (`op`) and its sizes.  Where `own` is false run() computes them in elementary torch
operations, in fp32; where it is true it makes the calls of aetherkv.paged and aetherkv.prompt.  Inputs come from the
seed alone.  Keys and values are coded as PolarQuant codes them: per vector, the signs `diag`, a Walsh-Hadamard
transform, one absmax scale, 8- or 4-bit codes (the even element in the low nibble).  Heads are 12 x 128, the
framework's own, with as many or fewer KV heads, and generic others.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"
PKG = str(Path(__file__).resolve().parent.parent / "deepseek-v4-codebase_amd")


def listed():
    return [
        # a decode step of 64 sequences: one token each goes into the cache (latency: once per layer and token)
        dict(name="append_step_64", op="append", batch=64, tokens=1, packed=False, kv_heads=4, dim=128, bits=4, dtype="bf16", page=64, track=True),
        # eight prompts of different lengths go into the cache at once, every head with its own K and V
        dict(name="append_prompts", op="append", batch=8, tokens=8192, packed=True, kv_heads=12, dim=128, bits=4, dtype="bf16", page=64, track=False),
        # one interactive sequence shortly after its prompt
        dict(name="attend_one_short", op="attend", batch=1, tokens=1, heads=12, kv_heads=4, dim=128, bits=4, dtype="bf16", page=64, length=333, ragged=False, sink=False, track=False),
        # a full batch's decode step, contexts of different lengths, weights kept for eviction
        dict(name="attend_batch_64", op="attend", batch=64, tokens=1, heads=12, kv_heads=4, dim=128, bits=4, dtype="bf16", page=64, length=16384, ragged=True, sink=False, track=True),
        # one sequence at 262144 tokens, a KV head for every query head, with a sink
        dict(name="attend_one_262k", op="attend", batch=1, tokens=1, heads=12, kv_heads=12, dim=128, bits=4, dtype="bf16", page=256, length=262144, ragged=False, sink=True, track=False),
        # the last 16 tokens of eight prompts look back, for their weights (before a first eviction); 8 bits, narrow heads
        dict(name="attend_observe_16", op="attend", batch=8, tokens=16, heads=16, kv_heads=2, dim=64, bits=8, dtype="f16", page=16, length=5001, ragged=True, sink=False, track=True),
        # 16 sequences brought back to their budget of 1024 after 64 more tokens
        dict(name="evict_step_16", op="evict", batch=16, kv_heads=4, dim=128, bits=4, page=64, length=1088, keep=1024, first=4, recent=128),
        # eight long prompts cut to a quarter
        dict(name="evict_prompts", op="evict", batch=8, kv_heads=12, dim=128, bits=8, page=64, length=16384, keep=4096, first=4, recent=512),
        # one short prompt (latency)
        dict(name="prompt_short", op="prompt", batch=1, length=77, prefix=0, heads=12, kv_heads=4, dim=128, dtype="bf16", ragged=False, sink=False, lse=False, pad=0),
        # later chunks of three prompts over the keys that are there, narrow heads, with the sums for a merge
        dict(name="prompt_chunk", op="prompt", batch=3, length=512, prefix=3501, heads=16, kv_heads=2, dim=64, dtype="f16", ragged=True, sink=False, lse=True, pad=0),
        # a batch of prompts packed into one buffer, its end unused
        dict(name="prompt_packed_16", op="prompt", batch=16, length=2048, prefix=0, heads=12, kv_heads=4, dim=128, dtype="bf16", ragged=True, sink=True, lse=False, pad=61),
        # one long prompt
        dict(name="prompt_long", op="prompt", batch=1, length=16384, prefix=0, heads=12, kv_heads=4, dim=128, dtype="bf16", ragged=False, sink=False, lse=False, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "prompt", "prompt"])
    dim, bits, dtype = rng.choice([64, 128]), rng.choice([4, 8]), rng.choice(["bf16", "f16"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 6, 8, 12])
    batch = _log(rng, 1, 64)
    if op == "append":
        packed = rng.random() < 0.5
        tokens = _log(rng, 1, max(1, 300000 // (batch * kv_heads))) if packed else _log(rng, 1, 16)
        return dict(op=op, batch=batch, tokens=tokens, packed=packed, kv_heads=kv_heads, dim=dim, bits=bits, dtype=dtype, page=page, track=rng.random() < 0.5)
    if op == "attend":
        tokens = rng.choice([1, 1, 1, 2, 4, 5, 16])
        length = _log(rng, tokens, max(tokens, min(131072, 2500000 // (batch * kv_heads))))
        return dict(op=op, batch=batch, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, bits=bits, dtype=dtype, page=page, length=length,
                    ragged=rng.random() < 0.6, sink=rng.random() < 0.4, track=rng.random() < 0.5)
    if op == "evict":
        length = _log(rng, 40, max(40, min(65536, 1500000 // (batch * kv_heads))))
        keep = max(20, int(length * rng.uniform(0.1, 0.98)))
        return dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, bits=bits, page=page, length=length, keep=keep, first=rng.choice([0, 1, 4]), recent=rng.randint(0, keep // 2))
    batch = _log(rng, 1, 16)
    heads = kv_heads * group if kv_heads * group <= 32 else kv_heads
    length = _log(rng, 1, max(1, min(8192, int(math.sqrt(1.5e9 / (batch * heads))))))
    prefix = rng.choice([0, 0, 1, rng.randint(2, 2000)])
    return dict(op=op, batch=batch, length=length, prefix=prefix, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, ragged=rng.random() < 0.6, sink=rng.random() < 0.3,
                lse=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 37]))


def _lengths(case, longest, ragged, least=1):
    """One length for each sequence, by the case alone: the first is the longest, the others spread below it."""
    if not ragged:
        return [longest] * case["batch"]
    rng = random.Random("%s %s %s" % (case["batch"], longest, least))
    return [longest] + [max(least, int(longest * rng.uniform(0.05, 1.0))) for _ in range(case["batch"] - 1)]


def _row_bytes(case):
    return case["dim"] * case["bits"] // 8


def work(case):
    op, d = case["op"], case["dim"]
    if op == "append":
        n = sum(_lengths(case, case["tokens"], case["packed"])) * case["kv_heads"]
        return {"bytes": n * 2 * (2 * d + _row_bytes(case) + 4) + (8 * n if case["track"] else 0), "flops": n * 2 * d * (math.log2(d) + 4)}
    if op == "attend":
        n, t = sum(_lengths(case, case["length"], case["ragged"], case["tokens"])), case["tokens"]
        rows = case["batch"] * t * case["heads"]
        return {"bytes": n * case["kv_heads"] * (2 * (_row_bytes(case) + 4) + (8 if case["track"] else 0)) + 4 * rows * d, "flops": 4.0 * t * case["heads"] * d * n}
    if op == "evict":
        n = case["batch"] * case["kv_heads"]
        moved = min(case["keep"], case["length"] - case["keep"]) * case["keep"] / max(1, case["length"])  # about: evicted ones below the budget
        return {"bytes": n * (8 * case["length"] + moved * 2 * (2 * (_row_bytes(case) + 4) + 8)), "flops": n * case["length"]}
    lq = _lengths(case, case["length"], case["ragged"])
    pairs = sum(x * (x + 1) / 2 + x * case["prefix"] for x in lq)
    nq, nk = sum(lq), sum(lq) + case["prefix"] * case["batch"]
    return {"bytes": 2 * d * (2 * nq * case["heads"] + 2 * nk * case["kv_heads"]) + (4 * nq * case["heads"] if case["lse"] else 0), "flops": 4.0 * case["heads"] * d * pairs}


def _signs(dim):
    """PolarQuant(seed=42)'s diagonal."""
    g = torch.Generator().manual_seed(42 * 10007 + dim)
    return torch.where(torch.rand(dim, generator=g) > 0.5, 1.0, -1.0)


def _hadamard(dim):
    h = torch.ones(1, 1)
    while h.size(0) < dim:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h


def _offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def _codes(gen, shape, bits):
    """Codes as coded Gaussian entries have them: the rotated values over their largest, in steps of it / 7 or 127."""
    v = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    if bits == 8:
        return (v * 42).round_().clamp_(-127, 127).to(torch.int8)
    v = (v * 2.4).round_().clamp_(-7, 7).to(torch.int8)
    return ((v[..., 0::2] & 15) | ((v[..., 1::2] & 15) << 4)).view(torch.uint8)


def _scales(gen, shape, bits, at):
    return torch.randn(shape, generator=gen, device=DEV).mul_(0.3).exp_().mul_(at / (7 if bits == 4 else 127))


def _table(gen, batch, slots, page):
    """Pages in no order, no page in two sequences, two pages of the pool unused."""
    per = max(1, -(-slots // page))
    return torch.randperm(batch * per + 2, generator=gen, device=DEV)[:batch * per].to(torch.int32).view(batch, per), batch * per + 2


def _cache(gen, case, slots):
    b, h, page, bits = case["batch"], case["kv_heads"], case["page"], case["bits"]
    table, pool = _table(gen, b, slots, page)
    at = 2.9  # the largest of a rotated vector of unit variance
    s = dict(table=table, capacity=table.size(1) * page, cache=None)
    for x in "kv":
        s[x + "_codes"] = _codes(gen, (pool, h, page, case["dim"]), bits)
        s[x + "_scale"] = _scales(gen, (pool, h, page), bits, at)
    return s


def _tracker(s, case):
    """Per sequence, KV head and slot: the accumulated weight (first half) and the token that the slot holds (second half)."""
    s["slots"] = torch.zeros(2, case["batch"], case["kv_heads"], s["capacity"], dtype=torch.int32, device=DEV)
    return s["slots"][0].view(torch.float32), s["slots"][1]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, b, d = case["op"], case["batch"], case["dim"]
    s = dict(case=case, signs=_signs(d).to(DEV), hadamard=_hadamard(d).to(DEV))
    if op == "append":
        lens = _lengths(case, case["tokens"], case["packed"])
        n, h, dt = sum(lens), case["kv_heads"], DT[case["dtype"]]
        before = [0 if case["packed"] else 5 + 37 * i for i in range(b)]
        # K and V as a projection leaves them, side by side in a row; 2% of K's channels are large
        kv = torch.randn(n, 2, h * d, generator=gen, device=DEV)
        kv[:, 0, torch.randperm(h * d, generator=gen, device=DEV)[:max(1, h * d // 50)]] *= 8
        kv = kv.to(dt)
        s["k"], s["v"] = kv[:, 0].view(n, h, d), kv[:, 1].view(n, h, d)
        s["cu"] = _offsets(lens).to(DEV)
        if not case["packed"]:
            s["k"], s["v"] = s["k"].unflatten(0, (b, case["tokens"])), s["v"].unflatten(0, (b, case["tokens"]))
        s["start"] = torch.tensor(before, dtype=torch.int32, device=DEV)
        s["table"], pool = _table(gen, b, max(x + y for x, y in zip(lens, before)), case["page"])
        s["capacity"], s["cache"] = s["table"].size(1) * case["page"], None
        for x in "kv":
            s[x + "_codes"] = torch.zeros(pool, h, case["page"], _row_bytes(case), dtype=torch.int8 if case["bits"] == 8 else torch.uint8, device=DEV)
            s[x + "_scale"] = torch.zeros(pool, h, case["page"], device=DEV)
        s["token"] = s["start"] + 1000
        if case["track"]:
            _tracker(s, case)[0].fill_(1.5)
        return s
    if op == "attend":
        lens = _lengths(case, case["length"], case["ragged"], case["tokens"])
        s |= _cache(gen, case, max(lens))
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = torch.randn(b, case["tokens"], case["heads"], d, generator=gen, device=DEV).mul_(1.5).to(DT[case["dtype"]])
        s["sink"] = torch.randn(case["heads"], generator=gen, device=DEV) if case["sink"] else None
        if case["track"]:  # the weights of some hundred steps before this one
            _tracker(s, case)[0].copy_(torch.randn(b, case["kv_heads"], s["capacity"], generator=gen, device=DEV).mul_(1.5).exp_().mul_(0.02))
        return s
    if op == "evict":
        s |= _cache(gen, case, case["length"])
        n, keep = case["length"], case["keep"]
        # one sequence in five is still within the budget
        s["lengths"] = torch.tensor([n if i % 5 < 4 else min(n, keep - i % 3) for i in range(b)], dtype=torch.int32, device=DEV)
        s["seen"] = s["lengths"] + 500
        weights, tokens = _tracker(s, case)
        w = torch.randn(weights.shape, generator=gen, device=DEV).mul_(1.5).exp_()
        weights.copy_(torch.where(torch.rand(weights.shape, generator=gen, device=DEV) < 0.05, 0.0, w))
        # slots hold tokens nearly in order: earlier evictions filled holes with later ones
        tokens.copy_((torch.arange(s["capacity"], device=DEV) + torch.rand(tokens.shape, generator=gen, device=DEV) * 40).argsort(-1).argsort(-1) + 500 * (torch.arange(s["capacity"], device=DEV) >= case["first"]))
        s["slots_before"] = s["slots"].clone()
        return s
    lq = _lengths(case, case["length"], case["ragged"])
    lk = [x + case["prefix"] for x in lq]
    h, hk, dt = case["heads"], case["kv_heads"], DT[case["dtype"]]
    nq, nk = sum(lq) + case["pad"], sum(lk) + case["pad"]
    if case["prefix"]:  # a chunk: its queries, and keys and values gathered from before
        s["q"] = torch.randn(nq, h, d, generator=gen, device=DEV).to(dt)
        kv = torch.randn(nk, 2, hk, d, generator=gen, device=DEV).to(dt)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
    else:  # the whole prompt's: one projection's output, heads side by side in a row
        qkv = torch.randn(nq, h + 2 * hk, d, generator=gen, device=DEV).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    s["cu_q"], s["cu_k"], s["most_q"], s["most_k"] = _offsets(lq).to(DEV), _offsets(lk).to(DEV), max(lq), max(lk)
    s["sink"] = torch.randn(h, generator=gen, device=DEV) if case["sink"] else None
    s["out"] = torch.zeros(nq, h, d, dtype=dt, device=DEV)
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------

def _encode(x, signs, bits):
    """PolarQuant.encode: butterflies in its order and roundings, so that the codes are equal bit for bit."""
    d, lead = x.size(-1), x.shape[:-1]
    x = x.float() * signs
    for h in [1 << i for i in range(d.bit_length() - 1)]:
        x = x.reshape(*lead, d // (2 * h), 2, h)
        x = torch.stack([x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]], -2)
    x = x.reshape(*lead, d) * d ** -0.5
    most = 127.0 if bits == 8 else 7.0
    m = x.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    c = (x / m * most).round().clamp(-most, most).to(torch.int8)
    return (c if bits == 8 else ((c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)).view(torch.uint8)), (m / most)[..., 0]


def _values(codes, bits):
    if bits == 8:
        return codes.float()
    c = codes.to(torch.int16)
    return torch.stack([((c & 15) ^ 8) - 8, ((c >> 4) ^ 8) - 8], -1).flatten(-2).float()


def _rows(s, x):
    """[B, Hkv, capacity, D]: K or V of every sequence in fp32, decoded."""
    page = s["table"].long()
    v = _values(s[x + "_codes"][page], s["case"]["bits"]) * s[x + "_scale"][page].unsqueeze(-1)
    v = v.transpose(1, 2).flatten(2, 3)
    return (v @ s["hadamard"]) * (s["signs"] * s["case"]["dim"] ** -0.5)


def _softmax(logits, sink):
    """Weights over the last dimension with the sink [.., 1] counted once; a row of -inf alone gives zeros.  Also log sums."""
    m = logits.amax(-1, keepdim=True)
    m = m if sink is None else torch.maximum(m, sink)
    m = torch.where(m.isinf(), 0.0, m)
    p = torch.exp(logits - m)
    total = p.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - m)
    return p / torch.where(total > 0, total, 1.0), (m + torch.log(total))[..., 0]


def _attend(s):
    c = s["case"]
    b, t, h, hk, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    k, v = _rows(s, "k"), _rows(s, "v")
    q = s["q"].float().view(b, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * t, d)
    logits = (q @ k.transpose(-1, -2)) * d ** -0.5
    seen = s["lengths"][:, None] - t + 1 + torch.arange(t, device=DEV)
    hidden = torch.arange(s["capacity"], device=DEV) >= seen[:, :, None]
    logits = logits.view(b, hk, h // hk, t, -1).masked_fill(hidden[:, None, None], -math.inf)
    p, _ = _softmax(logits, None if s["sink"] is None else s["sink"].view(hk, h // hk, 1, 1))
    if c["track"]:
        s["slots"][0].view(torch.float32).add_(p.sum((2, 3)))
    out = (p.flatten(2, 3) @ v).view(b, hk, h // hk, t, d)
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(s["q"].dtype)


def _append(s):
    k, v = (x.flatten(0, 1) if x.dim() == 4 else x for x in (s["k"], s["v"]))
    n = torch.arange(k.size(0), device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["cu"], n, right=True) - 1
    at = n - s["cu"][b]
    slot = s["start"][b] + at
    page, row = s["table"][b, slot // s["case"]["page"]].long(), slot % s["case"]["page"]
    for x, name in ((k, "k"), (v, "v")):
        codes, scale = _encode(x, s["signs"], s["case"]["bits"])
        s[name + "_codes"][page, :, row] = codes
        s[name + "_scale"][page, :, row] = scale
    if s["case"]["track"]:
        s["slots"][0][b, :, slot] = 0
        s["slots"][1][b, :, slot] = (s["token"][b] + at)[:, None].expand(-1, k.size(1))


def _evict(s):
    c = s["case"]
    weights, tokens = s["slots"][0].view(torch.float32), s["slots"][1]
    b, h, capacity = weights.shape
    keep, slot = c["keep"], torch.arange(capacity, device=DEV)
    there = slot < s["lengths"][:, None, None]
    held = (tokens < c["first"]) | (tokens >= s["seen"][:, None, None] - c["recent"])
    rank = torch.where(there, torch.where(held, math.inf, weights), -math.inf).sort(dim=-1, descending=True, stable=True)[1]
    kept = torch.zeros(weights.shape, dtype=torch.bool, device=DEV).scatter_(-1, rank[..., :keep], True) & there
    hole, mover = there & ~kept & (slot < keep), kept & (slot >= keep)
    most = min(keep, capacity - keep)
    dst = hole.int().sort(dim=-1, descending=True, stable=True)[1][..., :most]
    src = mover.int().sort(dim=-1, descending=True, stable=True)[1][..., :most]
    src = torch.where(torch.arange(most, device=DEV) < hole.sum(-1, keepdim=True), src, dst)
    seq = torch.arange(b, device=DEV)[:, None, None]
    head = torch.arange(h, device=DEV)[None, :, None]
    from_page, to_page = s["table"][seq, src // c["page"]].long(), s["table"][seq, dst // c["page"]].long()
    from_row, to_row = src % c["page"], dst % c["page"]
    for name in ("k_codes", "k_scale", "v_codes", "v_scale"):
        s[name][to_page, head, to_row] = s[name][from_page, head, from_row]
    s["slots"].scatter_(-1, dst.expand(2, -1, -1, -1), s["slots"].gather(-1, src.expand(2, -1, -1, -1)))


def _prompt(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    lq, lk = s["cu_q"].diff(), s["cu_k"].diff()
    iq, ik = torch.arange(s["most_q"], device=DEV), torch.arange(s["most_k"], device=DEV)
    at_q = (s["cu_q"][:-1, None] + iq).clamp(max=s["q"].size(0) - 1)
    at_k = (s["cu_k"][:-1, None] + ik).clamp(max=s["k"].size(0) - 1)
    q = s["q"][at_q].float().unflatten(2, (hk, h // hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (x[at_k].float().transpose(1, 2) for x in (s["k"], s["v"]))
    logits = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(lq.size(0), hk, h // hk, s["most_q"], s["most_k"])
    hidden = (ik > iq[:, None] + (lk - lq)[:, None, None]) | (ik >= lk[:, None, None])
    logits.masked_fill_(hidden[:, None, None], -math.inf)
    p, lse = _softmax(logits, None if s["sink"] is None else s["sink"].view(hk, h // hk, 1, 1))
    out = (p.flatten(2, 3) @ v).view(lq.size(0), h, s["most_q"], d)
    n = torch.arange(s["q"].size(0), device=DEV, dtype=torch.int32)  # back to the packed rows; those past the end stay
    b = (torch.searchsorted(s["cu_q"], n, right=True) - 1).clamp(max=lq.size(0) - 1)
    i = (n - s["cu_q"][b]).clamp(max=s["most_q"] - 1)
    inside = (n < s["cu_q"][-1])[:, None]
    s["out"].copy_(torch.where(inside[:, :, None], out[b, :, i].to(s["out"].dtype), s["out"]))
    return (s["out"], lse.flatten(1, 2)[b, :, i].masked_fill(~inside, -math.inf)) if c["lse"] else s["out"]


# ---- the framework's -----------------------------------------------------------------------------------------------

def _handle(s):
    """The cache as the framework holds it: made from the tensors once, as a program does."""
    if s["cache"] is None:
        from aetherkv import PolarQuant
        from aetherkv.paged import PagedKVCache, SlotTracker

        s["cache"] = PagedKVCache.from_tensors(PolarQuant(s["case"]["bits"]), s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"])
        s["tracker"] = SlotTracker.from_tensor(s["slots"]) if "slots" in s else None
    return s["cache"], s["tracker"]


def _own_append(s):
    from aetherkv.paged import append_tokens

    cache, tracker = _handle(s)
    append_tokens(cache, s["k"], s["v"], s["table"], s["start"], cu_seqlens=s["cu"] if s["case"]["packed"] else None, tracker=tracker, token=s["token"] if tracker is not None else None)


def _own_attend(s):
    from aetherkv.paged import paged_attention

    cache, tracker = _handle(s)
    return paged_attention(s["q"], cache, s["table"], s["lengths"], s["case"]["dim"] ** -0.5, sink=s["sink"], tracker=tracker)


def _own_evict(s):
    from aetherkv.paged import evict_by_weight

    cache, tracker = _handle(s)
    evict_by_weight(cache, s["table"], s["lengths"], tracker, s["seen"], s["case"]["keep"], first=s["case"]["first"], recent=s["case"]["recent"])


def _own_prompt(s):
    from aetherkv.prompt import prompt_attention

    c = s["case"]
    return prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], c["dim"] ** -0.5, cu_seqlens_k=s["cu_k"], sink=s["sink"], return_lse=c["lse"], out=s["out"])


def run(s):
    if own and PKG not in sys.path:
        sys.path.insert(0, PKG)
    op = s["case"]["op"]
    if op == "prompt":
        return _own_prompt(s) if own else _prompt(s)
    held = [s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]]
    if op == "append":
        _own_append(s) if own else _append(s)
        return held + ([s["slots"]] if s["case"]["track"] else [])
    if op == "attend":
        out = _own_attend(s) if own else _attend(s)
        return [out] + ([s["slots"][0].view(torch.float32)] if s["case"]["track"] else [])
    s["slots"].copy_(s["slots_before"])  # moved in place: a pass starts from the same weights
    _own_evict(s) if own else _evict(s)
    return held + [s["slots"][0].view(torch.float32), s["slots"][1]]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _kron(dim):
    w, two = torch.ones(1, 1, dtype=torch.float64, device=DEV), torch.tensor([[1.0, 1.0], [1.0, -1.0]], dtype=torch.float64, device=DEV)
    while w.size(0) < dim:
        w = torch.kron(two, w)
    return w / math.sqrt(dim)


def _exact_rows(s, x, b, head, n):
    """K or V of the first n slots of one sequence and head."""
    c = s["case"]
    slots = torch.arange(n, device=DEV)
    pages = s["table"][b].to(torch.int64)[torch.div(slots, c["page"], rounding_mode="floor")]
    codes = s[x + "_codes"][pages, head, slots % c["page"]].to(torch.int64)
    if c["bits"] == 4:
        low, high = codes % 16, torch.div(codes, 16, rounding_mode="floor")
        codes = torch.empty(n, c["dim"], dtype=torch.int64, device=DEV)
        codes[:, 0::2], codes[:, 1::2] = torch.where(low > 7, low - 16, low), torch.where(high > 7, high - 16, high)
    rotated = codes.double() * s[x + "_scale"][pages, head, slots % c["page"]].double()[:, None]
    return torch.mm(rotated, _kron(c["dim"])) * s["signs"].double()


def _exact_head(q, k, v, first_seen, sink):
    """(out, weights summed over the queries, log sums) of queries [n, D], the i-th of which sees first_seen + i keys, a
    piece of the queries at a time."""
    outs, sums, logs = [], torch.zeros(k.size(0), dtype=torch.float64, device=DEV), []
    for at in range(0, q.size(0), 2048):
        piece = q[at:at + 2048].double()
        e = torch.mm(piece, k.t()) / math.sqrt(k.size(1))
        count = first_seen + at + torch.arange(piece.size(0), device=DEV)
        e = torch.where(torch.arange(k.size(0), device=DEV)[None] < count[:, None], e, torch.full_like(e, -math.inf))
        if sink is not None:
            e = torch.cat([e, sink.double().expand(piece.size(0), 1)], 1)
        top = e.max(1, keepdim=True)[0]
        e = torch.exp(e - torch.where(top == -math.inf, torch.zeros_like(top), top))
        z = e.sum(1, keepdim=True)
        logs.append((top + z.log())[:, 0])
        e = torch.nan_to_num(e / z)[:, :k.size(0)]
        outs.append(torch.mm(e, v))
        sums += e.sum(0)
    return torch.cat(outs), sums, torch.cat(logs)


def _exact_attend(s):
    c = s["case"]
    t, g = c["tokens"], c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], t, c["heads"], c["dim"], dtype=torch.float64, device=DEV)
    weights = s["slots"][0].view(torch.float32).double() if c["track"] else None
    for b, n in enumerate(s["lengths"].tolist()):
        for j in range(c["kv_heads"]):
            k, v = _exact_rows(s, "k", b, j, n), _exact_rows(s, "v", b, j, n)
            for h in range(j * g, j * g + g):
                out[b, :, h], w, _ = _exact_head(s["q"][b, :, h], k, v, n - t + 1, None if s["sink"] is None else s["sink"][h])
                if weights is not None:
                    weights[b, j, :n] += w
    return [out] + ([weights] if c["track"] else [])


def _exact_prompt(s):
    c = s["case"]
    g = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["out"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(c["batch"]):
        for h in range(c["heads"]):
            rows = slice(cq[b], cq[b + 1])
            k, v = (s[x][ck[b]:ck[b + 1], h // g].double() for x in "kv")
            out[rows, h], _, lse[rows, h] = _exact_head(s["q"][rows, h], k, v, ck[b + 1] - ck[b] - (cq[b + 1] - cq[b]) + 1, None if s["sink"] is None else s["sink"][h])
    return [out, lse] if c["lse"] else out


def _exact_append(s):
    """The scales alone: the codes are decided by comparisons of rounded values, and whole."""
    c, outs = s["case"], []
    for name in "kv":
        scale = s[name + "_scale"].double()
        x = s[name].reshape(-1, c["kv_heads"], c["dim"]).double() * s["signs"].double()
        m = torch.mm(x.reshape(-1, c["dim"]), _kron(c["dim"])).abs().max(1)[0].view(-1, c["kv_heads"])
        m = torch.clamp(m, min=1e-8) / (127 if c["bits"] == 8 else 7)
        cu = s["cu"].tolist()
        for b, start in enumerate(s["start"].tolist()):
            slots = start + torch.arange(cu[b + 1] - cu[b], device=DEV)
            scale[s["table"][b].to(torch.int64)[slots // c["page"]], :, slots % c["page"]] = m[cu[b]:cu[b + 1]]
        outs += [None, scale]
    return outs + ([None] if c["track"] else [])


def _exact_evict(s):
    """The scales and weights, row by row: nothing is computed, values move."""
    c, page = s["case"], s["case"]["page"]
    weights, scales = s["slots"][0].view(torch.float32).double(), [s["k_scale"].double(), s["v_scale"].double()]
    lengths, seen, tables = s["lengths"].tolist(), s["seen"].tolist(), s["table"].to(torch.int64)
    for b in range(c["batch"]):
        n = lengths[b]
        if n <= c["keep"]:
            continue
        for h in range(c["kv_heads"]):
            token, w = s["slots"][1][b, h, :n].tolist(), weights[b, h, :n].tolist()
            order = sorted(range(n), key=lambda i: (not (token[i] < c["first"] or token[i] >= seen[b] - c["recent"]), -w[i], i))
            stays = set(order[:c["keep"]])
            holes = [i for i in range(c["keep"]) if i not in stays]
            movers = sorted(i for i in stays if i >= c["keep"])
            holes, movers = torch.tensor(holes, dtype=torch.int64, device=DEV), torch.tensor(movers, dtype=torch.int64, device=DEV)
            for x in scales:
                x[tables[b, holes // page], h, holes % page] = x[tables[b, movers // page], h, movers % page]
            weights[b, h, holes] = weights[b, h, movers]
    return [None, scales[0], None, scales[1], weights, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "prompt":
        return _exact_prompt(s)
    return _exact_evict(s)
