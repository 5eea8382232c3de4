"""Operators around per-head caches: rotary positions on several axes, attention over an encoder's states, and the life of
a cache's pages (given, shared by forks, copied on write, released, compacted).

A case names one operator (`op`) and its sizes.  Where `own` is false run() computes them in elementary torch
operations, in fp32 (angles in fp64); where it is true it makes the calls of aetherkv.rotary, aetherkv.cross and
aetherkv.pages.  Inputs come from the seed alone.  Heads are 12 x 128, the framework's own, with as many or fewer KV heads,
and generic others; pages hold codes of 28 layers' caches, the framework's own depth, or of fewer.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"
PKG = str(Path(__file__).resolve().parent.parent / "deepseek-v4-codebase_amd")


def listed():
    return [
        # a decode step: one token of each of 64 sequences, somewhere in a long context (latency: once per layer and token)
        dict(name="rotate_step_64", op="rotate", tokens=64, heads=12, kv_heads=4, dim=128, rope=128, pairs="halves", axes=3, dtype="bf16", far=262144),
        # a long prompt of text and images, q and k as one projection leaves them; half of each head is rotated
        dict(name="rotate_prompt", op="rotate", tokens=32768, heads=12, kv_heads=4, dim=128, rope=64, pairs="adjacent", axes=3, dtype="bf16", far=1000),
        # an image encoder in fp32, rows and columns alone, an odd number of patches
        dict(name="rotate_patches", op="rotate", tokens=5003, heads=16, kv_heads=16, dim=64, rope=48, pairs="halves", axes=2, dtype="f32", far=0),
        # one interactive sequence's new token over one encoder input of 1500 frames
        dict(name="cross_one", op="cross", batch=1, tokens=1, ragged=False, states=1, states_length=1500, heads=12, kv_heads=4, dim=128, dtype="bf16", sink=False, lse=False),
        # a full batch's decode step, every sequence with encoder states of its own, of different lengths
        dict(name="cross_step_64", op="cross", batch=64, tokens=1, ragged=False, states=64, states_length=4096, heads=12, kv_heads=4, dim=128, dtype="bf16", sink=False, lse=False),
        # eight inputs with eight answers (or beams) each: sequences share their encoder states; every head its own K and V
        dict(name="cross_beams", op="cross", batch=64, tokens=1, ragged=False, states=8, states_length=2999, heads=16, kv_heads=16, dim=64, dtype="f16", sink=True, lse=False),
        # prompts of different lengths over states of different lengths, with the sums for a merge
        dict(name="cross_prompts", op="cross", batch=16, tokens=512, ragged=True, states=16, states_length=2048, heads=16, kv_heads=2, dim=64, dtype="f16", sink=False, lse=True),
        # one long document over another
        dict(name="cross_long", op="cross", batch=1, tokens=8192, ragged=False, states=1, states_length=16384, heads=12, kv_heads=4, dim=128, dtype="bf16", sink=False, lse=False),
        # a decode step of 64 sequences, in pairs that were forked just before: room for one token each (latency)
        dict(name="pages_step_64", op="reserve", batch=64, share=2, length=500, tokens=1, whole=False, layers=28, kv_heads=4, dim=128, bits=4, page=64),
        # 16 beams are reordered and take their next token
        dict(name="pages_beams_16", op="fork", batch=16, share=16, length=2001, tokens=1, whole=False, layers=28, kv_heads=4, dim=128, bits=4, page=64),
        # eight answers to one prompt get pages of their own, before they evict by weight
        dict(name="pages_own_8", op="reserve", batch=8, share=8, length=4100, tokens=64, whole=True, layers=28, kv_heads=4, dim=128, bits=4, page=64),
        # half of a batch has ended: its pages are released, the rest move to the pool's low end
        dict(name="pages_compact", op="compact", batch=32, share=1, length=4096, tokens=0, whole=False, layers=28, kv_heads=4, dim=128, bits=4, page=64),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "cross", "cross", "cross", "reserve", "fork", "compact"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 12])
    heads = heads if heads <= 32 else kv_heads
    if op == "rotate":
        dim = rng.choice([64, 80, 128, 256])
        tokens = _log(rng, 1, 60000000 // ((heads + kv_heads) * dim))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rope=rng.choice([dim, dim // 2, dim * 3 // 4 // 8 * 8]), pairs=rng.choice(["adjacent", "halves"]),
                    axes=rng.choice([1, 2, 3]), dtype=rng.choice(["bf16", "f16", "f32"]), far=_log(rng, 1, 1000000))
    if op == "cross":
        batch = _log(rng, 1, 64)
        states = batch if rng.random() < 0.6 else rng.randint(1, batch)
        length = _log(rng, 1, min(16384, 8000000 // (states * kv_heads)))
        tokens = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, min(4096, int(1.0e9 / (batch * heads * length)))))
        return dict(op=op, batch=batch, tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7, states=states, states_length=length, heads=heads, kv_heads=kv_heads, dim=dim,
                    dtype=rng.choice(["bf16", "f16"]), sink=rng.random() < 0.3, lse=rng.random() < 0.5)
    bits, page = rng.choice([4, 8]), rng.choice([16, 32, 64, 128, 256])
    batch = _log(rng, 1, 64)
    share = 1 if op == "compact" else rng.choice([2, 4, batch]) if op == "fork" else rng.choice([1, 2, 4, batch])
    length = _log(rng, 1, min(32768, 100000 // batch))
    token_bytes = 2 * kv_heads * (dim * bits // 8 + 4)
    layers = max(1, min(28, int(4.0e8 / (token_bytes * batch * (length + 2 * page)))))
    return dict(op=op, batch=batch, share=share, length=length, tokens=0 if op == "compact" else rng.choice([1, 1, 2, 16, 100]), whole=op == "reserve" and rng.random() < 0.3,
                layers=layers, kv_heads=kv_heads, dim=dim, bits=bits, page=page)


def _lengths(case, count, longest, ragged, least=1):
    """`count` lengths, by the case alone: the first is the longest, the others spread below it."""
    if not ragged:
        return [longest] * count
    rng = random.Random("%s %s %s" % (count, longest, least))
    return [longest] + [max(least, int(longest * rng.uniform(0.05, 1.0))) for _ in range(count - 1)]


def _state_lengths(case):
    return _lengths(case, case["states"], case["states_length"], True)


def _reads(case):
    """The states that each sequence reads: its own, or shared ones in turn."""
    return [b * case["states"] // case["batch"] for b in range(case["batch"])]


def _families(case):
    """The filled length of every sequence: those that share a prompt are equally long."""
    lens = _lengths(case, -(-case["batch"] // case["share"]), case["length"], True)
    return [lens[b // case["share"]] for b in range(case["batch"])]


def _page_bytes(case):
    return case["layers"] * 2 * case["kv_heads"] * case["page"] * (case["dim"] * case["bits"] // 8 + 4)


def work(case):
    op = case["op"]
    if op == "rotate":
        n, d = case["tokens"] * (case["heads"] + case["kv_heads"]), case["dim"]
        return {"bytes": n * d * 2 * (4 if case["dtype"] == "f32" else 2) + 4 * case["axes"] * case["tokens"], "flops": 3.0 * n * case["rope"] + 40.0 * case["tokens"] * case["rope"]}
    if op == "cross":
        lq, lk, reads = _lengths(case, case["batch"], case["tokens"], case["ragged"]), _state_lengths(case), _reads(case)
        keys = sum(lk[e] for e in set(reads))
        rows = sum(lq) * case["heads"]
        return {"bytes": 2 * case["dim"] * (2 * rows + 2 * keys * case["kv_heads"]) + (4 * rows if case["lse"] else 0),
                "flops": 4.0 * case["heads"] * case["dim"] * sum(a * lk[e] for a, e in zip(lq, reads))}
    lens, page = _families(case), case["page"]
    entries = sum(-(-(n + case["tokens"]) // page) for n in lens)
    if op == "reserve":
        first = [case["share"] * i == b for b, i in ((b, b // case["share"]) for b in range(case["batch"]))]
        copies = sum(0 if f else -(-n // page) if case["whole"] else int(n % page > 0) for n, f in zip(lens, first))
        touched = entries if case["whole"] else case["batch"] * (1 + case["tokens"] // page)
    elif op == "fork":  # every family's members pick a parent among themselves: parents' first children need no copy
        sizes = [min(case["share"], case["batch"] - at) for at in range(0, case["batch"], case["share"])]
        copies = sum(s * (1.0 - 1.0 / s) ** s if lens[at * case["share"]] % page else 0.0 for at, s in enumerate(sizes))
        touched = 3 * entries
    else:  # live pages are spread evenly over the pool: those past the live ones' number move
        left = sum(-(-n // page) for b, n in enumerate(lens) if b % 2)
        pool = _pool_pages(case)
        copies = left * (1.0 - left / pool)
        touched = entries + pool
    return {"bytes": 2.0 * copies * _page_bytes(case) + 8 * touched, "flops": float(touched)}


# ---- inputs --------------------------------------------------------------------------------------------------------

def _offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def _positions(case, gen):
    """int32 [axes, tokens].  Three axes: text, alike on all, and image grids (time, row, column) in turn; two: rows and
    columns of a grid; one: text.  A single token each where sequences are far along."""
    n, a = case["tokens"], case["axes"]
    at = torch.arange(n, device=DEV)
    if n <= 64:
        p = torch.randint(0, case["far"] + 1, (n,), generator=gen, device=DEV)
        return torch.stack([p - torch.randint(0, 40, (n,), generator=gen, device=DEV) * (i > 0) for i in range(a)]).to(torch.int32)
    if a == 2:
        return torch.stack([at // 71, at % 71]).to(torch.int32)
    base = int(torch.randint(0, case["far"] + 1, (1,), generator=gen, device=DEV))
    text = at + base
    if a == 1:
        return text[None].to(torch.int32)
    block, inner = at // 1024, at % 1024  # 128 tokens of text, then an image of 28 x 32 patches
    grid = inner >= 128
    patch = inner - 128
    start = base + block * 160 + 128
    place = [start, start + patch // 32, start + patch % 32]
    return torch.stack([torch.where(grid, p, base + block * 160 + inner) for p in place]).to(torch.int32)


def _axis_of(pair, case):
    """Three axes take a quarter and two times three eighths of the pairs, two axes a half each."""
    r, a = case["rope"] // 2, case["axes"]
    ends = [r] if a == 1 else [r // 2, r] if a == 2 else [r // 4, r // 4 + (r - r // 4) // 2, r]
    return next(i for i, e in enumerate(ends) if pair < e)


def _pool_pages(case):
    """As many pages as the sequences hold, what a call can take at most, and three more."""
    lens, page = _families(case), case["page"]
    held = sum(-(-n // page) for b, n in enumerate(lens) if b % case["share"] == 0)
    return held + 3 + (0 if case["op"] == "compact" else sum(-(-(n + case["tokens"]) // page) + 1 for n in lens))


def _prepare_pages(case, seed, gen):
    lens, page, b = _families(case), case["page"], case["batch"]
    pool, width = _pool_pages(case), max(-(-(n + case["tokens"]) // page) for n in lens)
    numbers, at = torch.randperm(pool, generator=gen, device=DEV).tolist(), 0
    rows = []
    for i in range(b):
        n = -(-lens[i] // page)
        if i % case["share"]:
            rows.append(list(rows[-1]))
        else:
            rows.append(numbers[at:at + n] + [-1] * (width - n))
            at += n
    refs = [0] * pool
    for r in rows:
        for p in r:
            if p >= 0:
                refs[p] += 1
    rng = random.Random(seed)
    share = case["share"]
    source = [rng.randrange(i // share * share, min(b, i // share * share + share)) for i in range(b)]
    s = dict(case=case, pool=None, table_before=torch.tensor(rows, dtype=torch.int32, device=DEV), refs_before=torch.tensor(refs, dtype=torch.int32, device=DEV),
             filled=torch.tensor(lens, dtype=torch.int32, device=DEV), source=torch.tensor(source, dtype=torch.int32, device=DEV),
             target=torch.arange(b, dtype=torch.int32, device=DEV))
    s["table"], s["refs"] = s["table_before"].clone(), s["refs_before"].clone()
    s["wanted"], s["zero"] = s["filled"] + case["tokens"], torch.zeros_like(s["filled"])
    s["keep"] = torch.where(s["target"] % 2 > 0, s["filled"], 0)
    shape = (case["layers"], pool, case["kv_heads"], page)
    for x in "kv":
        if case["bits"] == 8:
            s[x + "_codes"] = torch.randint(-127, 128, shape + (case["dim"],), generator=gen, device=DEV, dtype=torch.int8)
        else:
            s[x + "_codes"] = torch.randint(0, 256, shape + (case["dim"] // 2,), generator=gen, device=DEV, dtype=torch.uint8)
        s[x + "_scale"] = torch.rand(shape, generator=gen, device=DEV).add_(0.1)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "rotate":
        n, h, hk, d, r = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rope"] // 2
        s = dict(case=case, rotary=None)
        qkv = torch.randn(n, h + 2 * hk, d, generator=gen, device=DEV).to(DT[case["dtype"]])  # one projection's output
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + hk]
        s["positions"] = _positions(case, gen)
        s["freq"] = (1.0 / 10000.0 ** (torch.arange(r, dtype=torch.float64) / r)).float().to(DEV)
        s["axis"] = [_axis_of(i, case) for i in range(r)]
        s["axis_index"] = torch.tensor(s["axis"], device=DEV)
        return s
    if op == "cross":
        lq, lk = _lengths(case, case["batch"], case["tokens"], case["ragged"]), _state_lengths(case)
        h, hk, d, dt = case["heads"], case["kv_heads"], case["dim"], DT[case["dtype"]]
        s = dict(case=case, q=torch.randn(sum(lq), h, d, generator=gen, device=DEV).mul_(1.5).to(dt))
        kv = torch.randn(sum(lk), 2, hk, d, generator=gen, device=DEV).to(dt)  # one projection of the encoder's output
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        s["cu_q"], s["cu_k"], s["most_q"], s["most_k"] = _offsets(lq).to(DEV), _offsets(lk).to(DEV), max(lq), max(lk)
        s["reads"] = torch.tensor(_reads(case), dtype=torch.int32, device=DEV)
        s["sink"] = torch.randn(h, generator=gen, device=DEV) if case["sink"] else None
        return s
    return _prepare_pages(case, seed, gen)


# ---- the plain form ------------------------------------------------------------------------------------------------

def _rotate(s):
    c = s["case"]
    angle = s["positions"].double()[s["axis_index"]].t() * s["freq"].double()  # [tokens, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    first, r = c["dim"] - c["rope"], c["rope"] // 2
    one, two = (slice(first, None, 2), slice(first + 1, None, 2)) if c["pairs"] == "adjacent" else (slice(first, first + r), slice(first + r, None))
    outs = []
    for x in (s["q"], s["k"]):
        y = x.float()
        a, b = y[..., one], y[..., two]
        out = torch.empty(x.shape, dtype=x.dtype, device=DEV)
        out[..., :first] = x[..., :first]
        out[..., one] = (a * cos - b * sin).to(x.dtype)
        out[..., two] = (b * cos + a * sin).to(x.dtype)
        outs.append(out)
    return outs


def _cross(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    lq = s["cu_q"].diff()
    lk = s["cu_k"].diff()[s["reads"]]
    iq, ik = torch.arange(s["most_q"], device=DEV), torch.arange(s["most_k"], device=DEV)
    at_q = (s["cu_q"][:-1, None] + iq).clamp(max=s["q"].size(0) - 1)
    at_k = (s["cu_k"][s["reads"], None] + ik).clamp(max=s["k"].size(0) - 1)
    q = s["q"][at_q].float().unflatten(2, (hk, h // hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (x[at_k].float().transpose(1, 2).contiguous() for x in (s["k"], s["v"]))
    logits = (q @ k.transpose(-1, -2).contiguous()).mul_(d ** -0.5)
    logits.masked_fill_((ik >= lk[:, None])[:, None, None], -math.inf)
    logits = logits.view(lq.size(0), hk, h // hk, s["most_q"], s["most_k"])
    top = logits.amax(-1, keepdim=True)
    sink = None if s["sink"] is None else s["sink"].view(hk, h // hk, 1, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(top.isinf(), 0.0, top)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - top)
    out = (p.flatten(2, 3) @ v).view(lq.size(0), hk, h // hk, s["most_q"], d) / torch.where(total > 0, total, 1.0)
    n = torch.arange(s["q"].size(0), device=DEV, dtype=torch.int32)  # back to the packed rows
    b = torch.searchsorted(s["cu_q"], n, right=True) - 1
    i = n - s["cu_q"][b]
    packed = out.flatten(1, 2)[b, :, i].to(s["q"].dtype)
    return [packed, (top + torch.log(total))[..., 0].flatten(1, 2)[b, :, i]] if c["lse"] else [packed]


def _copy_pages(s, src, dst):
    for x in ("k_codes", "k_scale", "v_codes", "v_scale"):
        s[x][:, dst] = s[x][:, src]


def _count(refs, page, by):
    """refs[page] += by, for the entries where by is not 0."""
    refs.scatter_add_(0, page.clamp(0).flatten(), by.to(torch.int32).flatten())


def _reserve(s, filled, wanted, first):
    size, table, refs = s["case"]["page"], s["table"], s["refs"]
    i = torch.arange(table.size(1), device=DEV)
    inside = (i >= first[:, None] // size) & (i < (wanted[:, None] + size - 1) // size)
    page = table.long()
    at = page.clamp(0)
    shared = inside & (page >= 0) & (refs[at] > 1)
    entry = torch.arange(table.numel(), device=DEV).view(table.shape)
    holders = torch.zeros_like(refs)
    _count(holders, page, shared)
    last = torch.full_like(refs, -1, dtype=torch.int64).scatter_reduce_(0, at.flatten(), torch.where(shared, entry, -1).flatten(), "amax")
    shared &= ~((holders[at] == refs[at]) & (last[at] == entry))  # the last of a page's holders keeps it
    takes = inside & ((page < 0) | shared)
    rank = takes.flatten().cumsum(0).view(table.shape) - 1
    unused = refs == 0
    lowest = unused.int().sort(descending=True, stable=True)[1]
    new = torch.where(rank < unused.sum(), lowest[rank.clamp(0, refs.size(0) - 1)], -1)
    moved = shared & (i * size < filled[:, None]) & (new >= 0)
    src, dst = page[moved], new[moved]
    _count(refs, page, -shared.int())
    _count(refs, new, takes & (new >= 0))
    table.copy_(torch.where(takes, new, page))
    _copy_pages(s, src, dst)


def _fork(s, filled):
    size, table, source = s["case"]["page"], s["table"], s["source"].long()
    i = torch.arange(table.size(1), device=DEV)
    moves = (source != s["target"])[:, None]
    new = torch.where(i < (filled[source, None] + size - 1) // size, table[source], -1)
    new = torch.where(moves, new, table)
    _count(s["refs"], table.long(), -((table >= 0) & moves).int())
    _count(s["refs"], new.long(), (new >= 0) & moves)
    table.copy_(new)


def _release(s, keep):
    size, table = s["case"]["page"], s["table"]
    gone = torch.arange(table.size(1), device=DEV) >= (keep[:, None] + size - 1) // size
    _count(s["refs"], table.long(), -(gone & (table >= 0)).int())
    table.masked_fill_(gone, -1)


def _compact(s):
    table, refs = s["table"], s["refs"]
    number, live = torch.arange(refs.size(0), device=DEV), refs > 0
    count = live.sum()
    dst, src = number[~live & (number < count)], number[live & (number >= count)]
    _copy_pages(s, src, dst)
    to = number.clone()
    to[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, to[table.long().clamp(0)], table.long()))


# ---- the framework's -----------------------------------------------------------------------------------------------

def _own_rotate(s):
    from aetherkv.rotary import AxisRotary, rotate_axes

    if s["rotary"] is None:  # made once, as a program does
        s["rotary"] = AxisRotary(s["freq"], s["axis"], s["case"]["dim"], pairs=s["case"]["pairs"])
    return list(rotate_axes(s["q"], s["k"], s["positions"], s["rotary"]))


def _own_cross(s):
    from aetherkv.cross import cross_attention

    c = s["case"]
    out = cross_attention(s["q"], s["k"], s["v"], s["cu_k"], c["dim"] ** -0.5, cu_seqlens=s["cu_q"] if c["tokens"] > 1 else None,
                          states=s["reads"] if c["states"] != c["batch"] else None, sink=s["sink"], return_lse=c["lse"])
    return list(out) if c["lse"] else [out]


def _pool(s):
    if s["pool"] is None:  # the layers' caches and their pool, made once
        from aetherkv import PolarQuant
        from aetherkv.paged import PagedKVCache
        from aetherkv.pages import PagePool

        quant = PolarQuant(s["case"]["bits"])
        caches = [PagedKVCache.from_tensors(quant, *(s[x][i] for x in ("k_codes", "k_scale", "v_codes", "v_scale"))) for i in range(s["case"]["layers"])]
        s["pool"] = PagePool(caches, refs=s["refs"])
    return s["pool"]


def run(s):
    if own and PKG not in sys.path:
        sys.path.insert(0, PKG)
    c = s["case"]
    op = c["op"]
    if op == "rotate":
        return _own_rotate(s) if own else _rotate(s)
    if op == "cross":
        return _own_cross(s) if own else _cross(s)
    s["table"].copy_(s["table_before"])  # changed in place: a pass starts from the same tables
    s["refs"].copy_(s["refs_before"])
    if op == "reserve":
        first = s["zero"] if c["whole"] else s["filled"]
        _pool(s).reserve(s["table"], s["filled"], s["wanted"], first=first) if own else _reserve(s, s["filled"], s["wanted"], first)
    elif op == "fork":
        if own:
            _pool(s).fork(s["table"], s["filled"], s["source"], s["target"])
        else:
            _fork(s, s["filled"])
        filled = s["filled"][s["source"]]
        wanted = filled + c["tokens"]
        _pool(s).reserve(s["table"], filled, wanted) if own else _reserve(s, filled, wanted, filled)
    elif own:
        _pool(s).release(s["table"], s["keep"])
        _pool(s).compact(s["table"])
    else:
        _release(s, s["keep"])
        _compact(s)
    return [s["table"], s["refs"], s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _exact_rotate(s):
    """Pairs as complex numbers, turned by exp(i p f)."""
    c = s["case"]
    r = c["rope"] // 2
    theta = torch.stack([s["positions"][s["axis"][i]].double() * float(s["freq"][i]) for i in range(r)], 1)
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    outs = []
    for x in (s["q"], s["k"]):
        out = x.double().clone()
        part = out[..., c["dim"] - c["rope"]:]
        pair = part.unflatten(-1, (r, 2)) if c["pairs"] == "adjacent" else part.unflatten(-1, (2, r)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        part.copy_((turned if c["pairs"] == "adjacent" else turned.transpose(-1, -2)).flatten(-2))
        outs.append(out)
    return outs


def _exact_cross(s):
    c = s["case"]
    g = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b, e in enumerate(s["reads"].tolist()):
        for j in range(c["kv_heads"]):
            k, v = s["k"][ck[e]:ck[e + 1], j].double().t().contiguous(), s["v"][ck[e]:ck[e + 1], j].double().contiguous()
            for at in range(cq[b], cq[b + 1], 2048):
                to = min(cq[b + 1], at + 2048)
                heads = slice(j * g, j * g + g)
                e_ = torch.mm(s["q"][at:to, heads].double().reshape(-1, c["dim"]), k) / math.sqrt(c["dim"])
                if s["sink"] is not None:
                    e_ = torch.cat([e_, s["sink"][heads].double().repeat(to - at)[:, None]], 1)
                total = torch.logsumexp(e_, 1)
                lse[at:to, heads] = total.view(-1, g)
                out[at:to, heads] = torch.mm(torch.exp(e_ - total[:, None])[:, :k.size(1)].contiguous(), v).view(-1, g, c["dim"])
    return [out, lse] if c["lse"] else [out]


def _exact_pages(s):
    """The scales alone: nothing is computed, they move with their pages; tables and codes are whole numbers."""
    c, size = s["case"], s["case"]["page"]
    rows, refs = s["table_before"].tolist(), s["refs_before"].tolist()
    filled = s["filled"].tolist()
    src, dst = [], []
    if c["op"] == "compact":
        for b, keep in enumerate(s["keep"].tolist()):
            for p in rows[b][-(-keep // size):]:
                if p >= 0:
                    refs[p] -= 1
        live = [p for p in range(len(refs)) if refs[p] > 0]
        dst = [p for p in range(len(live)) if refs[p] <= 0]
        src = [p for p in live if p >= len(live)]
    else:
        if c["op"] == "fork":
            source = s["source"].tolist()
            new = [rows[b] if b == f else [p if i < -(-filled[f] // size) else -1 for i, p in enumerate(rows[f])] for b, f in enumerate(source)]
            filled = [filled[f] for f in source]
            for old, fresh in zip(rows, new):
                for p in old:
                    refs[p] -= p >= 0
                for p in fresh:
                    refs[p] += p >= 0
            rows = new
        held = {}
        for b, n in enumerate(filled):
            for i in range(0 if c["whole"] else n // size, -(-(n + c["tokens"]) // size)):
                if rows[b][i] >= 0 and refs[rows[b][i]] > 1:
                    held.setdefault(rows[b][i], []).append((b, i))
        keeps = {places[-1] for p, places in held.items() if len(places) == refs[p]}
        unused = (p for p in range(len(refs)) if refs[p] == 0)
        for b, n in enumerate(filled):
            for i in range(0 if c["whole"] else n // size, -(-(n + c["tokens"]) // size)):
                p = rows[b][i]
                if p < 0 or (p in held and (b, i) not in keeps):
                    fresh = next(unused)
                    if p >= 0 and i * size < n:
                        src.append(p)
                        dst.append(fresh)
    src, dst = torch.tensor(src, dtype=torch.int64, device=DEV), torch.tensor(dst, dtype=torch.int64, device=DEV)
    scales = []
    for x in ("k_scale", "v_scale"):
        moved = s[x].double().clone()
        moved[:, dst] = moved[:, src]
        scales.append(moved)
    return [None, None, None, scales[0], None, scales[1]]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s)
    if case["op"] == "cross":
        return _exact_cross(s)
    return _exact_pages(s)
