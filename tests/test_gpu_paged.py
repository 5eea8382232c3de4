"""Paged cache in TurboQuant codes on the GPU against plain 64-bit forms (paged_ref.py): append, attention, eviction, and
a run of them together."""
from __future__ import annotations

import math

import pytest
import torch

import paged_ref as R
from aetherkv import PolarQuant
from aetherkv.paged import (PagedKVCache, SlotTracker, append_tokens, evict_by_weight, evict_workspace, paged_attention,
                            paged_attention_workspace)
from conftest import randn_outliers

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _fill(dev, seed, bits, dim, heads, page, pages):
    """A pool of coded Gaussian entries, with NaN scales nowhere."""
    pq = PolarQuant(bits)
    x = torch.randn(2, pages, heads, page, dim, device=dev, generator=_gen(dev, seed)).to(torch.bfloat16)
    kc, ks = pq.encode(x[0])
    vc, vs = pq.encode(x[1])
    return PagedKVCache.from_tensors(pq, kc, ks[..., 0].contiguous(), vc, vs[..., 0].contiguous())


def _cache(dev, seed, bits, dim, heads, page, lengths, spare=3):
    per = max(1, -(-max(max(lengths), 1) // page))
    pages = per * len(lengths) + spare
    cache = _fill(dev, seed, bits, dim, heads, page, pages)
    table = torch.randperm(pages, device=dev, generator=_gen(dev, seed + 1))[:per * len(lengths)].to(torch.int32).view(len(lengths), per)
    return cache, table, torch.tensor(lengths, dtype=torch.int32, device=dev)


def _poison(cache, table, lengths):
    """NaN scales in every slot past a sequence's length and in every page of no sequence: they must not matter."""
    used = torch.zeros(cache.pages, cache.page_size, dtype=torch.bool, device=table.device)
    for b, n in enumerate(lengths.tolist()):
        slot = torch.arange(max(0, n), device=table.device)
        used[table[b].long()[slot // cache.page_size], slot % cache.page_size] = True
    for s in (cache.k_scale, cache.v_scale):
        s.masked_fill_(~used[:, None, :], NAN)


def _check_attention(dev, bits, dim, dtype, page, heads, group, T, lengths, sink, track, seed=0, scale=None, gain=1.0):
    cache, table, n = _cache(dev, seed, bits, dim, heads, page, lengths)
    _poison(cache, table, n)
    B, H = len(lengths), heads * group
    q = (torch.randn(B, T, H, dim, device=dev, generator=_gen(dev, seed + 2)) * gain).to(dtype)
    sk = torch.randn(H, device=dev, generator=_gen(dev, seed + 3)) if sink else None
    tracker = before = None
    if track:
        tracker = SlotTracker(B, heads, table.size(1) * page, device=dev)
        tracker.weights.uniform_(0, 3, generator=_gen(dev, seed + 4))
        before = tracker.weights.double().cpu()
    scale = dim ** -0.5 if scale is None else scale
    got = paged_attention(q, cache, table, n, scale, sink=sk, tracker=tracker)
    want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, table), q.cpu(), lengths, scale, None if sk is None else sk.cpu(), tracker.capacity if track else None)
    R.within(got, want, bound, "out")
    if track:
        R.within(tracker.weights, before + w, wb + 2.0 ** -23 * (before + w), "weights")
        assert torch.equal(tracker.weights.cpu()[w == 0], before.float()[w == 0]), "weights of slots that nothing sees"


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 257, 300]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_every_type_and_length(dev, bits, dim, dtype):
    _check_attention(dev, bits, dim, dtype, 16, 2, 3, 1, LENGTHS, False, True, seed=bits + dim)


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 12), (12, 1), (3, 4), (2, 16), (1, 17), (1, 40)])
def test_attention_head_layouts(dev, heads, group):
    _check_attention(dev, 4, 128, torch.bfloat16, 32, heads, group, 1, [70, 1, 333], True, True, seed=group)


@pytest.mark.parametrize("T,heads,group", [(2, 2, 3), (5, 1, 4), (16, 2, 8), (7, 3, 1), (33, 1, 2)])
def test_attention_several_tokens(dev, T, heads, group):
    # (a sequence shorter than T: its first tokens see nothing)
    _check_attention(dev, 8, 64, torch.float16, 16, heads, group, T, [T, T + 1, 200, 3, 0], False, True, seed=T)


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
def test_attention_page_sizes(dev, page):
    _check_attention(dev, 4, 64, torch.bfloat16, page, 2, 2, 2, [5, page, page + 1, 3 * page - 7], True, True, seed=page)


@pytest.mark.parametrize("length", [1000, 4097, 20011])
def test_attention_long(dev, length):
    _check_attention(dev, 4, 128, torch.bfloat16, 64, 1, 3, 1, [length, length // 3], False, True, seed=length)


def test_attention_peaked_and_flat(dev):
    _check_attention(dev, 8, 128, torch.float16, 16, 2, 2, 1, [200, 90], False, True, gain=30.0)
    _check_attention(dev, 4, 128, torch.bfloat16, 16, 2, 2, 1, [200, 90], True, True, scale=0.0)
    _check_attention(dev, 4, 64, torch.bfloat16, 16, 2, 2, 1, [200, 90], True, False, scale=-0.2)


def test_attention_scales_of_many_sizes(dev):
    """V scales over twelve decades, the largest where the weight is small, and queries near the type's ends."""
    cache, table, n = _cache(dev, 5, 4, 128, 1, 16, [150])
    cache.v_scale.mul_(10 ** (12 * torch.rand(cache.v_scale.shape, device=dev, generator=_gen(dev, 6)) - 6))
    q = torch.randn(1, 1, 3, 128, device=dev, generator=_gen(dev, 7)).to(torch.bfloat16)
    for f in (1.0, 2.0 ** 60, 2.0 ** -60):
        qq = q * f
        got = paged_attention(qq, cache, table, n, 128 ** -0.5 / f)
        want, bound, _, _ = R.paged_attention_ref(R.HostCache(cache, table), qq.cpu(), [150], 128 ** -0.5 / f)
        R.within(got, want, bound, f"q times {f}")


def test_attention_sinks_at_the_ends(dev):
    cache, table, n = _cache(dev, 8, 4, 128, 1, 16, [40, 0, 1])
    q = torch.randn(3, 1, 2, 128, device=dev, generator=_gen(dev, 9)).to(torch.bfloat16)
    sink = torch.tensor([-math.inf, 200.0], device=dev)
    got = paged_attention(q, cache, table, n, 0.09, sink=sink)
    want, bound, _, _ = R.paged_attention_ref(R.HostCache(cache, table), q.cpu(), [40, 0, 1], 0.09, sink.cpu())
    R.within(got, want, bound, "out")
    assert not got[1].any()
    plain = paged_attention(q[:, :, :1], cache, table, n, 0.09)
    assert torch.equal(plain, got[:, :, :1])  # a sink of -inf is none


def test_attention_nan_stays_in_its_rows(dev):
    cache, table, n = _cache(dev, 10, 8, 64, 2, 16, [50, 60])
    q = torch.randn(2, 3, 4, 64, device=dev, generator=_gen(dev, 11)).to(torch.float16)
    clean = paged_attention(q, cache, table, n, 0.125)
    q2 = q.clone()
    q2[1, 2, 3] = NAN
    got = paged_attention(q2, cache, table, n, 0.125)
    assert got[1, 2, 3].isnan().all()
    keep = torch.ones(2, 3, 4, dtype=torch.bool, device=dev)
    keep[1, 2, 3] = False
    assert torch.equal(got[keep], clean[keep])
    # a NaN entry in the newest slot: the earlier tokens do not see it
    cache.v_scale[table[0, 49 // 16].long(), 0, 49 % 16] = NAN
    got = paged_attention(q, cache, table, n, 0.125)
    assert got[0, 2, :2].isnan().all() and torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1], clean[1])


def test_attention_skips_bad_pages_and_clamps_lengths(dev):
    cache, table, n = _cache(dev, 12, 4, 128, 2, 16, [100, 100, 100])
    table[0, 2], table[1, 0], table[1, 6] = -1, cache.pages, 0x7fffffff
    n = torch.tensor([100, 100, 5000], dtype=torch.int32, device=dev)
    q = torch.randn(3, 1, 4, 128, device=dev, generator=_gen(dev, 13)).to(torch.bfloat16)
    tracker = SlotTracker(3, 2, 112, device=dev)
    got = paged_attention(q, cache, table, n, 0.09, tracker=tracker)
    want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, table), q.cpu(), [100, 100, 5000], 0.09, capacity=112)
    R.within(got, want, bound, "out")
    R.within(tracker.weights, w, wb, "weights")
    neg = paged_attention(q, cache, table, torch.tensor([-5, 0, -(2 ** 31)], dtype=torch.int32, device=dev), 0.09)
    assert not neg.any()
    assert not paged_attention(q, cache, torch.full_like(table, -1), n, 0.09).any()
    assert not paged_attention(q, cache, table[:, :0], n, 0.09, tracker=tracker).any()


def test_attention_tracker_smaller_than_the_table(dev):
    """Slots behind the tracker's last have nowhere to be counted: a tracked call ends at its capacity."""
    cache, table, n = _cache(dev, 14, 4, 64, 1, 16, [90])
    q = torch.randn(1, 1, 2, 64, device=dev, generator=_gen(dev, 15)).to(torch.bfloat16)
    storage = torch.zeros(2, 1, 1, 70, dtype=torch.int32, device=dev)
    tracker = SlotTracker.from_tensor(storage)
    got = paged_attention(q, cache, table, n, 0.125, tracker=tracker)
    want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, table), q.cpu(), [90], 0.125, capacity=70)
    R.within(got, want, bound, "out")
    R.within(tracker.weights, w, wb, "weights")


def test_attention_strided_query_given_output_and_workspace(dev):
    cache, table, n = _cache(dev, 16, 4, 128, 2, 32, [77, 200])
    wide = torch.randn(2, 3, 9, 128, device=dev, generator=_gen(dev, 17)).to(torch.bfloat16)
    q = wide[:, :, 1:5]
    want = paged_attention(q.contiguous(), cache, table, n, 0.09)
    out = torch.empty(2, 3, 4, 128, dtype=torch.bfloat16, device=dev)
    ws = paged_attention_workspace(2, 3, 4, 2, 128, table.size(1) * 32, dev)
    ws.fill_(255)
    assert paged_attention(q, cache, table, n, 0.09, out=out, workspace=ws).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    odd = torch.empty(2 * 3 * 4 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 3, 4, 128).copy_(q)
    assert torch.equal(paged_attention(odd, cache, table, n.long(), 0.09), want)  # misaligned: copied
    back = torch.empty(2, 4, 128, 3, dtype=torch.bfloat16, device=dev).copy_(q.permute(0, 2, 3, 1)).permute(0, 3, 1, 2)
    assert torch.equal(paged_attention(back, cache, table.long(), n, 0.09), want)  # strided in D: copied


def test_attention_repeats_and_streams(dev):
    """The same call gives the same bits, on its own stream or another, beside a call on a second stream."""
    cache, table, n = _cache(dev, 18, 4, 128, 4, 64, [3000, 1500, 64, 5])
    q = torch.randn(4, 1, 12, 128, device=dev, generator=_gen(dev, 19)).to(torch.bfloat16)
    want = paged_attention(q, cache, table, n, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(paged_attention(q, cache, table, n, 0.09))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_attention_tracked_repeats_bit_for_bit(dev):
    cache, table, n = _cache(dev, 20, 4, 128, 2, 64, [5000, 700])
    q = torch.randn(2, 4, 6, 128, device=dev, generator=_gen(dev, 21)).to(torch.bfloat16)
    got = []
    for _ in range(3):
        tracker = SlotTracker(2, 2, table.size(1) * 64, device=dev)
        got.append((paged_attention(q, cache, table, n, 0.09, tracker=tracker), tracker.weights))
    for o, w in got[1:]:
        assert torch.equal(o, got[0][0]) and torch.equal(w, got[0][1])


def test_attention_offsets_past_31_bits(dev):
    """A pool of more than 2 GiB of codes, the sequence in its last pages."""
    pq = PolarQuant(8)
    pages, page = 4200, 4096
    codes = torch.zeros(pages, 1, page, 128, dtype=torch.int8, device=dev)  # 2.2 GB
    scale = torch.zeros(pages, 1, page, device=dev)
    x = torch.randn(2, page, 128, device=dev, generator=_gen(dev, 22)).to(torch.bfloat16)
    c, s = pq.encode(x)
    codes[-2:, 0], scale[-2:, 0] = c, s[..., 0]
    cache = PagedKVCache.from_tensors(pq, codes, scale, codes, scale)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    q = torch.randn(1, 1, 2, 128, device=dev, generator=_gen(dev, 23)).to(torch.bfloat16)
    got = paged_attention(q, cache, table, torch.tensor([4500], dtype=torch.int32, device=dev), 0.09)
    small = PagedKVCache.from_tensors(pq, codes[-2:].clone(), scale[-2:].clone(), codes[-2:].clone(), scale[-2:].clone())
    st = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    want, bound, _, _ = R.paged_attention_ref(R.HostCache(small, st), q.cpu(), [4500], 0.09)
    R.within(got, want, bound, "out")


def test_refusals(dev):
    cache, table, n = _cache(dev, 24, 4, 128, 2, 16, [20, 30])
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device=dev)
    tracker = SlotTracker(2, 2, 32, device=dev)
    for bad in (q.float(), q[..., :64], q[:, :, :3], q[:1], q[0]):
        with pytest.raises(RuntimeError):
            paged_attention(bad, cache, table, n, 0.1)
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n[:1], 0.1)
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n.cpu(), 0.1)
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n, 0.1, sink=torch.zeros(3, device=dev))
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n, 0.1, tracker=SlotTracker(2, 3, 32, device=dev))
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n, 0.1, out=torch.empty_like(q, dtype=torch.float16))
    with pytest.raises(RuntimeError):
        paged_attention(q, cache, table, n, 0.1, tracker=tracker, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    k = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError):
        append_tokens(cache, k, k.half(), table, n)
    with pytest.raises(RuntimeError):
        append_tokens(cache, k, k[:, :, :1], table, n)
    with pytest.raises(RuntimeError):
        append_tokens(cache, k, k, table, n, tracker=tracker)  # without token
    with pytest.raises(RuntimeError):
        append_tokens(cache, k[:, 0], k[:, 0], table, n, cu_seqlens=n)  # [B + 1] wanted
    with pytest.raises(ValueError):
        evict_by_weight(cache, table, n, tracker, n, 8, first=5, recent=4)
    with pytest.raises(RuntimeError):
        evict_by_weight(cache, table, n, tracker, n, 8, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError):
        PagedKVCache.from_tensors(cache.quant, cache.k_codes, cache.k_scale[:1], cache.v_codes, cache.v_scale)
    with pytest.raises(RuntimeError):
        PagedKVCache.from_tensors(PolarQuant(8), cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)


# ---- append ----------------------------------------------------------------------------------------------------

def _expect_append(cache, k, v, table, start, cu):
    """The pools after the append, by PolarQuant.encode and plain indexing."""
    pools = [cache.k_codes.clone(), cache.k_scale.clone(), cache.v_codes.clone(), cache.v_scale.clone()]
    for x, pc, ps in ((k, pools[0], pools[1]), (v, pools[2], pools[3])):
        codes, scale = cache.quant.encode(x.contiguous())
        for b in range(table.size(0)):
            for i, r in enumerate(range(max(0, cu[b]), min(cu[b + 1], x.size(0)))):
                p = start[b] + i
                page = int(table[b, p // cache.page_size]) if 0 <= p < table.size(1) * cache.page_size else -1
                if 0 <= page < cache.pages:
                    pc[page, :, p % cache.page_size] = codes[r]
                    ps[page, :, p % cache.page_size] = scale[r, :, 0]
    return pools


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append_bit_exact(dev, bits, dim, dtype):
    heads, B, T, page = 3, 4, 5, 16
    cache, table, _ = _cache(dev, 30, bits, dim, heads, page, [40] * B)
    kv = randn_outliers((B, T, 2 * heads, dim), seed=31).to(dev).to(dtype)
    k, v = kv[:, :, :heads], kv[:, :, heads:]  # views of one projection
    start = [0, 14, 30, 46]  # the last one runs past its table
    want = _expect_append(cache, k.reshape(B * T, heads, dim), v.reshape(B * T, heads, dim), table.cpu(), start, [T * b for b in range(B + 1)])
    tracker = SlotTracker(B, heads, 48, device=dev)
    tracker.weights.fill_(9.0)
    tracker.tokens.fill_(-7)
    append_tokens(cache, k, v, table, torch.tensor(start, dtype=torch.int32, device=dev), tracker=tracker, token=torch.tensor([0, 100, 200, 300], dtype=torch.int32, device=dev))
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(got, w)
    for b in range(B):
        for p in range(48):
            i = p - start[b]
            assert (tracker.weights[b, :, p] == (0.0 if 0 <= i < T else 9.0)).all()
            assert (tracker.tokens[b, :, p] == (100 * b + i if 0 <= i < T else -7)).all()


@pytest.mark.parametrize("lens", [[1], [0, 3, 0, 40, 1], [257, 64, 0]])
def test_append_packed(dev, lens):
    heads, dim, page = 2, 128, 16
    B = len(lens)
    cache, table, _ = _cache(dev, 32, 4, dim, heads, page, [max(lens) + 20] * B)
    N = sum(lens) + 5  # rows behind the last sequence
    k, v = (randn_outliers((N, heads, dim), seed=33 + i).to(dev) for i in range(2))
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    start = [3 * b for b in range(B)]
    want = _expect_append(cache, k, v, table.cpu(), start, cu)
    append_tokens(cache, k, v, table, torch.tensor(start, dtype=torch.int32, device=dev), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(got, w)


def test_append_special_values_and_many_sequences(dev):
    """Zeros, infinities and NaN code as PolarQuant codes them; 300 sequences of one packed token each."""
    cache, table, _ = _cache(dev, 34, 4, 64, 1, 16, [16] * 300)
    k = torch.randn(300, 1, 64, device=dev, generator=_gen(dev, 35)).to(torch.bfloat16)
    k[0], k[1, 0, 3], k[2, 0, 5], k[3] = 0, math.inf, NAN, 1e-30
    v = k.flip(0)
    cu = torch.arange(301, dtype=torch.int32, device=dev)
    start = torch.arange(300, dtype=torch.int32, device=dev) % 16
    want = _expect_append(cache, k, v, table.cpu(), start.tolist(), cu.tolist())
    append_tokens(cache, k, v, table, start, cu_seqlens=cu)
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        fine = ~torch.isnan(w) if w.is_floating_point() else torch.ones_like(w, dtype=torch.bool)
        assert torch.equal(got[fine], w[fine])
        assert not w.is_floating_point() or got[~fine].isnan().all()


def test_append_skips_bad_pages_and_counts(dev):
    cache, table, _ = _cache(dev, 36, 8, 64, 2, 16, [64, 64, 64])
    table[0, 1], table[1, 0] = -3, cache.pages
    k, v = (torch.randn(3, 4, 2, 64, device=dev, generator=_gen(dev, 37 + i)).to(torch.bfloat16) for i in range(2))
    start = [14, 14, -2]  # a negative start: the first two have no slot
    want = _expect_append(cache, k.flatten(0, 1), v.flatten(0, 1), table.cpu(), start, [0, 4, 8, 12])
    append_tokens(cache, k, v, table, torch.tensor(start, dtype=torch.int32, device=dev))
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(got, w)
    before = cache.k_codes.clone()
    append_tokens(cache, k[:, :0], v[:, :0], table, torch.tensor(start, dtype=torch.int32, device=dev))
    assert torch.equal(cache.k_codes, before)


@pytest.mark.parametrize("bits,dim,dtype", [(4, 64, torch.bfloat16), (4, 128, torch.bfloat16), (8, 64, torch.float16), (8, 128, torch.float16), (4, 128, torch.float32)])
def test_append_many_rows(dev, bits, dim, dtype):
    """Large calls take another layout: packed sequences of odd lengths with zeros, infinities, NaN, values near ties of the
    rounding and the smallest and largest numbers among them, and a uniform batch of strided views."""
    heads, page = 5, 32
    lens = [700, 0, 1, 33, 1501]
    B, N = len(lens), sum(lens) + 9
    cache, table, _ = _cache(dev, 38, bits, dim, heads, page, [1600] * B)
    table[3, 0] = -1
    kv = randn_outliers((N, 2, heads, dim), seed=39).to(dev)
    kv[5, 0, 2], kv[17, 1, 1, 7], kv[40, 0, 0, 3], kv[700, 1] = 0, math.inf, NAN, 2.0 ** -130
    kv[900:1000] = torch.randint(-3, 4, (100, 2, heads, dim), device=dev, generator=_gen(dev, 40)).to(kv.dtype)  # many ties
    kv[1100:1110] *= 2.0 ** 100 if dtype != torch.float16 else 2.0 ** 10
    kv = kv.to(dtype)
    k, v = kv[:, 0], kv[:, 1]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    start = [3, 0, 5, 60, 100]
    want = _expect_append(cache, k, v, table.cpu(), start, cu)
    tracker = SlotTracker(B, heads, 1600, device=dev)
    tracker.weights.fill_(2.0)
    append_tokens(cache, k, v, table, torch.tensor(start, dtype=torch.int32, device=dev), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev), tracker=tracker,
                  token=torch.tensor(start, dtype=torch.int32, device=dev))
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        if w.is_floating_point():
            nan = w.isnan()
            assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], w[~nan])
    # the two vectors that hold an infinity or a NaN (tokens 17 and 40 of the first sequence) have no codes to compare
    for got, w, token, head in ((cache.k_codes, want[0], 40, 0), (cache.v_codes, want[2], 17, 1)):
        fine = torch.ones(w.shape[:3], dtype=torch.bool, device=dev)
        fine[int(table[0, (3 + token) // page]), head, (3 + token) % page] = False
        assert torch.equal(got[fine], w[fine])
    for b in range(B):
        for h in range(heads):
            t, wt = tracker.tokens[b, h].tolist(), tracker.weights[b, h].tolist()
            # (slot 1600 is past the table: the last token has no place)
            assert t[start[b]:start[b] + lens[b]] == list(range(start[b], min(start[b] + lens[b], 1600))) or b == 3
            assert all(x == 2.0 for x in wt[:start[b]]) and all(x == 2.0 for x in wt[start[b] + lens[b]:])
    T = 260
    cache, table, _ = _cache(dev, 41, bits, dim, heads, page, [300] * 4)
    kv = randn_outliers((4, T, 2 * heads, dim), seed=42).to(dev).to(dtype)
    k, v = kv[:, :, :heads], kv[:, :, heads:]
    want = _expect_append(cache, k.reshape(4 * T, heads, dim), v.reshape(4 * T, heads, dim), table.cpu(), [0, 7, 60, 31], [T * b for b in range(5)])
    append_tokens(cache, k, v, table, torch.tensor([0, 7, 60, 31], dtype=torch.int32, device=dev))
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(got, w)


# ---- eviction --------------------------------------------------------------------------------------------------

def _check_evict(dev, bits, dim, heads, page, lengths, keep, first, recent, weights=None, seed=0, capacity=None):
    cache, table, n = _cache(dev, seed, bits, dim, heads, page, lengths)
    B = len(lengths)
    cap = capacity if capacity is not None else table.size(1) * page
    tracker = SlotTracker(B, heads, cap, device=dev)
    w = torch.randn(B, heads, cap, generator=torch.Generator().manual_seed(seed + 5)).exp() if weights is None else weights(B, heads, cap)
    tracker.weights.copy_(w)
    tok = torch.stack([torch.randperm(cap, generator=torch.Generator().manual_seed(seed + i)) for i in range(B * heads)]).view(B, heads, cap)
    tracker.tokens.copy_(tok)
    seen = torch.tensor([max(x, 0) for x in lengths], dtype=torch.int32, device=dev)
    pools = [x.clone() for x in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
    ww, tt, tc = w.clone(), tok.clone(), table.cpu().long()
    w = tracker.weights.cpu()
    for b in range(B):
        for h in range(heads):
            m = min(lengths[b], cap, table.size(1) * page)
            for src, dst in R.evict_ref(w[b, h].tolist(), tok[b, h].tolist(), m, int(seen[b]), keep, first, recent):
                ps, pd = int(tc[b, src // page]), int(tc[b, dst // page])
                if 0 <= ps < cache.pages and 0 <= pd < cache.pages:
                    for x, y in zip(pools, (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)):
                        x[pd, h, dst % page] = y[ps, h, src % page]
                ww[b, h, dst], tt[b, h, dst] = w[b, h, src], tok[b, h, src]
    evict_by_weight(cache, table, n, tracker, seen, keep, first=first, recent=recent)
    assert torch.equal(tracker.tokens.cpu().long(), tt)
    assert torch.equal(tracker.weights.cpu().view(torch.int32), ww.float().view(torch.int32))
    for got, want in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), pools):
        assert torch.equal(got, want)


@pytest.mark.parametrize("bits,dim", [(4, 64), (4, 128), (8, 64), (8, 128)])
def test_evict_moves_whole_rows(dev, bits, dim):
    _check_evict(dev, bits, dim, 2, 16, [0, 1, 39, 40, 41, 64, 100, 200], 40, 4, 10, seed=bits + dim)


@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 1, 0), (7, 0, 7), (500, 2, 100), (999, 0, 0), (1024, 4, 128), (1025, 0, 1)])
def test_evict_budgets(dev, keep, first, recent):
    _check_evict(dev, 4, 64, 1, 64, [1500, 1025, 300], keep, first, recent, seed=keep)


@pytest.mark.parametrize("length", [1023, 1024, 1025, 2049, 5000, 9000, 33000])
def test_evict_long_rows(dev, length):
    _check_evict(dev, 4, 64, 2, 256, [length, length - 1], length // 3, 4, 64, seed=length)


def test_evict_keeps_nothing(dev):
    _check_evict(dev, 4, 64, 1, 16, [50], 0, 0, 0)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "tiny", "special"])
def test_evict_ties_and_special_weights(dev, kind):
    def weights(B, heads, cap):
        g = torch.Generator().manual_seed(3)
        if kind == "equal":
            return torch.ones(B, heads, cap)
        if kind == "few":
            return torch.randint(0, 3, (B, heads, cap), generator=g).float()
        if kind == "zeros":  # both zeros are one weight
            return torch.where(torch.rand(B, heads, cap, generator=g) < 0.5, 0.0, -0.0)
        if kind == "tiny":
            return torch.randint(0, 5, (B, heads, cap), generator=g).float() * 2.0 ** -149
        w = torch.randn(B, heads, cap, generator=g)
        w[..., 3::17], w[..., 5::19], w[..., 7::23], w[..., 8::29] = NAN, math.inf, -math.inf, -NAN
        return w
    _check_evict(dev, 4, 64, 2, 32, [700, 2500], 300, 2, 20, weights=weights)


def test_evict_bad_pages_short_tracker_and_given_workspace(dev):
    _check_evict(dev, 8, 64, 1, 16, [300, 200], 100, 0, 0, capacity=250)
    cache, table, n = _cache(dev, 40, 4, 64, 2, 16, [120, 120])
    table[0, 0], table[1, 6] = -1, cache.pages + 5
    tracker = SlotTracker(2, 2, 128, device=dev)
    tracker.weights.uniform_(generator=_gen(dev, 41))
    tracker.tokens.copy_(torch.arange(128, device=dev).expand(2, 2, 128))
    kc, w = cache.k_codes.clone(), tracker.weights.cpu()
    ws = evict_workspace(2, 2, 64, 128, dev)
    ws.fill_(255)
    seen = n.clone()
    evict_by_weight(cache, table, n, tracker, seen, 64, workspace=ws)
    tc = table.cpu().long()
    for b in range(2):
        for h in range(2):
            for src, dst in R.evict_ref(w[b, h].tolist(), list(range(128)), 120, 120, 64, 0, 0):
                ps, pd = int(tc[b, src // 16]), int(tc[b, dst // 16])
                if 0 <= ps < cache.pages and 0 <= pd < cache.pages:
                    kc[pd, h, dst % 16] = cache.k_codes[ps, h, src % 16]
    assert torch.equal(cache.k_codes, kc)


# ---- together --------------------------------------------------------------------------------------------------

def test_prompt_decode_evict_together(dev):
    """Prompts attended and coded into the cache, decode steps with weights, an eviction, more steps: every attention
    against the plain form over the cache as it is, and the cache against what PolarQuant and the rules say."""
    from aetherkv.prompt import prompt_attention

    heads, group, dim, page, keep = 2, 3, 128, 16, 48
    H, lens, steps = heads * group, [90, 33, 61], 4
    pq = PolarQuant(4)
    gen = _gen(dev, 50)
    table = torch.randperm(27, device=dev, generator=gen)[:24].to(torch.int32).view(3, 8)
    cache = PagedKVCache(pq, 27, heads, dim, page_size=page, device=dev)
    tracker = SlotTracker(3, heads, 128, device=dev)
    lengths = torch.zeros(3, dtype=torch.int32, device=dev)
    seen = torch.zeros(3, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 90, 123, 184], dtype=torch.int32, device=dev)
    qkv = torch.randn(184, H + 2 * heads, dim, device=dev, generator=gen).to(torch.bfloat16)
    q, k, v = qkv[:, :H], qkv[:, H:H + heads], qkv[:, H + heads:]
    out = prompt_attention(q, k, v, cu, dim ** -0.5)
    want, bound, _, _ = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), cu.tolist(), cu.tolist(), dim ** -0.5)
    R.within(out, want, bound, "prompt")
    append_tokens(cache, k, v, table, lengths, cu_seqlens=cu, tracker=tracker, token=seen)
    new = torch.tensor(lens, dtype=torch.int32, device=dev)
    lengths += new
    seen += new
    kk, vv = cache.decode(table[0], 90, torch.float32)
    for got, x in ((kk, k), (vv, v)):
        assert torch.equal(got, pq.decode(*pq.encode(x[:90].contiguous()), out_dtype=torch.float32).transpose(0, 1))

    def step():
        qkv = torch.randn(3, 1, H + 2 * heads, dim, device=dev, generator=gen).to(torch.bfloat16)
        append_tokens(cache, qkv[:, :, H:H + heads], qkv[:, :, H + heads:], table, lengths, tracker=tracker, token=seen)
        lengths.add_(1)
        seen.add_(1)
        before = tracker.weights.double().cpu()
        out = paged_attention(qkv[:, :, :H], cache, table, lengths, dim ** -0.5, tracker=tracker)
        want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, table), qkv[:, :, :H].cpu(), lengths.tolist(), dim ** -0.5, capacity=128)
        R.within(out, want, bound, "step")
        R.within(tracker.weights, before + w, wb + 2.0 ** -23 * (before + w), "weights")

    for _ in range(steps):
        step()
    kept = []
    for b, n in enumerate(lengths.tolist()):
        for h in range(heads):
            w, t = tracker.weights[b, h].tolist(), tracker.tokens[b, h].tolist()
            slots = list(range(min(n, keep)))
            for src, dst in R.evict_ref(w, t, n, int(seen[b]), keep, 4, 8):
                slots[dst] = src
            kept.append([t[i] for i in slots])
    evict_by_weight(cache, table, lengths, tracker, seen, keep, first=4, recent=8)
    lengths.clamp_(max=keep)
    for b, n in enumerate(lengths.tolist()):
        for h in range(heads):
            assert tracker.tokens[b, h, :n].tolist() == kept[b * heads + h]
            assert set(range(4)) | set(range(int(seen[b]) - 8, int(seen[b]))) <= set(kept[b * heads + h])
    for _ in range(steps):
        step()


def test_step_captured_and_replayed(dev):
    """One captured graph of a whole step (append, attention with weights, eviction), replayed among eager work and equal
    to the eager calls on copies every time."""
    heads, H, dim, page, keep = 2, 6, 128, 16, 64
    cache, table, n = _cache(dev, 60, 4, dim, heads, page, [64, 40])
    table = torch.arange(12, dtype=torch.int32, device=dev).view(2, 6)[:, :5].contiguous()
    tracker = SlotTracker(2, heads, 80, device=dev)
    tracker.weights.uniform_(generator=_gen(dev, 61))
    tracker.tokens.copy_(torch.arange(80, device=dev).expand(2, heads, 80))
    lengths, seen = n.clone(), n.clone()
    qkv = torch.randn(2, 1, H + 2 * heads, dim, device=dev, generator=_gen(dev, 62)).to(torch.bfloat16)

    def step(c, t, ln, sn):
        append_tokens(c, qkv[:, :, H:H + heads], qkv[:, :, H + heads:], table, ln, tracker=t, token=sn)
        ln.add_(1)
        sn.add_(1)
        out = paged_attention(qkv[:, :, :H], c, table, ln, dim ** -0.5, tracker=t)
        evict_by_weight(c, table, ln, t, sn, keep, first=2, recent=4)
        ln.clamp_(max=keep)
        return out

    def copy():
        c = PagedKVCache.from_tensors(cache.quant, *(x.clone() for x in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)))
        return c, SlotTracker.from_tensor(tracker.storage.clone()), lengths.clone(), seen.clone()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*copy())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(cache, tracker, lengths, seen)
    for rep in range(4):
        qkv.copy_(torch.randn(qkv.shape, device=dev, generator=_gen(dev, 70 + rep)))
        c, t, ln, sn = copy()
        want = step(c, t, ln, sn)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {rep}"
        assert torch.equal(tracker.storage, t.storage) and torch.equal(lengths, ln)
        for x, y in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), (c.k_codes, c.k_scale, c.v_codes, c.v_scale)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("bits,dim", [(4, 64), (4, 128), (8, 64), (8, 128)])
def test_evict_many_moves(dev, bits, dim):
    """More moves than the selecting workgroup makes by itself (256), and as many."""
    _check_evict(dev, bits, dim, 2, 16, [700, 560, 301, 300], 300, 4, 10, seed=bits + dim)
    _check_evict(dev, bits, dim, 1, 16, [512, 300], 256, 4, 10, seed=bits + dim)


@pytest.mark.parametrize("keep", [200, 19900])
def test_evict_few_moves_of_long_rows(dev, keep):
    _check_evict(dev, 4, 64, 2, 256, [20000, 17000], keep, 4, 64, seed=keep)


@pytest.mark.parametrize("bits,dim", [(4, 64), (4, 128), (8, 64), (8, 128)])
def test_attention_more_rows_than_the_weights_pass_holds(dev, bits, dim):
    _check_attention(dev, bits, dim, torch.bfloat16, 16, 1, 3, 70, [90, 33, 150], True, True, seed=bits + dim)


def test_workspaces_that_are_no_bytes_are_refused(dev):
    from aetherkv.prompt import prompt_attention

    cache = PagedKVCache(PolarQuant(4), 4, 2, 64, page_size=16, device=dev)
    table = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    n = torch.full((1,), 3, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device=dev)
    for ws in (torch.empty(1 << 16, dtype=torch.float32, device=dev), torch.empty(1 << 17, dtype=torch.uint8, device=dev)[::2]):
        with pytest.raises(RuntimeError, match="workspace"):
            paged_attention(q, cache, table, n, 0.1, workspace=ws)
        with pytest.raises(RuntimeError, match="workspace"):
            evict_by_weight(cache, table, n, SlotTracker(1, 2, 64, device=dev), n, 1, workspace=ws)
        with pytest.raises(RuntimeError, match="workspace"):
            prompt_attention(q[0], q[0], q[0], torch.tensor([0, 1], dtype=torch.int32, device=dev), 0.1, workspace=ws)


@pytest.mark.parametrize("B,heads", [(50, 16), (66, 12)])
def test_attention_of_a_ragged_batch_longest_first(dev, B, heads):
    """Batches of more workgroups than run together start their longest sequences first (up to 64 sequences and beyond in
    two forms): lengths of one bucket, equal ones, none, the longest last."""
    lens = [(0, 3, 17, 18, 1, 40, 17, 33)[i % 8] for i in range(B)]
    lens[1], lens[-2], lens[-1] = 300, 290, 4096
    _check_attention(dev, 4, 64, torch.bfloat16, 16, heads, 1, 1, lens, False, True, seed=B)


@pytest.mark.parametrize("length", [8191, 8192, 8193])
def test_evict_around_the_rows_of_more_waves(dev, length):
    _check_evict(dev, 8, 128, 1, 16, [length, length - 100, 90], length - 200, 4, 64, seed=length)
    _check_evict(dev, 4, 64, 1, 16, [length, length // 2], length // 3, 4, 64, seed=length)


@pytest.mark.parametrize("shape", ["three each", "one each", "short packed", "packed from the second row on"])
def test_append_large_calls_of_many_sequences(dev, shape):
    """A wave's tokens of a large call belong to many sequences: equal ones, and packed ones with empty ones between."""
    heads, dim, page = 4, 128, 16
    if shape.endswith("each"):
        B, T = (1400, 3) if shape[0] == "t" else (2100, 1)
        lens, off = [T] * B, 0
    else:
        lens, off = [(0, 1, 0, 5, 2, 0, 0, 40, 3)[i % 9] for i in range(450)], (1 if "second" in shape else 0)
        B, T = len(lens), 0
    cache, table, _ = _cache(dev, 60, 4, dim, heads, page, [max(lens) + 16] * B)
    N = off + sum(lens) + (3 if not T else 0)
    k, v = (torch.randn(N, heads, dim, device=dev, generator=_gen(dev, 61 + i)).to(torch.bfloat16) for i in range(2))
    cu = [off]
    for n in lens:
        cu.append(cu[-1] + n)
    start = [b % 16 for b in range(B)]
    assert N * 2 * heads * dim >= 1 << 21
    tracker = SlotTracker(B, heads, table.size(1) * page, device=dev)
    tracker.weights.fill_(9.0)
    token = torch.arange(B, dtype=torch.int32, device=dev) * 100
    want = _expect_append(cache, k, v, table.cpu(), start, cu)
    args = dict(tracker=tracker, token=token)
    if T:
        k, v = k.view(B, T, heads, dim), v.view(B, T, heads, dim)
    else:
        args["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    append_tokens(cache, k, v, table, torch.tensor(start, dtype=torch.int32, device=dev), **args)
    for got, w in zip((cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale), want):
        assert torch.equal(got, w)
    i = torch.arange(tracker.capacity, device=dev)[None] - torch.tensor(start, device=dev)[:, None]
    new = ((i >= 0) & (i < torch.tensor(lens, device=dev)[:, None]))[:, None].expand_as(tracker.weights)
    assert torch.equal(tracker.weights, torch.where(new, 0.0, 9.0))
    assert torch.equal(tracker.tokens[new], (token[:, None] + i)[:, None].expand_as(new)[new].int())


def test_attention_shared_and_repeated_pages(dev):
    """Pages that sequences share, and a page that a sequence has twice; a query expanded over the heads."""
    cache = _fill(dev, 80, 4, 128, 2, 16, 9)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [6, 6, 6, 7]], dtype=torch.int32, device=dev)
    n = torch.tensor([64, 50, 60], dtype=torch.int32, device=dev)
    q = torch.randn(3, 1, 1, 128, device=dev, generator=_gen(dev, 81)).to(torch.bfloat16).expand(3, 1, 6, 128)
    tracker = SlotTracker(3, 2, 64, device=dev)
    got = paged_attention(q, cache, table, n, 0.1, tracker=tracker)
    want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, table), q.cpu(), n.tolist(), 0.1, None, 64)
    R.within(got, want, bound, "out")
    R.within(tracker.weights, w, wb + 2.0 ** -23 * w, "weights")


@pytest.mark.parametrize("T", [1, 9])
def test_long_tracked_attention_in_two_graphs_and_streams(dev, T):
    """Two captured calls in pieces, with logits (T = 1) and with the scores again (T = 9), replayed on two streams at once
    and among eager calls: each graph has a workspace of its own."""
    heads, H, dim, page, lens = 2, 6, 64, 64, [3000, 700, 0]
    cache, table, n = _cache(dev, 82, 8, dim, heads, page, lens)
    q = torch.randn(2, 3, T, H, dim, device=dev, generator=_gen(dev, 83)).to(torch.float16)
    trackers = [SlotTracker(3, heads, table.size(1) * page, device=dev) for _ in range(3)]
    call = lambda i, t: paged_attention(q[i], cache, table, n, 0.125, tracker=trackers[t])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0, 2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            outs.append(call(i, i))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(3):
        q.copy_(torch.randn(q.shape, device=dev, generator=_gen(dev, 90 + rep)))
        want, weights = [], []
        for i in range(2):
            trackers[2].storage.zero_()
            want.append(call(i, 2).clone())
            weights.append(trackers[2].weights.clone())
            trackers[i].storage.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        call(0, 2)
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i]) and torch.equal(trackers[i].weights, weights[i]), f"graph {i}, replay {rep}"


# ---- bounds of sequences and trackers ----------------------------------------------------------------------------

def _ref_by_token(cache, table, q, lengths, scale, sink, capacity):
    """The plain form one token at a time: token t of T is the newest one of a sequence of lengths - T + 1 + t slots, of which
    those past the table, or the tracker, are cut off."""
    B, T, H, _ = q.shape
    parts = [R.paged_attention_ref(R.HostCache(cache, table), q[:, t:t + 1].cpu(), [n - T + 1 + t for n in lengths], scale,
                                   None if sink is None else sink.cpu(), capacity) for t in range(T)]
    out, bound, w, wb = zip(*parts)
    # (the tokens' weights add up in fp32: T additions)
    return torch.cat(out, 1), torch.cat(bound, 1), sum(w), sum(wb) + 2.0 ** -23 * T * sum(w)


@pytest.mark.parametrize("bits,dim", [(4, 64), (8, 128)])
@pytest.mark.parametrize("T,group", [(4, 2), (9, 2), (3, 7)])
@pytest.mark.parametrize("lengths,slots,capacity", [([90, 72, 71, 70, 40], 96, 70), ([5000, 97, 99, 96, 3], 96, None), ([5000, 98, 96, 2, 0], 96, 96),
                                                    ([2 ** 31 - 1, 1283, 1290, -(2 ** 31)], 1280, None), ([1282, 1279, 1300], 1280, 1276)])
def test_attention_causal_bound_of_lengths_past_the_end(dev, bits, dim, T, group, lengths, slots, capacity):
    """The causal bound counts back from the given length; what lies past the table or the tracker is cut off afterwards, so
    that earlier tokens of a sequence that is longer than both see all that is there."""
    heads, page, B = 2, 16, len(lengths)
    cache, table, _ = _cache(dev, 100 + T, bits, dim, heads, page, [slots] * B)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    q = torch.randn(B, T, heads * group, dim, device=dev, generator=_gen(dev, 101)).to(torch.bfloat16)
    sink = torch.randn(heads * group, device=dev, generator=_gen(dev, 102))
    tracker = None
    if capacity is not None:
        tracker = SlotTracker(B, heads, capacity, device=dev)
        tracker.weights.uniform_(0, 3, generator=_gen(dev, 103))
        before = tracker.weights.double().cpu()
    got = paged_attention(q, cache, table, n, dim ** -0.5, sink=sink, tracker=tracker)
    want, bound, w, wb = _ref_by_token(cache, table, q, lengths, dim ** -0.5, sink, capacity)
    R.within(got, want, bound, "out")
    if tracker is not None:
        R.within(tracker.weights, before + w, wb + 2.0 ** -23 * (before + w), "weights")


@pytest.mark.parametrize("T,group", [(2, 2), (3, 5), (9, 2), (12, 3)])
@pytest.mark.parametrize("length", [60, 1290])
def test_attention_nan_row_leaves_the_weights_of_slots_it_does_not_see(dev, T, group, length):
    """A query that holds NaN adds NaN to the slots that it sees, and nothing to a missing page's or to later tokens' slots."""
    heads, dim, page = 2, 64, 16
    cache, table, n = _cache(dev, 110, 4, dim, heads, page, [length, length])
    table[0, 1] = -1
    q = torch.randn(2, T, heads * group, dim, device=dev, generator=_gen(dev, 111)).to(torch.bfloat16)
    clean, got = (SlotTracker(2, heads, table.size(1) * page, device=dev) for _ in range(2))
    for t in (clean, got):
        t.weights.uniform_(0, 3, generator=_gen(dev, 112))
    paged_attention(q, cache, table, n, 0.125, tracker=clean)
    q[0, 0, 1] = NAN  # the first token, KV head 0: it does not see the last T - 1 slots
    paged_attention(q, cache, table, n, 0.125, tracker=got)
    sees = torch.zeros(2, heads, clean.capacity, dtype=torch.bool, device=dev)
    sees[0, 0, :length - T + 1] = True
    sees[0, 0, page:2 * page] = False
    assert got.weights[sees].isnan().all()
    assert torch.equal(got.weights[~sees], clean.weights[~sees])


def test_decode_of_missing_pages_and_past_the_table(dev):
    """PagedKVCache.decode gives 0 for the slots of a page that a table does not have, and refuses what lies past the table."""
    cache, table, _ = _cache(dev, 120, 4, 64, 2, 16, [60])
    want = cache.decode(table[0], 60, torch.float32)
    row = table[0].clone()
    row[1] = -1
    row[3] = cache.pages
    for got, w in zip(cache.decode(row, 60, torch.float32), want):
        assert not got[:, 16:32].any() and torch.equal(got[:, :16], w[:, :16]) and torch.equal(got[:, 32:48], w[:, 32:48])
        assert not got[:, 48:].any()
    assert all(x.shape == (2, 64, 64) for x in cache.decode(table[0], 64))
    assert all(x.shape == (2, 0, 64) for x in cache.decode(table[0], 0))
    for length in (65, 1000, -1):
        with pytest.raises(RuntimeError, match="slots"):
            cache.decode(table[0], length)
    with pytest.raises(RuntimeError, match="page_table"):
        cache.decode(table, 60)
    empty = PagedKVCache.from_tensors(cache.quant, cache.k_codes[:0], cache.k_scale[:0], cache.v_codes[:0], cache.v_scale[:0])
    assert all(x.shape == (2, 20, 64) and not x.any() for x in empty.decode(table[0], 20))


@pytest.mark.parametrize("given", [False, True])
def test_first_calls_of_a_cache_captured(dev, given):
    """A cache whose quantiser has coded nothing yet: its first append and attention may be the captured ones."""
    heads, dim, page = 2, 64, 16
    k, v = (torch.randn(2, 1, heads, dim, device=dev, generator=_gen(dev, 130 + i)).to(torch.bfloat16) for i in range(2))
    q = torch.randn(2, 1, 4, dim, device=dev, generator=_gen(dev, 132)).to(torch.bfloat16)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    zero = torch.zeros(2, dtype=torch.int32, device=dev)

    def make():
        c = PagedKVCache(PolarQuant(4, seed=7), 4, heads, dim, page_size=page, device=dev)
        return PagedKVCache.from_tensors(PolarQuant(4, seed=7), c.k_codes, c.k_scale, c.v_codes, c.v_scale) if given else c

    def step(c):
        append_tokens(c, k, v, table, zero)
        return paged_attention(q, c, table, zero + 1, 0.125)

    eager, captured = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step(eager)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(captured)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(captured.k_codes, eager.k_codes) and torch.equal(captured.v_scale, eager.v_scale)


def test_attention_large_workspace_is_given_back(dev):
    """A tracked call over a wide table takes more workspace than is kept between calls: the same results, nothing held."""
    cache, few, n = _cache(dev, 140, 4, 64, 2, 16, [100, 37, 0, 64])
    wide = torch.full((4, 1 << 16), -1, dtype=torch.int32, device=dev)
    wide[:, :few.size(1)] = few
    q = torch.randn(4, 2, 16, 64, device=dev, generator=_gen(dev, 141)).to(torch.bfloat16)
    size = paged_attention_workspace(4, 2, 16, 2, 64, wide.numel() // 4 * 16, "meta", tracked=True).numel()
    assert size > 64 << 20
    tracker = SlotTracker(4, 2, wide.size(1) * 16, device=dev)
    paged_attention(q, cache, few, n, 0.125, tracker=SlotTracker(4, 2, few.size(1) * 16, device=dev))
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated(dev)
    got = paged_attention(q, cache, wide, n, 0.125, tracker=tracker)
    want, bound, w, wb = R.paged_attention_ref(R.HostCache(cache, few), q.cpu(), n.tolist(), 0.125, capacity=112)
    R.within(got, want, bound, "out")
    del got
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(dev) - held < 1 << 20
    R.within(tracker.weights[..., :112], w, wb, "weights")
    assert not tracker.weights[..., 112:].any()


@pytest.mark.parametrize("keep,slots", [(16, 32), (300, 608)])
def test_evict_more_rows_than_a_grid_dimension(dev, keep, slots):
    """70000 (sequence, KV head) rows, with the moves made by the selecting workgroup and by a launch of their own."""
    B, heads, page = (1000, 70, 16) if slots < 300 else (5000, 14, 16)
    lens = torch.randint(0, slots + 1, (B,), generator=torch.Generator().manual_seed(1))
    lens[-1] = slots
    per = slots // page
    codes = torch.randint(0, 256, (2, B * per, heads, page, 32), dtype=torch.uint8, device=dev, generator=_gen(dev, 150))
    scale = torch.rand(2, B * per, heads, page, device=dev, generator=_gen(dev, 151))
    cache = PagedKVCache.from_tensors(PolarQuant(4), codes[0], scale[0], codes[1], scale[1])
    table = torch.arange(B * per, dtype=torch.int32, device=dev).view(B, per)
    tracker = SlotTracker(B, heads, slots, device=dev)
    # weights that are all different: a permutation of each row's places
    tracker.weights.copy_(torch.rand(B, heads, slots, device=dev, generator=_gen(dev, 152)).argsort(-1))
    tracker.tokens.copy_(torch.arange(slots, device=dev).expand(B, heads, slots))
    n = lens.to(torch.int32).to(dev)
    weights = tracker.weights.clone()
    rows = lambda c: c.view(B, per, heads, page, -1).transpose(1, 2).reshape(B, heads, slots, -1)  # noqa: E731
    before = [rows(x).clone() for x in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    evict_by_weight(cache, table, n, tracker, n, keep)
    # stays[slot], and the source of every slot below keep: itself, or for the i-th hole the i-th slot that moves
    there = torch.arange(slots, device=dev) < n[:, None, None]
    rank = weights.masked_fill(~there, -1.0).argsort(-1, descending=True)
    stays = torch.zeros_like(there.expand_as(weights)).scatter_(-1, rank[..., :keep], True) & there
    place = torch.arange(slots, device=dev).expand_as(weights)
    hole = ~stays & (place < keep) & (n > keep)[:, None, None]
    mover = stays & (place >= keep)
    assert torch.equal(hole.sum(-1), mover.sum(-1))
    source = place.clone()
    source[hole] = place[mover]  # (both in row-major order)
    for got, x in zip((cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale), before):
        assert torch.equal(rows(got), x.gather(2, source[..., None].expand_as(x)))
    assert torch.equal(tracker.tokens.long(), source) and torch.equal(tracker.weights, weights.gather(-1, source))
