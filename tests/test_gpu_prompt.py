"""Causal prompt attention over packed sequences on the GPU against the plain 64-bit form (paged_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

import paged_ref as R
from aetherkv.prompt import prompt_attention

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _inputs(dev, seed, dtype, dim, H, hk, lq, lk, pad=0, gain=1.0):
    nq, nk = sum(lq) + pad, sum(lk) + pad
    if lq == lk:  # one projection's rows
        qkv = torch.randn(nq, H + 2 * hk, dim, device=dev, generator=_gen(dev, seed))
        qkv[:, :H] *= gain
        qkv = qkv.to(dtype)
        return qkv[:, :H], qkv[:, H:H + hk], qkv[:, H + hk:]
    q = (torch.randn(nq, H, dim, device=dev, generator=_gen(dev, seed)) * gain).to(dtype)
    kv = torch.randn(nk, 2, hk, dim, device=dev, generator=_gen(dev, seed + 1)).to(dtype)
    return q, kv[:, 0], kv[:, 1]


def _check(dev, dtype, dim, H, hk, lq, lk=None, sink=False, pad=0, seed=0, gain=1.0, scale=None):
    lk = lq if lk is None else lk
    q, k, v = _inputs(dev, seed, dtype, dim, H, hk, lq, lk, pad, gain)
    cq, ck = _cu(lq), _cu(lk)
    sk = torch.randn(H, device=dev, generator=_gen(dev, seed + 2)) if sink else None
    scale = dim ** -0.5 if scale is None else scale
    out, lse = prompt_attention(q, k, v, torch.tensor(cq, dtype=torch.int32, device=dev), scale,
                                cu_seqlens_k=None if lq == lk else torch.tensor(ck, dtype=torch.int32, device=dev), sink=sk, return_lse=True)
    want, bound, wl, lb = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), cq, ck, scale, None if sk is None else sk.cpu())
    R.within(out, want, bound, "out")
    got = lse.double().cpu()
    none = wl == -math.inf
    assert torch.equal(got == -math.inf, none)
    R.within(got[~none], wl[~none], lb[~none], "lse")
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_prompt_lengths(dev, dtype, dim, n):
    _check(dev, dtype, dim, 2, 1, [n], seed=n)


@pytest.mark.parametrize("H,hk", [(1, 1), (3, 3), (12, 4), (12, 1), (16, 2), (10, 2)])
def test_prompt_head_layouts(dev, H, hk):
    _check(dev, torch.bfloat16, 128, H, hk, [70, 33], sink=True, seed=H)


@pytest.mark.parametrize("lens", [[0], [0, 5, 0, 0, 130, 1], [1] * 70, [300, 1, 64, 65], [17, 200, 129]])
@pytest.mark.parametrize("pad", [0, 3])
def test_prompt_packed(dev, lens, pad):
    if sum(lens) + pad == 0:
        out = prompt_attention(*(torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(3)), torch.zeros(2, dtype=torch.int32, device=dev), 0.1)
        assert out.shape == (0, 2, 64)
        return
    out, lse = _check(dev, torch.bfloat16, 64, 4, 2, lens, pad=pad, seed=len(lens))
    if pad:
        assert not out[-pad:].any() and (lse[-pad:] == -math.inf).all()


@pytest.mark.parametrize("lq,lk", [([1], [200]), ([5, 64, 1], [6, 300, 129]), ([130], [131]), ([64], [64 + 1000]), ([40, 7], [20, 0]), ([100, 3], [30, 3])])
@pytest.mark.parametrize("sink", [False, True])
def test_prompt_chunks(dev, lq, lk, sink):
    """More keys than queries, and fewer: the first queries then see nothing."""
    out, _ = _check(dev, torch.float16, 128, 4, 2, lq, lk, sink=sink, seed=sum(lk))
    if lq == [40, 7]:
        assert not out[:20].any() and not out[40:].any()


def test_prompt_long(dev):
    _check(dev, torch.bfloat16, 128, 1, 1, [1300], seed=5)
    _check(dev, torch.float16, 64, 2, 1, [900, 513], seed=6)


def test_prompt_peaked_flat_and_negative_scale(dev):
    _check(dev, torch.float16, 64, 2, 2, [150], gain=20.0)
    _check(dev, torch.bfloat16, 128, 2, 2, [150], scale=0.0)
    _check(dev, torch.bfloat16, 64, 2, 2, [150], scale=-0.3, sink=True)


def test_prompt_rows_behind_the_last_are_left(dev):
    q, k, v = _inputs(dev, 8, torch.bfloat16, 64, 4, 2, [60], [60], pad=10)
    cu = torch.tensor([0, 60], dtype=torch.int32, device=dev)
    out = torch.full((70, 4, 64), 7.0, dtype=torch.bfloat16, device=dev)
    assert prompt_attention(q, k, v, cu, 0.125, out=out).data_ptr() == out.data_ptr()
    assert (out[60:] == 7).all()
    assert torch.equal(out[:60], prompt_attention(q[:60], k[:60], v[:60], cu, 0.125))
    mid = torch.tensor([5, 20, 20, 50], dtype=torch.int32, device=dev)  # rows before the first too
    out.fill_(7.0)
    prompt_attention(q, k, v, mid, 0.125, out=out)
    assert (out[:5] == 7).all() and (out[50:] == 7).all()
    want, bound, _, _ = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), [5, 20, 20, 50], [5, 20, 20, 50], 0.125)
    R.within(out[5:50], want[5:50], bound[5:50], "out")


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_masked_places_do_not_matter(dev, bad, dtype):
    """Entries that a row does not see may hold anything: later tokens, other sequences, rows behind the last."""
    q, k, v = (x.clone() for x in _inputs(dev, 9, dtype, 128, 2, 1, [100, 90], [100, 90], pad=20))
    cu = torch.tensor([0, 100, 190], dtype=torch.int32, device=dev)
    clean, clean_lse = prompt_attention(q, k, v, cu, 0.09, return_lse=True)
    for x in (k, v):
        x[190:] = bad
        x[60, 0, ::7] = bad
        x[180] = bad
    got, lse = prompt_attention(q, k, v, cu, 0.09, return_lse=True)
    for rows in (slice(0, 60), slice(100, 180)):
        assert torch.equal(got[rows], clean[rows]) and torch.equal(lse[rows], clean_lse[rows])
    if bad != bad:
        assert got[60:100].isnan().any(-1).all() and got[180:190].isnan().all()


def test_prompt_infinite_value_reaches_the_rows_that_see_it(dev):
    q, k, v = (x.clone() for x in _inputs(dev, 10, torch.bfloat16, 128, 2, 1, [100], [100]))
    cu = torch.tensor([0, 100], dtype=torch.int32, device=dev)
    clean = prompt_attention(q, k, v, cu, 0.09)
    v[70, 0, 5], v[40, 0, 6] = math.inf, -math.inf
    got = prompt_attention(q, k, v, cu, 0.09)
    assert (got[70:, :, 5] == math.inf).all() and (got[40:, :, 6] == -math.inf).all()
    got[70:, :, 5], got[40:, :, 6] = clean[70:, :, 5], clean[40:, :, 6]
    assert torch.equal(got, clean)


def test_prompt_strides_streams_and_devices(dev):
    q, k, v = _inputs(dev, 11, torch.bfloat16, 128, 4, 2, [130, 40], [130, 40])
    cu = torch.tensor([0, 130, 170], dtype=torch.int32, device=dev)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, 0.09)
    assert torch.equal(prompt_attention(q, k, v, cu.long(), 0.09), want)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*heads_first, cu, 0.09), want)
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device=dev)[1:].view(x.shape).copy_(x) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*odd, cu, 0.09), want)
    shared = k[:, :1].expand(-1, 2, -1)  # one head under two names
    assert torch.equal(prompt_attention(q, shared, v, cu, 0.09), prompt_attention(q, shared.contiguous(), v, cu, 0.09))
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(s[i % 2]):
            outs.append(prompt_attention(q, k, v, cu, 0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_prompt_captured_and_replayed(dev):
    q, k, v = (x.clone() for x in _inputs(dev, 12, torch.bfloat16, 128, 6, 2, [100, 60], [100, 60], pad=8))
    cu = torch.tensor([0, 100, 160], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt_attention(q, k, v, cu, 0.09, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = prompt_attention(q, k, v, cu, 0.09, return_lse=True)
    for rep, lens in enumerate(([0, 100, 160], [0, 7, 168], [0, 168, 168], [3, 3, 90])):
        q.copy_(torch.randn(q.shape, device=dev, generator=_gen(dev, rep)))
        cu.copy_(torch.tensor(lens, dtype=torch.int32))
        want, wl = prompt_attention(q, k, v, cu, 0.09, return_lse=True)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wl), f"replay {rep}"


def test_prompt_refusals(dev):
    q, k, v = _inputs(dev, 13, torch.bfloat16, 128, 4, 2, [50], [50])
    cu = torch.tensor([0, 50], dtype=torch.int32, device=dev)
    for args in ((q.float(), k, v, cu), (q, k.half(), v, cu), (q[:, :3], k, v, cu), (q, k, v[:, :1], cu), (q[:40], k, v, cu), (q, k, v, cu[:1]), (q, k, v, cu.cpu()),
                 (q, k, v, cu.float()), (q[..., :96], k[..., :96], v[..., :96], cu), (q[0], k, v, cu)):
        with pytest.raises(RuntimeError):
            prompt_attention(*args, 0.09)
    with pytest.raises(RuntimeError):
        prompt_attention(q, k, v, cu, 0.09, sink=torch.zeros(3, device=dev))
    with pytest.raises(RuntimeError):
        prompt_attention(q, k, v, cu, 0.09, out=torch.empty(50, 4, 64, dtype=torch.bfloat16, device=dev))
    with pytest.raises(RuntimeError):
        prompt_attention(q, k, v, cu, 0.09, cu_seqlens_k=torch.zeros(3, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("dtype,dim,H,hk,lens", [(torch.bfloat16, 128, 16, 8, [3000, 1, 1203, 64]), (torch.float16, 64, 32, 8, [2500]), (torch.bfloat16, 64, 24, 12, [700] * 5)])
def test_prompt_many_rows(dev, dtype, dim, H, hk, lens):
    """Launches of many rows take larger row tiles: sampled rows of every sequence against the plain form in 64 bits."""
    q, k, v = _inputs(dev, 20, dtype, dim, H, hk, lens, lens, pad=2)
    cu = _cu(lens)
    scale = dim ** -0.5
    out, lse = prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), scale, return_lse=True)
    assert not out[cu[-1]:].any() and (lse[cu[-1]:] == -math.inf).all()
    for b, n in enumerate(lens):
        kk, vv = (x[cu[b]:cu[b + 1]].cpu() for x in (k, v))
        rows = sorted({0, n - 1, n // 2, *(int(i) for i in torch.randint(0, n, (6,), generator=torch.Generator().manual_seed(b)))})
        for i in rows:
            one = q[cu[b] + i:cu[b] + i + 1].cpu()
            want, bound, wl, lb = R.prompt_attention_ref(one, kk[:i + 1], vv[:i + 1], [0, 1], [0, i + 1], scale)
            R.within(out[cu[b] + i:cu[b] + i + 1], want, bound, f"row {i} of {b}")
            R.within(lse[cu[b] + i:cu[b] + i + 1].double().cpu(), wl, lb, f"lse of row {i} of {b}")


def test_prompt_many_rows_masked_places(dev):
    """The larger row tiles keep what a row does not see out of it as the others do."""
    lens, H, hk, dim = [2300, 2000], 16, 8, 128
    q, k, v = (x.clone() for x in _inputs(dev, 21, torch.bfloat16, dim, H, hk, lens, lens, pad=5))
    cu = torch.tensor(_cu(lens), dtype=torch.int32, device=dev)
    clean = prompt_attention(q, k, v, cu, 0.09)
    for x in (k, v):
        x[4300:] = NAN
        x[1111, 3] = NAN
        x[2300 + 1990] = math.inf
    got = prompt_attention(q, k, v, cu, 0.09)
    assert torch.equal(got[:1111], clean[:1111]) and torch.equal(got[2300:2300 + 1990], clean[2300:2300 + 1990])
    assert torch.equal(got[1111:2300, :6], clean[1111:2300, :6]) and torch.equal(got[1111:2300, 8:], clean[1111:2300, 8:])
    assert got[1111:2300, 6:8].isnan().all()


@pytest.mark.parametrize("dtype,dim,H,hk,lq,lk", [(torch.bfloat16, 128, 4, 2, [3, 1, 70], [1500, 513, 2100]), (torch.float16, 64, 8, 1, [1], [5003]), (torch.bfloat16, 64, 2, 2, [600], [600]),
                                                  (torch.float16, 128, 12, 4, [5, 0, 40], [100, 3000, 1030]), (torch.bfloat16, 64, 2, 2, [2000], [2000])])
@pytest.mark.parametrize("sink", [False, True])
def test_prompt_few_rows_over_many_keys(dev, dtype, dim, H, hk, lq, lk, sink):
    """Launches of few rows split the keys over workgroups: rows that see one piece, all of them, or none."""
    from aetherkv.prompt import prompt_workspace

    q, k, v = _inputs(dev, 30, dtype, dim, H, hk, lq, lk, pad=3)
    cq, ck = (torch.tensor(_cu(x), dtype=torch.int32, device=dev) for x in (lq, lk))
    # (600 queries over their own keys see too few for pieces to pay; 2000 do not)
    assert (prompt_workspace(len(lq), q.size(0), k.size(0), H, hk, dim, dev).numel() > 0) == (lk != [600])
    sk = torch.randn(H, device=dev, generator=_gen(dev, 31)) if sink else None
    scale = dim ** -0.5
    ws = prompt_workspace(len(lq), q.size(0), k.size(0), H, hk, dim, dev).fill_(255)
    out, lse = prompt_attention(q, k, v, cq, scale, cu_seqlens_k=ck, sink=sk, return_lse=True, workspace=ws)
    want, bound, wl, lb = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), _cu(lq), _cu(lk), scale, None if sk is None else sk.cpu())
    R.within(out, want, bound, "out")
    none = wl == -math.inf
    got = lse.double().cpu()
    assert torch.equal(got == -math.inf, none)
    R.within(got[~none], wl[~none], lb[~none], "lse")
    again, lse2 = prompt_attention(q, k, v, cq, scale, cu_seqlens_k=ck, sink=sk, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    given = torch.full_like(out, 5.0)
    prompt_attention(q, k, v, cq, scale, cu_seqlens_k=ck, sink=sk, out=given)
    assert (given[-3:] == 5).all() and torch.equal(given[:-3], out[:-3])


def test_prompt_split_masked_places_and_captured(dev):
    lq, lk, H, hk, dim = [50, 20], [1200, 700], 4, 2, 64
    q, k, v = (x.clone() for x in _inputs(dev, 32, torch.bfloat16, dim, H, hk, lq, lk, pad=2))
    cq, ck = (torch.tensor(_cu(x), dtype=torch.int32, device=dev) for x in (lq, lk))
    clean = prompt_attention(q, k, v, cq, 0.125, cu_seqlens_k=ck)
    for x in (k, v):
        x[1190], x[1200 + 699], x[1900:] = NAN, math.inf, NAN
    got = prompt_attention(q, k, v, cq, 0.125, cu_seqlens_k=ck)
    assert torch.equal(got[:40], clean[:40]) and torch.equal(got[50:69], clean[50:69]) and got[40:50].isnan().all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt_attention(q, k, v, cq, 0.125, cu_seqlens_k=ck)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:  # two graphs, each with a workspace of its own
        with torch.cuda.graph(g):
            outs.append(prompt_attention(q, k, v, cq, 0.125, cu_seqlens_k=ck))
    for rep in range(3):
        q.copy_(torch.randn(q.shape, device=dev, generator=_gen(dev, rep)))
        k.copy_(torch.randn(k.shape, device=dev, generator=_gen(dev, 10 + rep)))
        v.copy_(torch.randn(v.shape, device=dev, generator=_gen(dev, 20 + rep)))
        want = prompt_attention(q, k, v, cq, 0.125, cu_seqlens_k=ck)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("B", [2, 63, 64, 65])
@pytest.mark.parametrize("H,hk,most", [(32, 32, 40), (48, 16, 90)])
def test_prompt_many_tiles_of_many_sequences(dev, B, H, hk, most):
    """More tiles than run together, of chunks with different numbers of keys before them, fewer keys than queries, and
    nothing: each row is written once, whatever the order that the tiles are taken in."""
    rng = torch.Generator().manual_seed(B)
    lq = [int(x) for x in torch.randint(0, most, (B,), generator=rng)]
    lk = [max(0, n + (0, 70, -3, 300)[i % 4]) for i, n in enumerate(lq)]
    if B == 2:
        lq, lk = [most * 9, most * 3], [most * 9, most * 3 + 700]
    _check(dev, torch.bfloat16, 64, H, hk, lq, lk, sink=True, seed=B, pad=2)


@pytest.mark.parametrize("dtype,dim,H,hk,lq,lk", [(torch.bfloat16, 128, 12, 4, [130, 1, 66], [66000, 66000, 40000]), (torch.float16, 64, 16, 2, [200], [33000])])
def test_prompt_wide_pieces(dev, dtype, dim, H, hk, lq, lk):
    """128 rows to a workgroup with the keys in pieces: enough work, few row tiles.  Checked on some rows."""
    q, k, v = _inputs(dev, 7, dtype, dim, H, hk, lq, lk)
    cq, ck = _cu(lq), _cu(lk)
    out = prompt_attention(q, k, v, torch.tensor(cq, dtype=torch.int32, device=dev), dim ** -0.5,
                           cu_seqlens_k=torch.tensor(ck, dtype=torch.int32, device=dev))
    for b, n in enumerate(lq):
        for i in sorted({0, n // 2, n - 1}):
            see = max(0, i + 1 + lk[b] - n)  # one query over the keys that it sees
            r = cq[b] + i
            one = slice(ck[b], ck[b] + see)
            want, bound, _, _ = R.prompt_attention_ref(q[r:r + 1].cpu(), k[one].cpu(), v[one].cpu(), [0, 1], [0, see], dim ** -0.5)
            R.within(out[r:r + 1], want, bound, f"sequence {b}, query {i}")


@pytest.mark.parametrize("B", [129, 4096, 4100])
def test_prompt_very_many_sequences(dev, B):
    """Sequences are searched 64 at a time: one round to 64, two to 4096, three beyond; with rows before the first one."""
    lq = [(1, 0, 2, 0, 3, 1)[i % 6] for i in range(B)]
    lq[B // 2] = 150
    q, k, v = _inputs(dev, 3, torch.bfloat16, 64, 2, 1, [5] + lq, [5] + lq, pad=4)
    cu = [c for c in _cu([5] + lq)[1:]]
    out, lse = prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), 0.125, return_lse=True)
    want, bound, wl, lb = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), cu, cu, 0.125)
    R.within(out, want, bound, "out")
    none = wl == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, none)
    R.within(lse.double().cpu()[~none], wl[~none], lb[~none], "lse")


@pytest.mark.parametrize("dtype,dim,H,hk,lq,lk", [(torch.bfloat16, 128, 16, 2, [512] * 8, [600] * 8), (torch.float16, 64, 32, 16, [200, 0, 333, 90, 512, 1, 400, 256] * 2, [300, 10, 400, 90, 700, 1500, 512, 300] * 2)])
def test_prompt_tiles_that_about_fill_the_chip(dev, dtype, dim, H, hk, lq, lk):
    """Several sequences whose 128-row tiles run together: every tile has its place, in the sequences' order without gaps.
    Checked on some rows, and every row against the call on its sequence alone, up to the kernels' own roundings."""
    q, k, v = _inputs(dev, 9, dtype, dim, H, hk, lq, lk, pad=3)
    cq, ck = _cu(lq), _cu(lk)
    out = prompt_attention(q, k, v, torch.tensor(cq, dtype=torch.int32, device=dev), dim ** -0.5,
                           cu_seqlens_k=torch.tensor(ck, dtype=torch.int32, device=dev))
    assert not out[cq[-1]:].any()
    for b, n in enumerate(lq):
        if n == 0:
            continue
        one = prompt_attention(q[cq[b]:cq[b + 1]], k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]], torch.tensor([0, n], dtype=torch.int32, device=dev), dim ** -0.5,
                               cu_seqlens_k=torch.tensor([0, lk[b]], dtype=torch.int32, device=dev))
        # (both are within the same bound of the exact value; values are below 6, weights sum to 1)
        tol = 4 * torch.finfo(dtype).eps
        assert ((out[cq[b]:cq[b + 1]].float() - one.float()).abs() <= tol * (1 + one.float().abs()) * 6).all(), f"sequence {b}"
        for i in sorted({0, n - 1}):
            see, r = max(0, i + 1 + lk[b] - n), cq[b] + i
            keys = slice(ck[b], ck[b] + see)
            want, bound, _, _ = R.prompt_attention_ref(q[r:r + 1].cpu(), k[keys].cpu(), v[keys].cpu(), [0, 1], [0, see], dim ** -0.5)
            R.within(out[r:r + 1], want, bound, f"sequence {b}, query {i}")


def _all_rows(q, k, v, lq, lk, scale, lift=0.0):
    """Every row's output in 64 bits, on the device, and its bound: u |out| + (u + 2 delta + (n + 16) 2^-24) sum p |v|, u of
    the type (the output's rounding, and each weight's), delta a logit's error, and `lift` times sum |v|, for weights below
    the type's normal numbers."""
    H, hk, D, u = q.size(1), k.size(1), q.size(2), R.U[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, R.TINY[q.dtype])
    cq, ck = _cu(lq), _cu(lk)
    for b in range(len(lq)):
        hidden = torch.arange(lk[b], device=q.device) > torch.arange(lq[b], device=q.device)[:, None] + lk[b] - lq[b]
        none = hidden.all(-1)
        for h in range(H):
            qq, kk, vv = q[cq[b]:cq[b + 1], h].double(), k[ck[b]:ck[b + 1], h // (H // hk)].double(), v[ck[b]:ck[b + 1], h // (H // hk)].double()
            if none.all():
                continue
            x = (qq @ kk.t() * scale).masked_fill_(hidden, -math.inf)
            p = torch.softmax(x, -1).masked_fill_(none[:, None], 0.0)
            o = p @ vv
            size = abs(scale) * (qq.abs() @ kk.abs().t()) * (D + 8) * 2.0 ** -24 + x.abs() * 2.0 ** -21
            delta = size.masked_fill_(hidden, 0.0).amax(-1, keepdim=True)
            n = (~hidden).sum(-1, keepdim=True)
            out[cq[b]:cq[b + 1], h] = o
            bound[cq[b]:cq[b + 1], h] += u * o.abs() + (u + 2 * delta + (n + 16) * 2.0 ** -24) * (p @ vv.abs()) + lift * ((~hidden).double() @ vv.abs())
    return out, bound


@pytest.mark.parametrize("dim,H,hk,lq,lk", [(64, 2, 1, [40], [16384]), (64, 48, 48, [1024], [16384]), (128, 8, 4, [3000, 64], [17000, 16384]), (64, 2, 2, [17000], [17000]),
                                            (128, 2, 1, [3, 5, 8], [20000, 33000, 16384])])
def test_prompt_small_weights_under_one_dominant_key(dev, dim, H, hk, lq, lk):
    """A first key that takes nearly all of the weight and holds no value: the output is made of the small weights alone, which
    have to keep their bits although they are far below the largest."""
    dtype, gap = torch.float16, 17.0
    q, k, v = (x.clone() for x in _inputs(dev, 40, dtype, dim, H, hk, lq, lk))
    q *= 0.3
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    v += 1.0
    for c in _cu(lk)[:-1]:
        k[c], v[c] = 0.0, 0.0
        k[c, :, 0] = gap * dim ** 0.5 / 8.0
    cu = lambda x: torch.tensor(_cu(x), dtype=torch.int32, device=dev)  # noqa: E731
    out = prompt_attention(q, k, v, cu(lq), dim ** -0.5, cu_seqlens_k=cu(lk))
    # a weight is held as 2^7 and up times exp2(its distance to the reference), the largest at 2^7 at least: one that is no
    # normal fp16 number is off by half of 2^-24, 2^-32 of the sum of weights
    want, bound = _all_rows(q, k, v, lq, lk, dim ** -0.5, lift=2.0 ** -32)
    R.within(out, want.cpu(), bound.cpu(), "out")


@pytest.mark.parametrize("dtype,size", [(torch.float16, 300.0), (torch.float16, 20000.0), (torch.bfloat16, 2.0 ** 14), (torch.bfloat16, 2.0 ** 40)])
@pytest.mark.parametrize("dim,H,hk,lq,lk", [(64, 4, 2, [150], [150]), (128, 2, 2, [20], [1500]), (128, 32, 16, [2100], [2100])])
def test_prompt_logits_far_from_zero(dev, dtype, size, dim, H, hk, lq, lk):
    """Logits so large that neighbouring fp32 numbers lie further apart than the exponentials reach: equal keys share the weight
    and a larger one takes it all, as where every logit is rounded to fp32 before the largest is subtracted."""
    q, k, v = (x.clone() for x in _inputs(dev, 41, dtype, dim, H, hk, lq, lk))
    q.fill_(size)
    k.fill_(size)
    first = lk[0] - lq[0] + 10  # the key that counts: the first ten queries do not see it
    k[first] = size * 1.25
    cu = lambda x: torch.tensor(_cu(x), dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = prompt_attention(q, k, v, cu(lq), dim ** -0.5, cu_seqlens_k=cu(lk), return_lse=True)
    vv = v.double().repeat_interleave(H // hk, 1)
    n = torch.arange(lk[0] - lq[0] + 1, first + 1, device=dev)[:, None, None]
    want = vv[first].expand(lq[0], H, dim).clone()
    want[:10] = vv.cumsum(0)[n[:, 0, 0] - 1] / n
    weight = want.abs()
    weight[:10] = vv.abs().cumsum(0)[n[:, 0, 0] - 1] / n
    # equal weights are rounded alike: the output's rounding, and the sums'
    u = R.U[dtype]
    R.within(out, want.cpu(), (u * want.abs() + (2 * u + (lk[0] + 16) * 2.0 ** -24) * weight + R.TINY[dtype]).cpu(), "out")
    top = torch.where(torch.arange(lq[0]) < 10, float(q[0, 0, 0]), float(k[first, 0, 0])).double() * size * dim ** 0.5
    count = torch.where(torch.arange(lq[0]) < 10, torch.arange(lq[0]) + lk[0] - lq[0] + 1, 1).double().log()
    # the product's sum, the scale in log2 units, and back: (dim + 8) roundings of the size of the logit
    R.within(lse.double().cpu(), (top + count)[:, None].expand(lq[0], H), ((dim + 8) * 2.0 ** -24 * top + 2.0 ** -20 * (1 + count))[:, None].expand(lq[0], H), "lse")


@pytest.mark.parametrize("lens", [[100], [4000]])
def test_prompt_far_row_leaves_its_neighbours_bits(dev, lens):
    q, k, v = (x.clone() for x in _inputs(dev, 44, torch.bfloat16, 128, 16, 8, lens, lens))
    cu = torch.tensor(_cu(lens), dtype=torch.int32, device=dev)
    clean = prompt_attention(q, k, v, cu, 0.09)
    q[70, 3] *= 2.0 ** 40
    got = prompt_attention(q, k, v, cu, 0.09)
    # the far row: the value of its largest logit
    top = (q[70, 3].double() @ k[:71, 1].double().t()).argmax()
    assert torch.equal(got[70, 3], v[top, 1])
    got[70, 3] = clean[70, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,H,hk,lq,lk", [(64, 4, 2, [40, 7, 90], [20, 0, 200]), (128, 2, 1, [30], [2000]), (128, 32, 16, [2100], [2000])])
def test_prompt_scale_that_is_no_number(dev, dtype, dim, H, hk, lq, lk):
    """A NaN scale gives NaN to every row that sees a key, as any other NaN would, and 0 to one that sees nothing."""
    q, k, v = _inputs(dev, 42, dtype, dim, H, hk, lq, lk)
    cu = lambda x: torch.tensor(_cu(x), dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = prompt_attention(q, k, v, cu(lq), NAN, cu_seqlens_k=cu(lk), return_lse=True)
    none = torch.cat([torch.arange(a) + b - a < 0 for a, b in zip(lq, lk)]).to(dev)
    assert out[~none].isnan().all() and lse[~none].isnan().all()
    assert not out[none].any() and (lse[none] == -math.inf).all()


@pytest.mark.parametrize("dtype,dim,H,hk,lq,lk", [
    # in the sequences' order without gaps: 128 rows to a tile, 64, and 64 with the keys in pieces
    (torch.bfloat16, 128, 16, 2, [512] * 8, [4096] * 8), (torch.float16, 128, 16, 2, [512] * 5, [4096, 4000, 4096, 3900, 512]),
    (torch.bfloat16, 128, 12, 4, [700, 0, 77, 513, 64, 1, 300], [700, 0, 77, 513, 64, 1, 300]),
    (torch.float16, 64, 8, 2, [64, 3, 0, 200] * 2, [3000, 700, 50, 5000] * 2),
    # by their work
    (torch.bfloat16, 128, 16, 2, [512] * 8, [600] * 8), (torch.bfloat16, 128, 12, 4, [512] * 10, [512] * 10),
    (torch.float16, 64, 32, 16, [200, 0, 333, 90, 512, 1, 400, 256] * 2, [300, 10, 400, 90, 700, 1500, 512, 300] * 2),
    (torch.bfloat16, 128, 12, 4, [700, 33, 2048, 1, 900] * 2, [700, 33, 2048, 1, 900] * 2),
    # in the sequences' order with gaps: more than 64 of them
    (torch.bfloat16, 64, 16, 4, [(30, 0, 130, 64, 1)[i % 5] for i in range(90)], [(30, 5, 200, 64, 70)[i % 5] for i in range(90)])])
def test_prompt_every_row_of_packed_sequences(dev, dtype, dim, H, hk, lq, lk):
    """Every row of batches whose tiles are taken in each of the orders, within the bound of the kernels' own roundings: a tile
    left out or given another sequence's keys would show in all its rows."""
    q, k, v = _inputs(dev, 43, dtype, dim, H, hk, lq, lk, pad=3)
    cu = lambda x: torch.tensor(_cu(x), dtype=torch.int32, device=dev)  # noqa: E731
    out = prompt_attention(q, k, v, cu(lq), dim ** -0.5, cu_seqlens_k=cu(lk))
    assert not out[sum(lq):].any()
    # (2^-32: weights below fp16's normal numbers; bf16 has fp32's range)
    want, bound = _all_rows(q, k, v, lq, lk, dim ** -0.5, lift=2.0 ** -32 if dtype == torch.float16 else 0.0)
    R.within(out, want.cpu(), bound.cpu(), "out")
