"""Attention over an encoder's states on the GPU against the plain 64-bit form (caches_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

import caches_ref as C
import paged_ref as R
from aetherkv.cross import cross_attention, cross_workspace

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _t(x, dev):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


def _check(dev, dtype, dim, H, hk, lq, lk, states=None, sink=False, pad=0, seed=0, gain=1.0, scale=None, offsets=True):
    nq, nk = sum(lq) + pad, sum(lk) + pad
    q = (torch.randn(nq, H, dim, device=dev, generator=_gen(dev, seed)) * gain).to(dtype)
    kv = torch.randn(nk, 2, hk, dim, device=dev, generator=_gen(dev, seed + 1)).to(dtype)
    k, v = kv[:, 0], kv[:, 1]
    cq, ck = _cu(lq), _cu(lk)
    sk = torch.randn(H, device=dev, generator=_gen(dev, seed + 2)) if sink else None
    scale = dim ** -0.5 if scale is None else scale
    out, lse = cross_attention(q, k, v, _t(ck, dev), scale, cu_seqlens=_t(cq, dev) if offsets else None, states=_t(states, dev), sink=sk, return_lse=True)
    want, bound, wl, lb = C.cross_attention_ref(q.cpu(), k.cpu(), v.cpu(), cq, ck, states, scale, None if sk is None else sk.cpu())
    R.within(out, want, bound, "out")
    got = lse.double().cpu()
    none = wl == -math.inf
    assert torch.equal(got == -math.inf, none)
    R.within(got[~none], wl[~none], lb[~none], "lse")
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700])
def test_one_query_lengths(dev, dtype, dim, n):
    _check(dev, dtype, dim, 6, 2, [1], [n], seed=n, offsets=n % 2 == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk", [(40, 1), (64, 63), (65, 64), (127, 65), (128, 129), (200, 300), (33, 1000), (1000, 40)])
def test_many_queries(dev, dtype, dim, lq, lk):
    _check(dev, dtype, dim, 4, 2, [lq], [lk], seed=lq + lk, sink=lq % 2 == 1)


@pytest.mark.parametrize("H,hk", [(1, 1), (3, 3), (12, 4), (12, 1), (16, 2), (10, 2), (32, 1), (33, 1), (48, 1), (64, 1), (40, 2)])
@pytest.mark.parametrize("lq", [[1, 1, 1], [3, 1, 2], [20, 30, 5]])
def test_head_layouts(dev, H, hk, lq):
    _check(dev, torch.bfloat16, 128, H, hk, lq, [70, 333, 129], sink=True, seed=H)


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("lq,lk", [([0], [5]), ([0, 5, 0, 0, 30, 1], [7, 0, 3, 0, 260, 1]), ([1] * 70, [(37 * i) % 300 for i in range(70)]), ([3, 1, 200], [500, 0, 65])])
def test_packed(dev, lq, lk, pad):
    out, lse = _check(dev, torch.bfloat16, 64, 4, 2, lq, lk, pad=pad, seed=len(lq)) if sum(lq) + pad else (None, None)
    if pad:
        assert not out[-pad:].any() and (lse[-pad:] == -math.inf).all()


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("states", [[0] * 9, [0, 0, 0, 1, 1, 2, 2, 2, 2], [2, 0, 1, 1, 0, 2, 2, 0, 0], [1, -1, -1, 3, 0, 7, 2, 2, 2 ** 31 - 1]])
def test_shared_states(dev, states, offsets):
    _check(dev, torch.float16, 64, 8, 8, [1] * 9, [300, 41, 0], states=states, seed=1, offsets=offsets, sink=True)
    _check(dev, torch.bfloat16, 128, 6, 2, [5, 0, 7, 1, 1, 30, 2, 0, 9], [300, 41, 0], states=states, seed=2)
    _check(dev, torch.bfloat16, 64, 6, 2, [50, 0, 70, 1, 1, 130, 20, 0, 9], [300, 41, 0], states=states, seed=3)


@pytest.mark.parametrize("B,lq", [(64, 1), (65, 1), (200, 1), (256, 1), (257, 1), (600, 1), (300, 3)])
@pytest.mark.parametrize("shared", [False, True])
def test_many_sequences(dev, B, lq, shared):
    E = 5 if shared else B
    states = [b * E // B for b in range(B)] if shared else None
    _check(dev, torch.bfloat16, 64, 2, 1, [lq] * B, [(53 * i) % 180 for i in range(E)], states=states, seed=B, offsets=lq > 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq", [1, 2, 100])
@pytest.mark.parametrize("gain,scale", [(1.0, 0.0), (1.0, -0.3), (30.0, None), (1.0, 1e-30), (300.0, 1.0), (100.0, 1000.0)])
def test_scales(dev, dtype, lq, gain, scale):
    _check(dev, dtype, 64, 4, 2, [lq], [333], seed=3, gain=gain, scale=scale)


def test_the_next_sequences_states_and_the_rows_behind_do_not_reach(dev):
    """Keys and values outside a sequence's states are NaN and infinities: nothing of them is read."""
    for lq in (1, 3, 90):
        q = torch.randn(2 * lq, 4, 128, device=dev, generator=_gen(dev, 0)).bfloat16()
        k = torch.randn(400, 2, 128, device=dev, generator=_gen(dev, 1)).bfloat16()
        v = torch.randn(400, 2, 128, device=dev, generator=_gen(dev, 2)).bfloat16()
        clean = cross_attention(q, k, v, _t([30, 67, 200], dev), 0.1, cu_seqlens=_t([0, lq, 2 * lq], dev))
        k[:30], k[200:], v[:30], v[200:] = NAN, math.inf, math.inf, NAN
        assert torch.equal(clean, cross_attention(q, k, v, _t([30, 67, 200], dev), 0.1, cu_seqlens=_t([0, lq, 2 * lq], dev)))
        # what a sequence sees, it answers for, and the other does not
        k[40, 0] = NAN
        out = cross_attention(q, k, v, _t([30, 67, 200], dev), 0.1, cu_seqlens=_t([0, lq, 2 * lq], dev))
        assert out[:lq, :2].isnan().all() and torch.equal(out[:, 2:], clean[:, 2:]) and torch.equal(out[lq:], clean[lq:])


@pytest.mark.parametrize("lq", [1, 80])
def test_sinks_infinities_and_nan_scale(dev, lq):
    q = torch.randn(lq, 4, 64, device=dev, generator=_gen(dev, 0)).half()
    k, v = (torch.randn(150, 2, 64, device=dev, generator=_gen(dev, i)).half() for i in (1, 2))
    cu, cq = _t([0, 150], dev), _t([0, lq], dev)
    plain, lse = cross_attention(q, k, v, cu, 0.125, cu_seqlens=cq, return_lse=True)
    low, lse2 = cross_attention(q, k, v, cu, 0.125, cu_seqlens=cq, sink=torch.full((4,), -math.inf, device=dev), return_lse=True)
    assert torch.equal(plain, low) and torch.equal(lse, lse2)
    lowest, _ = cross_attention(q, k, v, cu, 0.125, cu_seqlens=cq, sink=torch.full((4,), torch.finfo(torch.float32).min, device=dev), return_lse=True)
    assert torch.equal(plain, lowest)
    assert cross_attention(q, k, v, cu, NAN, cu_seqlens=cq).isnan().all()
    assert not cross_attention(q, k, v, _t([0, 0], dev), NAN, cu_seqlens=cq).any()  # nothing seen
    k[7, 0] = -math.inf  # logits of -inf and inf by the queries' signs, or NaN
    out = cross_attention(q, k, v, cu, 0.125, cu_seqlens=cq)
    assert out[:, :2].isnan().all() and torch.equal(out[:, 2:], plain[:, 2:])


@pytest.mark.parametrize("H,hk,dim,lq", [(4, 2, 64, 1), (4, 2, 64, 70), (6, 3, 128, 1), (6, 1, 128, 40)])
def test_views_are_read_in_place(dev, H, hk, dim, lq):
    for pick in (lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: torch.stack([t, t], 1)[:, 1], lambda t: t[:, :, :].clone().as_strided(t.shape, t.contiguous().stride())):
        q = pick(torch.randn(lq, H, dim, device=dev, generator=_gen(dev, 0)).bfloat16())
        k, v = (pick(torch.randn(97, hk, dim, device=dev, generator=_gen(dev, i)).bfloat16()) for i in (1, 2))
        want, bound, _, _ = C.cross_attention_ref(q.cpu(), k.cpu(), v.cpu(), [0, lq], [0, 97], None, 0.1)
        R.within(cross_attention(q, k, v, _t([0, 97], dev), 0.1, cu_seqlens=_t([0, lq], dev)), want, bound, "out")
    base = torch.randn(97 * hk * dim + 4, device=dev, generator=_gen(dev, 5)).bfloat16()
    odd = base[4:].view(97, hk, dim)  # rows off 16 bytes are copied
    q = torch.randn(lq, H, dim, device=dev, generator=_gen(dev, 0)).bfloat16()
    assert torch.equal(cross_attention(q, odd, odd, _t([0, 97], dev), 0.1, cu_seqlens=_t([0, lq], dev)),
                       cross_attention(q, odd.clone(), odd.clone(), _t([0, 97], dev), 0.1, cu_seqlens=_t([0, lq], dev)))


def test_out_keeps_rows_in_no_sequence_and_workspaces_are_taken(dev):
    for lq in (1, 60):
        q = torch.randn(2 * lq + 4, 4, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
        k, v = (torch.randn(500, 2, 64, device=dev, generator=_gen(dev, i)).bfloat16() for i in (1, 2))
        cq, ck = _t([3, 3 + lq, 3 + 2 * lq], dev), _t([0, 200, 500], dev)
        want = cross_attention(q, k, v, ck, 0.1, cu_seqlens=cq)
        assert not want[:3].any() and not want[-1:].any()
        out = torch.full_like(q, 7.0)
        ws = cross_workspace(2, 2, q.size(0), 500, 4, 2, 64, dev).fill_(255)
        assert cross_attention(q, k, v, ck, 0.1, cu_seqlens=cq, out=out, workspace=ws) is out
        assert (out[:3] == 7).all() and (out[-1:] == 7).all() and torch.equal(out[3:-1], want[3:-1])


def test_offsets_that_are_no_prefix_sums_stay_in_bounds(dev):
    """Bad offsets give some result, within the tensors."""
    for N, M, cq, ck in ((64, 300, [0, 64, -5, 64, 0, 1 << 30, 64], [50, 10, 1 << 30, -7, 300, 0, 300]), (6, 300, [5, 0, 6, 0, 6, 3, 6], [300] * 7)):
        for H in (4, 2):
            q = torch.randn(N, H, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
            k, v = (torch.randn(M, 2, 64, device=dev, generator=_gen(dev, i)).bfloat16() for i in (1, 2))
            out = cross_attention(q, k, v, _t(ck, dev), 0.1, cu_seqlens=_t(cq, dev))
            torch.cuda.synchronize()
            assert out.shape == q.shape


@pytest.mark.parametrize("per", [1, 30])
def test_bad_offsets_write_nothing_beside_the_output(dev, per):
    """Offsets that are no prefix sums, states out of range: what lies before and behind `out` and the workspace, whose last byte the
    call may use, is as it was."""
    for cq, ck in (([0, 2, -5, 2, 0, 1 << 30, 2], [50, 10, 1 << 30, -7, 300, 0, 300]), ([5, 0, 6, 0, 6, 3, 6], [300] * 7), ([0, 1, 2, 3, 4, 5, 6], [0, 50, 100, 150, 200, 250, 300])):
        B, H, N, M = 6, 4, 6 * per, 300
        q = torch.randn(N, H, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
        k, v = (torch.randn(M, 2, 64, device=dev, generator=_gen(dev, i)).bfloat16() for i in (1, 2))
        rows = torch.full((N + 512, H, 64), 7.0, dtype=torch.bfloat16, device=dev)
        out = rows[256:256 + N]
        size = cross_workspace(B, 6, N, M, H, 2, 64, dev).numel()
        room = torch.full((size + (2 << 20),), 0xA5, dtype=torch.uint8, device=dev)
        cross_attention(q, k, v, _t(ck, dev), 0.1, cu_seqlens=_t([per * c if 0 < c < 100 else c for c in cq], dev), out=out, states=_t([0, 3, -1, 6, 2 ** 31 - 1, 5], dev),
                        workspace=room[1 << 20:(1 << 20) + size])
        assert (rows[:256] == 7).all() and (rows[256 + N:] == 7).all()
        assert (room[:1 << 20] == 0xA5).all() and (room[(1 << 20) + size:] == 0xA5).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq", [1, 40])
def test_a_sequence_alone_and_among_others(dev, dtype, lq):
    """A sequence by itself against the same one in a batch: each is within the bound, so they are within twice the bound."""
    B, lk = 12, [(61 * i) % 400 + 1 for i in range(12)]
    cq, ck = _cu([lq] * B), _cu(lk)
    q = torch.randn(B * lq, 6, 64, device=dev, generator=_gen(dev, 0)).to(dtype)
    k, v = (torch.randn(sum(lk), 3, 64, device=dev, generator=_gen(dev, i)).to(dtype) for i in (1, 2))
    out, lse = cross_attention(q, k, v, _t(ck, dev), 0.125, cu_seqlens=_t(cq, dev), return_lse=True)
    _, bound, _, lb = C.cross_attention_ref(q.cpu(), k.cpu(), v.cpu(), cq, ck, None, 0.125)
    for b in range(B):
        rows, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        one, l1 = cross_attention(q[rows], k[keys], v[keys], _t([0, lk[b]], dev), 0.125, cu_seqlens=_t([0, lq], dev), return_lse=True)
        R.within(one, out[rows].double().cpu(), 2 * bound[rows], "alone")
        R.within(l1, lse[rows].double().cpu(), 2 * lb[rows], "alone, lse")


def test_a_rows_bits_do_not_depend_on_its_tiles_rows(dev):
    """A row whose logits rise by the margin up to a rounding (their rounded difference passes it, the exact one, rounded, does not),
    beside a row that rises far beyond it and beside one that does not: the same bits."""
    for scale, t0, a, c, e in (("0x1.939af8p+0", 0.55078125, 155, 215, 2), ("0x1.87e506p+0", 1.3828125, 166, 247, 2), ("0x1.92c440p+0", 0.828125, 181, 197, 2), ("0x1.2356bep-1", 1.8515625, 190, 250, 3)):
        q = torch.zeros(60, 1, 64, device=dev)
        k = torch.zeros(64, 1, 64, device=dev)
        v = torch.randn(64, 1, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
        q[:, 0, 2] = 1.0
        k[:, 0, 2] = -torch.rand(64, device=dev, generator=_gen(dev, 1)) * 3 - 0.1  # the other logits
        q[5, 0, 0], q[5, 0, 1] = 1.0, a / 128
        k[3, 0, 0], k[3, 0, 2] = t0, 0.0                       # the first block's largest
        k[40, 0, 1], k[40, 0, 2] = c / 128 * 2.0 ** (e - 1), 0.0  # the second's: a c 2^(e - 15)
        outs = []
        for far in (0.0, 50.0):
            q[6, 0, 3], k[50, 0, 3] = far, 1.0
            outs.append(cross_attention(q.bfloat16(), k.bfloat16(), v, _t([0, 64], dev), float.fromhex(scale), cu_seqlens=_t([0, 60], dev), return_lse=True))
        assert not torch.equal(outs[0][0][6], outs[1][0][6])
        for x, y in zip(*outs):
            assert torch.equal(x[5], y[5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,hk,dim,lq", [(4, 2, 64, 1), (12, 4, 128, 1), (12, 1, 64, 2), (8, 8, 128, 3)])
def test_few_rows_weights_keep_their_bits(dev, dtype, H, hk, dim, lq):
    """Values that nearly cancel: what is left is the difference of the weights.  With few rows a weight is its 16-bit rounding and the
    rounded rest, off by the square of the half step u (fp16, held 2^7 higher than the largest, by 2^-32 of it at least):
    |out - ref| <= u |ref| + (u^2 + 2 delta + (n + 16) 2^-24) sum_j p_j |v_j| + n 2^-32 max |v|."""
    for n in (2, 6, 40, 300):
        q = (0.2 * torch.randn(3 * lq, H, dim, device=dev, generator=_gen(dev, n))).to(dtype)
        k = (0.2 * torch.randn(3 * n, hk, dim, device=dev, generator=_gen(dev, n + 1))).to(dtype)
        v = torch.randn(3 * n // 2, hk, dim, device=dev, generator=_gen(dev, n + 2)).to(dtype)
        v = torch.stack([v, -v], 1).flatten(0, 1)
        cq, ck = _cu([lq] * 3), _cu([n] * 3)
        out = cross_attention(q, k, v, _t(ck, dev), dim ** -0.5, cu_seqlens=_t(cq, dev))
        want, bound, _, _ = C.cross_attention_ref(q.cpu(), k.cpu(), v.cpu(), cq, ck, None, dim ** -0.5)
        plain, weighted = torch.zeros_like(bound), torch.zeros_like(bound)
        u, d = R.U[dtype], dim ** -0.5
        for b in range(3):
            for h in range(H):
                rows, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
                qq, kk, vv = q[rows, h].cpu().double(), k[keys, h // (H // hk)].cpu().double(), v[keys, h // (H // hk)].cpu().double()
                logit = qq @ kk.T * d
                delta = (d * (qq.abs() @ kk.abs().T) * (dim + 8) * 2.0 ** -24 + logit.abs() * 2.0 ** -21).amax(1, keepdim=True)
                weighted[rows, h] = (u * u + 2 * delta + (n + 16) * 2.0 ** -24) * (torch.softmax(logit, 1) @ vv.abs()) + n * 2.0 ** -32 * vv.abs().max()
                plain[rows, h] = u * want[rows, h].abs()
        R.within(out, want, plain + weighted + R.TINY[dtype], "out")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,lq", [(64, 1), (64, 12), (128, 3), (128, 70)])
def test_infinite_values_that_are_seen(dev, dtype, dim, lq):
    """An infinite value gives infinities in its dim, a NaN gives NaN, and other dims do not see them."""
    q = (0.3 * torch.randn(lq, 4, dim, device=dev, generator=_gen(dev, 0))).to(dtype)
    k, v = (torch.randn(200, 2, dim, device=dev, generator=_gen(dev, i)).to(dtype) for i in (1, 2))
    args = k, _t([0, 200], dev), dim ** -0.5
    clean = cross_attention(q, args[0], v, *args[1:], cu_seqlens=_t([0, lq], dev))
    v[150, 0, 7], v[30, 1, 9], v[199, 1, 11] = math.inf, -math.inf, NAN
    out = cross_attention(q, args[0], v, *args[1:], cu_seqlens=_t([0, lq], dev))
    assert (out[:, :2, 7] == math.inf).all() and (out[:, 2:, 9] == -math.inf).all() and out[:, 2:, 11].isnan().all()
    out[:, :2, 7], out[:, 2:, 9], out[:, 2:, 11] = clean[:, :2, 7], clean[:, 2:, 9], clean[:, 2:, 11]
    assert torch.equal(out, clean)


def test_long_states_split_and_merged(dev):
    for lq, H, hk, n in ((1, 4, 1, 9001), (2, 2, 2, 5000), (50, 4, 4, 9001)):
        _check(dev, torch.bfloat16, 64, H, hk, [lq], [n], sink=True, seed=n)
    _check(dev, torch.float16, 128, 3, 1, [1, 1, 1], [6000, 3, 900], seed=9, offsets=False)


def test_results_do_not_depend_on_the_others(dev):
    """The same sequence alone and in a batch: within twice the bound (the parts of a line may lie differently); twice the same
    call: bit for bit."""
    q = torch.randn(40, 6, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
    k, v = (torch.randn(40 * 111, 3, 64, device=dev, generator=_gen(dev, i)).bfloat16() for i in (1, 2))
    ck = _t([111 * i for i in range(41)], dev)
    a, b = cross_attention(q, k, v, ck, 0.1), cross_attention(q, k, v, ck, 0.1)
    assert torch.equal(a, b)
    want, bound, _, _ = C.cross_attention_ref(q.cpu(), k.cpu(), v.cpu(), list(range(41)), [111 * i for i in range(41)], None, 0.1)
    R.within(a, want, bound, "out")


@pytest.mark.parametrize("lq", [1, 70])
def test_graphs_and_streams(dev, lq):
    """Two graphs captured on one stream, replayed on two with new lengths: each has a workspace of its own."""
    data, graphs, outs = [], [], []
    side = torch.cuda.Stream()
    for i in range(2):
        q = torch.randn(3 * lq, 4, 64, device=dev, generator=_gen(dev, i)).bfloat16()
        k, v = (torch.randn(3000, 2, 64, device=dev, generator=_gen(dev, 10 * i + j)).bfloat16() for j in (1, 2))
        data.append((q, k, v, _t([0, 1000, 1700, 3000], dev), _t([0, lq, 2 * lq, 3 * lq], dev)))
    call = lambda d: cross_attention(*d[:3], d[3], 0.1, cu_seqlens=d[4])  # noqa: E731
    with torch.cuda.stream(side):
        for d in data:
            call(d)
        side.synchronize()
        for d in data:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(call(d))
            graphs.append(g)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for ends in ([0, 1000, 1700, 3000], [0, 0, 2999, 3000], [5, 300, 300, 900]):
        for d in data:
            d[3].copy_(_t(ends, dev))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for d, out in zip(data, outs):
            assert torch.equal(out, call(d))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("shared", [False, True])
def test_many_rows_in_many_sequences(dev, dtype, dim, shared):
    """Long and short answers of more sequences than one launch takes."""
    B = 300
    lq = [(29 * i) % 90 if i % 7 else 0 for i in range(B)]
    states = [b // 9 if b % 50 else -1 for b in range(B)] if shared else None
    _check(dev, dtype, dim, 2, 1, lq, [(67 * i) % 230 for i in range(34 if shared else B)], states=states, seed=4, sink=True, pad=2)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("H,hk", [(8, 8), (12, 4), (12, 6), (9, 3), (32, 2)])
@pytest.mark.parametrize("kind", ["steps", "ragged", "runs"])
def test_heads_read_together(dev, dtype, dim, H, hk, kind):
    """Enough sequences for one workgroup to take two or four KV heads at a time: single queries, a few long answers among short ones
    (several tiles to a head), runs over the same states; states that end within every part of a unit."""
    B = 70
    lq = [1] * B if kind != "ragged" else [(0, 1, 2, 1)[b % 4] + (40 if b in (5, 44) else 0) for b in range(B)]
    states = [b // 2 for b in range(B)] if kind == "runs" else None
    lk = [(0, 1, 31, 32, 33, 63, 65, 96, 127, 128, 129, 255, 300, 700)[b % 14] for b in range(B)]
    _check(dev, dtype, dim, H, hk, lq, lk, states=states, seed=H, sink=hk % 2 == 0, offsets=kind == "ragged")


def test_a_captured_call_of_several_launches(dev):
    """More sequences than one launch takes, one workspace for all launches of a call, replayed with other states and lengths."""
    B = 300
    for per in (1, 25):
        q = torch.randn(per * B, 4, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
        k, v = (torch.randn(900, 2, 64, device=dev, generator=_gen(dev, i)).bfloat16() for i in (1, 2))
        ck, st, cq = _t([0, 500, 500, 900], dev), _t([b % 3 for b in range(B)], dev), _t([per * b for b in range(B + 1)], dev)
        call = lambda: cross_attention(q, k, v, ck, 0.1, cu_seqlens=cq, states=st, return_lse=True)  # noqa: E731
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = call()
        for ends, pick in (([0, 500, 500, 900], lambda b: b % 3), ([0, 10, 900, 900], lambda b: b // 100), ([0, 0, 0, 1], lambda b: 2), ([0, 300, 600, 900], lambda b: b % 4 - 1)):
            ck.copy_(_t(ends, dev))
            st.copy_(_t([pick(b) for b in range(B)], dev))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, call()):
                assert torch.equal(a, b)


def test_offsets_past_32_bits_and_shared_strides(dev):
    """Rows of keys and values 16 MB apart (their offsets pass 2^32 elements); heads that are one and the same."""
    stride, M = 8388600, 600
    base = torch.empty(M * stride, dtype=torch.bfloat16, device=dev)
    kv = base.view(M, stride)[:, :256].view(M, 2, 2, 64)
    kv.copy_(torch.randn(M, 2, 2, 64, device=dev, generator=_gen(dev, 1)))
    for lq in (1, 60):
        q = torch.randn(lq, 4, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
        cu, cq = _t([0, M], dev), _t([0, lq], dev)
        near = kv.contiguous()
        assert torch.equal(cross_attention(q, kv[:, 0], kv[:, 1], cu, 0.1, cu_seqlens=cq), cross_attention(q, near[:, 0], near[:, 1], cu, 0.1, cu_seqlens=cq))
        k, v = (near[:, i, :1].expand(M, 2, 64) for i in range(2))
        assert torch.equal(cross_attention(q, k, v, cu, 0.1, cu_seqlens=cq), cross_attention(q, k.contiguous(), v.contiguous(), cu, 0.1, cu_seqlens=cq))
    wide = base.as_strided((3, 2, 64), (8388608, 64, 1))
    with pytest.raises(RuntimeError, match="stride"):
        cross_attention(q, wide, wide, _t([0, 3], dev), 0.1, cu_seqlens=cq)


@pytest.mark.parametrize("lq", [1, 50])
def test_one_state_out_of_a_wide_buffer(dev, lq):
    """One row of keys and values, whose token stride is more than rows may lie apart."""
    base = torch.randn(1 << 24, device=dev, generator=_gen(dev, 1)).bfloat16()
    k, v = (base.as_strided((1, 2, 64), (1 << 24, 64, 1), at) for at in (0, 128))
    q = torch.randn(lq, 4, 64, device=dev, generator=_gen(dev, 0)).bfloat16()
    out = cross_attention(q, k, v, _t([0, 1], dev), 0.1, cu_seqlens=_t([0, lq], dev))
    assert torch.equal(out, v.repeat_interleave(2, 1).expand(lq, 4, 64))  # (a weight of 1)
    v[0, 1, 5] = math.inf
    out = cross_attention(q, k, v, _t([0, 1], dev), 0.1, cu_seqlens=_t([0, lq], dev))
    assert torch.equal(out, v.repeat_interleave(2, 1).expand(lq, 4, 64))


@pytest.mark.parametrize("lq", [1, 50])
def test_rows_that_overlap(dev, lq):
    """Keys and values whose rows are one and the same, or windows over one line: an infinite value stays in its own rows' dims."""
    q = torch.randn(lq, 2, 64, device=dev, generator=_gen(dev, 0)).bfloat16() * 0.1
    for step in (0, 8):
        for n in (41, 33, 10):
            line = torch.randn(64 + 8 * 40, device=dev, generator=_gen(dev, 1)).bfloat16()
            k = (line * 0.1).as_strided((41, 1, 64), (step, 64, 1))
            line[(n - 1) * step + 60] = math.inf  # dim 60 of the last row that is seen
            v = line.as_strided((41, 1, 64), (step, 64, 1))
            cu, cq = _t([0, n], dev), _t([0, lq], dev)
            out = cross_attention(q, k, v, cu, 0.1, cu_seqlens=cq)
            assert (out[..., 60] == math.inf).all() and torch.isfinite(out[..., [i for i in range(64) if i != 60]]).all()
            assert torch.equal(out, cross_attention(q, k.contiguous(), v.contiguous(), cu, 0.1, cu_seqlens=cq))


def test_empty_calls(dev):
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    assert cross_attention(q, k, k, _t([0], dev), 0.1).shape == (0, 4, 64)
    q = torch.randn(3, 4, 64, device=dev).bfloat16()
    out, lse = cross_attention(q, k, k, _t([0], dev), 0.1, states=_t([0, 1, -1], dev), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    out = cross_attention(q, k, k, _t([0, 0], dev), 0.1, cu_seqlens=_t([0, 3], dev), sink=torch.zeros(4, device=dev))
    assert not out.any()


def test_refusals(dev):
    q, k, cu = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev), torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=dev), _t([0, 2, 5], dev)
    for args, kw in (((q, k, k, cu), {}), ((q, k, k, cu), dict(states=_t([0, 1], dev))), ((q, k, k, cu), dict(states=torch.zeros(3, device=dev))), ((q, k, k, cu.cpu()), {}),
                     ((q, k, k[:4], cu), {}), ((q.float(), k.float(), k.float(), cu), {}), ((q, k, k, cu), dict(cu_seqlens=_t([0, 1, 2, 3], dev))),
                     ((q, k, k, cu), dict(cu_seqlens=_t([0, 1, 3], dev), out=q[:2].clone())), ((q, k, k, cu), dict(cu_seqlens=_t([0, 1, 3], dev), sink=torch.zeros(3, device=dev))),
                     ((q, k, k, cu), dict(cu_seqlens=_t([0, 1, 3], dev), workspace=torch.empty(16, dtype=torch.uint8, device=dev)))):
        with pytest.raises(RuntimeError):
            cross_attention(*args, 0.1, **kw)
