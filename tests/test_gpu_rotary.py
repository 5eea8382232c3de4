"""Rotary positions on several axes on the GPU against the plain 64-bit form (caches_ref.py)."""
from __future__ import annotations

import pytest
import torch

import caches_ref as C
import paged_ref as R
from aetherkv.cache import rope_inv_freq
from aetherkv.rotary import AxisRotary, axis_sections, rotate_axes

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _axis(R_, axes):
    return axis_sections([R_ // axes + (i < R_ % axes) for i in range(axes)], interleaved=axes > 2)


def _check(q, k, pos, rotary, axis, inverse=False, **kw):
    before = [None if x is None else x.cpu().clone() for x in (q, k)]
    out = rotate_axes(q, k, pos, rotary, inverse=inverse, **kw)
    for x, y in zip(before, out):
        if x is None:
            assert y is None
            continue
        N = x[..., 0, 0].numel()
        want, bound = C.rotate_ref(x.reshape(N, x.size(-2), x.size(-1)), pos.cpu().reshape(pos.size(0), N), rotary.inv_freq.cpu(), axis, rotary.first, rotary.pairs == "halves", inverse)
        R.within(y.cpu().reshape(want.shape), want, bound, "rotated")
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dim,R_,first", [(128, 64, None), (128, 32, None), (64, 32, 0), (64, 24, 0), (80, 40, None), (80, 20, 8), (72, 18, 2), (256, 16, 64), (6, 2, 0), (2, 1, None), (1024, 512, 0)])
def test_dims(dev, dtype, pairs, dim, R_, first):
    if pairs == "halves" and R_ % 2:
        R_, dim = 2, 4
    axis = _axis(R_, 3)
    rotary = AxisRotary(rope_inv_freq(2 * R_, 10000.0, dev), axis, dim, pairs=pairs, first=first)
    q = torch.randn(37, 3, dim, device=dev, generator=_gen(dev, dim)).to(dtype)
    k = torch.randn(37, 2, dim, device=dev, generator=_gen(dev, R_)).to(dtype)
    pos = torch.randint(-50, 5000, (3, 37), device=dev, generator=_gen(dev, 1))
    _check(q, k, pos, rotary, axis)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 1000, 1023, 1025, 4097])
@pytest.mark.parametrize("H,hk", [(1, 0), (12, 4), (5, 5), (64, 8), (130, 1)])
def test_tokens_and_heads(dev, n, H, hk):
    if n > 100 and H > 12:
        n = 100 + n % 100
    axis = _axis(32, 2)
    rotary = AxisRotary(rope_inv_freq(64, 10000.0, dev), axis, 128, pairs="halves" if n % 2 else "adjacent")
    q = torch.randn(n, H, 128, device=dev, generator=_gen(dev, n)).bfloat16()
    k = torch.randn(n, hk, 128, device=dev, generator=_gen(dev, H)).bfloat16() if hk else None
    pos = torch.randint(0, 262144, (2, n), device=dev, generator=_gen(dev, 1), dtype=torch.int32)
    _check(q, k, pos, rotary, axis)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_far_positions(dev, dtype):
    """Angles far beyond fp32's: the largest positions of either type's use."""
    axis = _axis(64, 3)
    rotary = AxisRotary(rope_inv_freq(128, 1e6, dev), axis, 128)
    far = 2 ** 31 - 1 if dtype is torch.int32 else 2 ** 40 + 12345
    pos = torch.tensor([[0, far, -far, 1000003], [1, far - 1, 17, 999], [2, 3, far // 3, 262143]], dtype=dtype, device=dev)
    q = torch.randn(4, 2, 128, device=dev, generator=_gen(dev, 0))
    # (a turn's remainder after 2^40: 2 pi to 106 bits, the product to 53, so that at most 2^40 2^-53 is lost)
    _check(q, None, pos, rotary, axis)


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_turns_in_fp32_are_off_by_their_roundings_alone(dev, pairs):
    """Cosine and sine are 64-bit sums rounded to fp32 once, off by 2^-25 at most (they are below 1), but for terms of up to 2^-8.6 that
    fp32 gives: their square of the angle, three steps of the series, its last product and the series' end are off by 2^-24 of them
    each, 2^-30 in all.  Of a pair's two products one is rounded, by 2^-24 of itself, and the sum by 2^-24:
    |y - ref| <= 2^-24 |y| + (|x1| + |x2|) (2^-25 + 2^-30 + 2^-24), and what the 64-bit angle leaves out is below 2^-10 of that.
    An angle rounded to fp32 is off by up to 2^-23."""
    axis = _axis(64, 2)
    rotary = AxisRotary(rope_inv_freq(128, 10000.0, dev), axis, 128, pairs=pairs)
    pos = torch.randint(-300000, 300000, (2, 3000), device=dev, generator=_gen(dev, 1))
    q = torch.randn(3000, 2, 128, device=dev, generator=_gen(dev, 0))
    q[1::3, :, ::2] = 0.0  # one of a pair alone
    q[2::3, :, :64] = 0.0
    for inverse in (False, True):
        out = rotate_axes(q, None, pos, rotary, inverse=inverse)[0]
        want, _ = C.rotate_ref(q.cpu(), pos.cpu(), rotary.inv_freq.cpu(), axis, 0, pairs == "halves", inverse)
        x = q.cpu().double().abs()
        both = x[..., ::2] + x[..., 1::2] if pairs == "adjacent" else x[..., :64] + x[..., 64:]
        both = both.repeat_interleave(2, -1) if pairs == "adjacent" else torch.cat([both, both], -1)
        R.within(out, want, (2.0 ** -24 * want.abs() + (1.5 * 2.0 ** -24 + 2.0 ** -30) * both) * (1 + 2.0 ** -10) + 2.0 ** -149, "turned")


def test_in_place_views_and_strides(dev):
    axis = _axis(32, 3)
    for pairs in ("adjacent", "halves"):
        rotary = AxisRotary(rope_inv_freq(64, 10000.0, dev), axis, 128, pairs=pairs)
        pos = torch.randint(0, 3000, (3, 50), device=dev, generator=_gen(dev, 1))
        qkv = torch.randn(50, 8, 128, device=dev, generator=_gen(dev, 0)).bfloat16()
        v = qkv[:, 6:].clone()
        fresh = rotate_axes(qkv[:, :4], qkv[:, 4:6], pos, rotary)
        q, k = _check(qkv[:, :4], qkv[:, 4:6], pos, rotary, axis, out_q=qkv[:, :4], out_k=qkv[:, 4:6])
        assert q.data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, :4], fresh[0]) and torch.equal(qkv[:, 4:6], fresh[1]) and torch.equal(qkv[:, 6:], v)
        # back again: each pass rounds once
        back = rotate_axes(q, k, pos, rotary, inverse=True)
        assert (back[0].float() - rotate_axes(fresh[0], None, pos, rotary, inverse=True)[0].float()).abs().max() == 0
        # one token of every sequence out of a longer buffer, [B, T, H, D] with expanded positions, rows two elements apart from 16 bytes
        x = torch.randn(5, 10, 3, 130, device=dev, generator=_gen(dev, 2)).bfloat16()[..., 2:]
        _check(x, None, pos[:, :10][:, None].expand(3, 5, 10), rotary, axis)
        _check(x[:, 3:4], None, pos[:, :5][:, :, None], rotary, axis)
        _check(x[:, ::2], None, pos.view(3, 5, 10)[:, :, ::2], rotary, axis)
        _check(x.transpose(0, 1), None, pos.view(3, 10, 5), rotary, axis)
        out = torch.full((50, 6, 128), 7.0, dtype=torch.bfloat16, device=dev)
        _check(qkv[:, :3], None, pos, rotary, axis, out_q=out[:, ::2])
        assert (out[:, 1::2] == 7).all()


def test_odd_strides_and_leading_dims_of_one(dev):
    """Rows an odd number of elements apart are copied, whichever leading dim they follow; a stride that no second row needs is not
    looked at."""
    axis = _axis(16, 2)
    for dtype in DTYPES:
        rotary = AxisRotary(rope_inv_freq(32, 10000.0, dev), axis, 32)
        base = torch.randn(4000, device=dev, generator=_gen(dev, 0)).to(dtype)
        pos = torch.randint(0, 3000, (2, 12), device=dev, generator=_gen(dev, 1))
        for shape, st, p in (((1, 5, 3, 32), (0, 97, 32, 1), pos[:, None, :5]), ((5, 1, 3, 32), (97, 7, 32, 1), pos[:, :5, None]), ((1, 1, 3, 32), (3, 5, 32, 1), pos[:, :1, None]),
                             ((5, 1, 32), (96, 1, 1), pos[:, :5]), ((5, 3, 32), (99, 33, 1), pos[:, :5]), ((2, 6, 3, 32), (582, 97, 32, 1), pos.view(2, 2, 6)), ((2, 6, 3, 32), (584, 96, 32, 1), pos.view(2, 2, 6)),
                             ((1, 1, 2, 3, 32), (0, 0, 96, 32, 1), pos[:, None, None, :2])):
            _check(base[2:].as_strided(shape, st, 2), None, p, rotary, axis)


def test_inverse_is_the_gradient(dev):
    """Turning back is the transpose: <rotate(x), y> = <x, inverse(y)>, and differences agree with it."""
    axis = _axis(16, 2)
    rotary = AxisRotary(rope_inv_freq(32, 100.0, dev), axis, 48)
    pos = torch.randint(0, 100, (2, 9), device=dev, generator=_gen(dev, 0))
    x, y = (torch.randn(9, 2, 48, device=dev, generator=_gen(dev, i)) for i in (1, 2))
    a = (rotate_axes(x, None, pos, rotary)[0].double() * y.double()).sum()
    b = (x.double() * rotate_axes(y, None, pos, rotary, inverse=True)[0].double()).sum()
    # each output is off by 2^-24 of itself and 2^-21 of a pair's sum (caches_ref): summed over both products
    assert abs(a - b) <= 2.0 ** -20 * 2 * ((x.abs() * y.abs()).sum().double() + (x.abs().sum(-1) * 2 * y.abs().amax(-1)).sum().double())


def test_not_numbers_stay_in_their_pairs(dev):
    axis = _axis(64, 1)
    for pairs in ("adjacent", "halves"):
        rotary = AxisRotary(rope_inv_freq(128, 10000.0, dev), axis, 128, pairs=pairs)
        pos = torch.arange(3, 8, device=dev)[None]
        q = torch.randn(5, 2, 128, device=dev, generator=_gen(dev, 0)).half()
        clean = rotate_axes(q, None, pos, rotary)[0]
        q[2, 1, 10] = float("nan")
        out = rotate_axes(q, None, pos, rotary)[0]
        pair = [10, 11] if pairs == "adjacent" else [10, 74]
        assert out[2, 1, pair].isnan().all()
        out[2, 1, pair] = clean[2, 1, pair]
        assert torch.equal(out, clean)


def test_graph_and_stream(dev):
    axis = _axis(64, 3)
    rotary = AxisRotary(rope_inv_freq(128, 10000.0, dev), axis, 128)
    pos = torch.randint(0, 3000, (3, 64), device=dev, generator=_gen(dev, 1), dtype=torch.int32)
    q = torch.randn(64, 4, 128, device=dev, generator=_gen(dev, 0)).bfloat16()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        rotate_axes(q, None, pos, rotary)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out, _ = rotate_axes(q, None, pos, rotary)
    torch.cuda.synchronize()
    for i in range(3):
        pos.add_(1000 * i)
        q.mul_(1 + i)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rotate_axes(q, None, pos, rotary)[0])


def test_offsets_past_32_bits(dev):
    """2^31 elements and more: the last tokens turn as they do by themselves."""
    n, H, D = 1_100_000, 16, 128
    x = torch.zeros(n, H, D, dtype=torch.bfloat16, device=dev)
    x[-300:] = torch.randn(300, H, D, device=dev, generator=_gen(dev, 0))
    pos = torch.arange(n, dtype=torch.int32, device=dev)[None]
    rotary = AxisRotary(rope_inv_freq(D, 10000.0, dev), [0] * 64, D)
    want, _ = rotate_axes(x[-300:].clone(), None, pos[:, -300:].clone(), rotary)
    out, _ = rotate_axes(x, None, pos, rotary, out_q=x)
    assert out is x and torch.equal(x[-300:], want) and not x[:-300].any()


def test_empty(dev):
    rotary = AxisRotary(rope_inv_freq(128, 10000.0, dev), [0] * 64, 128)
    q, k = torch.empty(0, 4, 128, device=dev), torch.empty(0, 2, 128, device=dev)
    out = rotate_axes(q, k, torch.empty(1, 0, dtype=torch.int32, device=dev), rotary)
    assert out[0].shape == q.shape and out[1].shape == k.shape


def test_refusals(dev):
    freq = rope_inv_freq(64, 10000.0, dev)
    for kw in (dict(axis=[0] * 31), dict(axis=[-1] * 32), dict(dim=62), dict(dim=63), dict(first=66), dict(first=1), dict(pairs="both")):
        with pytest.raises(ValueError):
            AxisRotary(freq, kw.pop("axis", [0] * 32), kw.pop("dim", 128), **kw)
    with pytest.raises(RuntimeError):
        AxisRotary(freq.double(), [0] * 32, 128)
    rotary = AxisRotary(freq, _axis(32, 3), 128)
    q, k, pos = torch.zeros(5, 4, 128, device=dev), torch.zeros(5, 2, 128, device=dev), torch.zeros(3, 5, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    for args, kw in (((q[..., :64], k, pos), {}), ((q, k[:4], pos), {}), ((q, k.half(), pos), {}), ((q.double(), k.double(), pos), {}), ((q, k, pos[:2]), {}), ((q, k, pos[:, :4]), {}),
                     ((q, k, pos.float()), {}), ((q, k, pos.cpu()), {}), ((q, None, pos), dict(out_k=out)), ((q, k, pos), dict(out_q=out[:4])), ((q, k, pos), dict(out_q=out.half())),
                     ((q, k, pos), dict(out_q=out[:1].expand(5, 4, 128))), ((q, k, pos), dict(out_q=torch.empty(5, 4, 256, device=dev)[..., ::2])), ((q[0], None, pos), {})):
        with pytest.raises(RuntimeError):
            rotate_axes(*args, rotary, **kw)
