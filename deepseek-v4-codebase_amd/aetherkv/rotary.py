"""Rotary positions on several axes (time, height, width of images and video; one axis: text), of q and k at once.

prompt_attention, append_tokens and cross_attention take keys and queries that carry their rotation.  attention_io's
rope_rmsnorm does the reference model's own step (one axis, bf16, its rounding points, with the norm); here every pair of
dims has an axis of its own, positions are given per axis, and the result is rounded once.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .paged import _TYPES, _one_device


def axis_sections(sections: Sequence[int], *, interleaved: bool = False) -> list:
    """The axis of every pair: sections[0] pairs of axis 0, then sections[1] of axis 1, ..; interleaved: in turn while they
    last (0, 1, 2, 0, 1, 2, ..)."""
    left = [int(n) for n in sections]
    if not left or min(left) < 0 or not sum(left):
        raise ValueError(f"sections must be counts of pairs, got {list(sections)}")
    if not interleaved:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


class AxisRotary:
    """Which dims turn, how fast and by which axis: made once for a model's layers.

    inv_freq fp32 [R] on the device (cache.rope_inv_freq, or a scaled model's own), axis: R axis numbers (axis_sections),
    dim: the head dim.  pairs "adjacent": dims first + 2 i and first + 2 i + 1; "halves": first + i and first + R + i.  first:
    dim - 2 R by default, the last dims, as the framework's other rotary parts."""

    def __init__(self, inv_freq: torch.Tensor, axis: Sequence[int], dim: int, *, pairs: str = "adjacent", first: Optional[int] = None):
        _lib.require_device("inv_freq", inv_freq)
        if pairs not in ("adjacent", "halves"):
            raise ValueError(f"pairs must be 'adjacent' or 'halves', got {pairs!r}")
        if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
            raise RuntimeError(f"inv_freq must be float32 [R], got {inv_freq.dtype} {tuple(inv_freq.shape)}")
        axis = [int(a) for a in axis]
        R, dim = inv_freq.numel(), int(dim)
        if len(axis) != R or R < 1 or min(axis) < 0:
            raise ValueError(f"axis must name an axis (0, 1, ..) for each of {R} pairs, got {len(axis)}")
        first = dim - 2 * R if first is None else int(first)
        if dim < 2 or dim > 1024 or dim % 2 or first < 0 or first % 2 or first + 2 * R > dim or (pairs == "halves" and R % 2):
            raise ValueError(f"{R} pairs ({pairs}) from dim {first} of {dim}: dims and first must be even, halves an even number of pairs")
        self.dim, self.pairs, self.first, self.count, self.axes = dim, pairs, first, R, max(axis) + 1
        self.device, self._index = inv_freq.device, inv_freq.get_device()
        self._freq = inv_freq.contiguous().clone()
        self._axis = torch.tensor(axis, dtype=torch.int32, device=inv_freq.device)
        self._args = (self._freq.data_ptr(), self._axis.data_ptr(), R, first, int(pairs == "halves"))

    inv_freq = property(lambda self: self._freq)
    axis = property(lambda self: self._axis)


def _token_stride(t: torch.Tensor) -> Optional[Tuple[int, int]]:
    """(token, head) strides of [.., heads, D], its leading dims as one, or None where they are not one stride apart."""
    shape, st = t.shape, t.stride()
    if shape[-1] > 1 and st[-1] != 1:
        return None
    token, tokens = 0, 1
    for i in range(len(shape) - 3, -1, -1):
        if shape[i] == 1:
            continue
        if tokens == 1:
            token = st[i]
        elif st[i] != token * tokens:
            return None
        tokens *= shape[i]
    return token, st[-2] if shape[-2] > 1 else 0


def _flat(t: torch.Tensor, unit: int) -> Tuple[torch.Tensor, int, int]:
    """t [.., heads, D], or a copy that the kernel can read, with its strides."""
    st = _token_stride(t)
    if st is None or st[0] % 2 or st[1] % 2 or t.data_ptr() % unit:
        t = _lib.aligned(t, 16)
        st = (t.size(-2) * t.size(-1), t.size(-1))
    return t, st[0], st[1]


def rotate_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: AxisRotary, *, inverse: bool = False,
                out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [.., H, D] and k [.., kv_heads, D] (or None) turned by their tokens' positions: (q, k) like them.

    bf16, fp16 or fp32 alike; the leading dims (one or more) are the tokens', strided views, such as parts of one projection's
    rows, are read in place.  positions int32 or int64 [axes, ..], with at least the rotary's axes, over the same tokens
    (expanded views too); negative ones turn back.  inverse turns by the negative angles.  out_q, out_k: written instead of new
    tensors; they may be q and k themselves, or other views with one stride per token."""
    shape, dtype = q.shape, q.dtype
    if len(shape) < 3 or shape[-1] != rotary.dim:
        raise RuntimeError(f"q must be [.., H, {rotary.dim}], got {tuple(shape)}")
    code = _TYPES.get(dtype)
    if code is None or (k is not None and k.dtype is not dtype):
        raise RuntimeError(f"q and k must be bfloat16, float16 or float32 alike, got {dtype} and {None if k is None else k.dtype}")
    if k is not None and (k.shape[:-2] != shape[:-2] or len(k.shape) != len(shape) or k.shape[-1] != rotary.dim):
        raise RuntimeError(f"k must be [.., kv_heads, {rotary.dim}] over q's tokens {tuple(shape[:-2])}, got {tuple(k.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.shape[1:] != shape[:-2] or positions.dim() < 2 or positions.size(0) < rotary.axes:
        raise RuntimeError(f"positions must be [axes, {', '.join(map(str, shape[:-2]))}] with {rotary.axes} axes or more, got "
                           f"{tuple(positions.shape)}")
    _one_device(rotary._index, q, k, positions, out_q, out_k)
    if k is None and out_k is not None:
        raise RuntimeError("out_k without k")
    n = math.prod(shape[:-2])
    if positions.dim() > 2:
        positions = positions.reshape(positions.size(0), n)
    unit = 4 if dtype is not torch.float32 else 8
    tensors = []
    for name, x, out in (("out_q", q, out_q), ("out_k", k, out_k)):
        if x is None:
            tensors.append((None, 0, 0, None, None, 0, 0, 0))
            continue
        if out is None:
            out = torch.empty(x.shape, dtype=dtype, device=x.device)
        elif out.shape != x.shape or out.dtype is not dtype:
            raise RuntimeError(f"{name} must be {dtype} {tuple(x.shape)}, got {out.dtype} {tuple(out.shape)}")
        to = _token_stride(out)
        if n and (to is None or to[0] % 2 or to[1] % 2 or out.data_ptr() % unit or (n > 1 and not to[0]) or (x.size(-2) > 1 and not to[1])):
            raise RuntimeError(f"{name}: rows must be contiguous, aligned to two elements and one stride per token apart, got strides {out.stride()}")
        flat, t, h = _flat(x, unit)
        tensors.append((flat.data_ptr(), t, h, out, out.data_ptr(), *(to or (0, 0)), x.size(-2)))
    (qp, qt, qh, oq, oqp, oqt, oqh, H), (kp, kt, kh, ok, okp, okt, okh, hk) = tensors
    if n == 0 or H + hk == 0:
        return oq, ok
    st = positions.stride()
    dev = rotary.device
    with _lib.on_device(dev):
        rc = _lib.hot("aekv_rotate_axes")(
            qp, kp, code, n, H, hk, rotary.dim, qt, qh, kt, kh, positions.data_ptr(), _lib.I32 if positions.dtype is torch.int32 else _lib.I64,
            positions.size(0), st[0], st[1], *rotary._args, int(bool(inverse)), oqp, okp, oqt, oqh, okt, okh, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "aekv_rotate_axes")
    return oq, ok
