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


def _token_stride(shape, st) -> Optional[Tuple[int, int]]:
    """(token, head) strides of [.., heads, D], its leading dims as one, or None where they are not one stride apart."""
    if st[-1] != 1 and shape[-1] > 1:
        return None
    if len(shape) == 3:
        return st[0], st[1]
    token, tokens = 0, 1
    for i in range(len(shape) - 3, -1, -1):
        if shape[i] == 1:
            continue
        if tokens == 1:
            token = st[i]
        elif st[i] != token * tokens:
            return None
        tokens *= shape[i]
    return token, st[-2]


def _readable(t: torch.Tensor, shape, n: int, unit: int):
    """t [.., heads, D] of n tokens, or a copy that the kernel can read; its address and (token, head) strides."""
    st, at = _token_stride(shape, t.stride()), t.data_ptr()
    if st is None or at % unit or (st[0] % 2 and n > 1) or (st[1] % 2 and shape[-2] > 1):
        t = _lib.aligned(t, 16)
        st, at = (shape[-2] * shape[-1], shape[-1]), t.data_ptr()
    return t, at, st[0] & -2, st[1] & -2  # (a stride that no second row needs may be odd)


def _writable(name: str, out: torch.Tensor, shape, n: int, dtype, unit: int):
    if out.shape != shape or out.dtype is not dtype:
        raise RuntimeError(f"{name} must be {dtype} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
    st, at = _token_stride(shape, out.stride()), out.data_ptr()
    if st is None or at % unit or (n > 1 and (st[0] % 2 or not st[0])) or (shape[-2] > 1 and (st[1] % 2 or not st[1])):
        raise RuntimeError(f"{name}: rows must be contiguous, aligned to two elements and one stride per token apart, got strides {out.stride()}")
    return at, st[0] & -2, st[1] & -2


def rotate_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: AxisRotary, *, inverse: bool = False,
                out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [.., H, D] and k [.., kv_heads, D] (or None) turned by their tokens' positions: (q, k) like them.

    bf16, fp16 or fp32 alike; the leading dims (one or more) are the tokens', strided views, such as parts of one projection's
    rows, are read in place.  positions int32 or int64 [axes, ..], with at least the rotary's axes, over the same tokens
    (expanded views too); negative ones turn back.  inverse turns by the negative angles.  out_q, out_k: written instead of new
    tensors; they may be q and k themselves, or other views with one stride per token that share no memory with q and k."""
    # (made once per layer and token: what a tensor method costs counts here, as in aetherkv.paged)
    shape, dtype, dim = q.shape, q.dtype, rotary.dim
    lead = shape[:-2]
    if len(shape) < 3 or shape[-1] != dim:
        raise RuntimeError(f"q must be [.., H, {dim}], got {tuple(shape)}")
    code = _TYPES.get(dtype)
    if code is None or (k is not None and k.dtype is not dtype):
        raise RuntimeError(f"q and k must be bfloat16, float16 or float32 alike, got {dtype} and {None if k is None else k.dtype}")
    ptype, pshape = positions.dtype, positions.shape
    if ptype is not torch.int32 and ptype is not torch.int64:
        raise RuntimeError(f"positions must be int32 or int64, got {ptype}")
    if pshape[1:] != lead or len(pshape) < 2 or pshape[0] < rotary.axes:
        raise RuntimeError(f"positions must be [axes, {', '.join(map(str, lead))}] with {rotary.axes} axes or more, got {tuple(pshape)}")
    index, dev = rotary._index, rotary.device
    _one_device(index, q, k, positions, out_q, out_k)
    kt = kh = hk = kot = koh = 0
    kp = kop = None
    if k is not None:
        kshape = k.shape
        if kshape[:-2] != lead or len(kshape) != len(shape) or kshape[-1] != dim:
            raise RuntimeError(f"k must be [.., kv_heads, {dim}] over q's tokens {tuple(lead)}, got {tuple(kshape)}")
        hk = kshape[-2]
    elif out_k is not None:
        raise RuntimeError("out_k without k")
    n = lead[0] if len(lead) == 1 else math.prod(lead)
    unit = 4 if dtype is not torch.float32 else 8
    H = shape[-2]
    if out_q is None:
        out_q = torch.empty(shape, dtype=dtype, device=dev)
        qop, qot, qoh = out_q.data_ptr(), H * dim, dim
    else:
        qop, qot, qoh = _writable("out_q", out_q, shape, n, dtype, unit)
    if k is not None:
        if out_k is None:
            out_k = torch.empty(kshape, dtype=dtype, device=dev)
            kop, kot, koh = out_k.data_ptr(), hk * dim, dim
        else:
            kop, kot, koh = _writable("out_k", out_k, kshape, n, dtype, unit)
    if n == 0 or H + hk == 0:
        return out_q, out_k
    q, qp, qt, qh = _readable(q, shape, n, unit)
    if k is not None:
        k, kp, kt, kh = _readable(k, kshape, n, unit)
    if len(pshape) > 2:
        positions = positions.reshape(pshape[0], n)
    pa, pt = positions.stride()
    with _lib.on_device(dev):
        rc = _lib.hot("aekv_rotate_axes")(
            qp, kp, code, n, H, hk, dim, qt, qh, kt, kh, positions.data_ptr(), _lib.I32 if ptype is torch.int32 else _lib.I64,
            pshape[0], pa, pt, *rotary._args, 1 if inverse else 0, qop, kop, qot, qoh, kot, koh, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "aekv_rotate_axes")
    return out_q, out_k
