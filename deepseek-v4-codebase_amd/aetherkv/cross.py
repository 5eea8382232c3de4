"""Attention over the states of an encoder, whose length is another than the queries': packed sequences, heads grouped over KV
heads, several sequences over the same states.  Beside the causal attention of prompts (aetherkv.prompt) and of a paged cache
(aetherkv.paged)."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .decode import _check_out, _sink_f32
from .paged import _TYPES, _counts, _given, _one_device, _rows


def cross_workspace(B: int, E: int, n_q: int, n_k: int, H: int, kv_heads: int, dim: int, device) -> torch.Tensor:
    """Workspace of cross_attention (B sequences over E states, n_q rows of q, n_k of k)."""
    return torch.empty(_lib.cross_ws_bytes(int(B), int(E), int(n_q), int(n_k), int(H), int(kv_heads), int(dim)), dtype=torch.uint8, device=device)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_k: torch.Tensor, softmax_scale: float, *,
                    cu_seqlens: Optional[torch.Tensor] = None, states: Optional[torch.Tensor] = None,
                    sink: Optional[torch.Tensor] = None, return_lse: bool = False, workspace: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None):
    """out_i = sum_j p_ij v_j over all keys j of the states that query i's sequence reads.

    q [N, H, D], k and v [M, kv_heads, D], bf16 or fp16, D 64 or 128, H a multiple of kv_heads (query head h reads KV head
    h // (H // kv_heads)); strided views, such as parts of one projection's rows, are read in place.  cu_seqlens_k int32
    [E + 1]: the e-th states are rows cu_seqlens_k[e] .. cu_seqlens_k[e + 1].  cu_seqlens int32 [B + 1] likewise for the
    queries; None: one query each (a decode step).  states int32 [B]: the states that sequence b reads (None: the b-th; one
    outside 0 .. E - 1: none); neighbours over the same states, such as the answers to one input, read them once for all.
    sink [H] (or a scalar): a logit counted once in the normaliser.  Each weight p_ij is rounded to the type of q, k and v for
    its product with v, off by 2^-8 (fp16 2^-11) of itself at most; where there are few rows (q rows times heads of a KV head, on
    average over the states in use at most 16, or 32 at D 64), the rest is multiplied as well, off by 2^-16 (2^-22).  All sums are
    fp32.  A query over no keys gives 0.  Rows of q in no sequence: a given `out` keeps
    them, a new one holds 0.  Returns out [N, H, D], with return_lse (out, lse fp32 [N, H]): the log of every row's sum of
    exponentials, the sink's among them (-inf for rows in no sequence)."""
    shape, dtype, ks = q.shape, q.dtype, k.shape
    if len(shape) != 3 or len(ks) != 3 or v.shape != ks or ks[2] != shape[2]:
        raise RuntimeError(f"cross_attention expects q [N, H, D] and k, v [M, kv_heads, D], got {tuple(shape)}, {tuple(ks)} and {tuple(v.shape)}")
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype is not dtype or v.dtype is not dtype:
        raise RuntimeError(f"q, k and v must be bfloat16 or float16 alike, got {dtype}, {k.dtype} and {v.dtype}")
    N, H, D = shape
    M, hk, _ = ks
    if hk < 1 or H % hk:
        raise RuntimeError(f"{H} query heads are no multiple of {hk} KV heads")
    if cu_seqlens_k.dim() != 1 or cu_seqlens_k.size(0) < 1:
        raise RuntimeError(f"cu_seqlens_k must be int32 [E + 1], got {tuple(cu_seqlens_k.shape)}")
    if cu_seqlens is not None and (cu_seqlens.dim() != 1 or cu_seqlens.size(0) < 2):
        raise RuntimeError(f"cu_seqlens must be int32 [B + 1], got {tuple(cu_seqlens.shape)}")
    E, B = cu_seqlens_k.size(0) - 1, N if cu_seqlens is None else cu_seqlens.size(0) - 1
    _lib.require_device("q", q)
    dev = q.device
    _one_device(q.get_device(), k, v, cu_seqlens_k, cu_seqlens, states, sink, workspace, out)
    ck = _counts("cu_seqlens_k", cu_seqlens_k, E + 1)
    cq = None if cu_seqlens is None else _counts("cu_seqlens", cu_seqlens, B + 1)
    if states is not None:
        states = _counts("states", states, B)
    elif E != B:
        raise RuntimeError(f"{B} sequences and {E} states: which of them each sequence reads is needed (states)")
    q, (qt, qh, _) = _rows(q)
    k, (kt, kh, _) = _rows(k)
    v, (vt, vh, _) = _rows(v)
    if (kt < D or vt < D) and M > 1:  # (rows that overlap: the kernels tell a sequence's end by where its last row ends)
        k, v = k.contiguous(), v.contiguous()
        (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
    sk = None if sink is None else _sink_f32(sink, H)
    clear = 0
    if out is None:
        out, clear = torch.empty(shape, dtype=dtype, device=dev), 1
    else:
        _check_out("out", out, dtype, q.numel(), dev)
    lse = torch.empty((N, H), dtype=torch.float32, device=dev) if return_lse else None
    need = _lib.cross_ws_bytes(B, E, N, M, H, hk, D) if workspace is None else 0
    with _lib.on_device(dev):
        stream = _lib.raw_stream(dev)
        ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream) if need else None
        rc = _lib.hot("aekv_cross_attention")(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _TYPES[dtype], qt, qh, kt, kh, vt, vh, None if cq is None else cq.data_ptr(),
            ck.data_ptr(), None if states is None else states.data_ptr(), B, E, N, M, H, hk, D, None if sk is None else sk.data_ptr(),
            float(softmax_scale), out.data_ptr(), None if lse is None else lse.data_ptr(), clear, None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel(), stream)
    if rc:
        _lib.check(rc, "aekv_cross_attention")
    out = out if out.dim() == 3 else out.view(shape)
    return (out, lse) if return_lse else out
