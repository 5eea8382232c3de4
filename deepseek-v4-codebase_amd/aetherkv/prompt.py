"""Causal attention over whole prompts: sequences of different lengths packed into one buffer, heads grouped over KV
heads.  The attention of the prefill that fills a paged cache (aetherkv.paged), beside the chunked prefill over
compressed blocks (aetherkv.prefill) and the dense drop-in (aetherkv.sparse_attention.tiled_prefill_attention), which
attend every source from every target."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .decode import _check_out, _sink_f32
from .paged import _TYPES, _counts, _given, _one_device, _rows


def prompt_workspace(B: int, n_q: int, n_k: int, H: int, kv_heads: int, dim: int, device) -> torch.Tensor:
    """Workspace of prompt_attention (B sequences, n_q rows of q, n_k of k; empty where it needs none)."""
    return torch.empty(_lib.prompt_ws_bytes(int(B), int(n_q), int(n_k), int(H), int(kv_heads), int(dim)), dtype=torch.uint8, device=device)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, softmax_scale: float, *,
                     cu_seqlens_k: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None,
                     return_lse: bool = False, workspace: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None):
    """out_i = sum_j p_ij v_j over the keys j <= i + (keys - queries) of query i's sequence.

    q [N, H, D], k and v [M, kv_heads, D], bf16 or fp16, D 64 or 128, H a multiple of kv_heads (query head h reads KV head
    h // (H // kv_heads)); strided views, such as parts of one projection's rows, are read in place.  cu_seqlens int32
    [B + 1]: sequence b's queries are rows cu_seqlens[b] .. cu_seqlens[b + 1]; cu_seqlens_k likewise for the keys (None:
    the same), so that a later chunk of a prompt comes with the keys before it.  sink [H] (or a scalar): a logit counted
    once in the normaliser.  Each weight p_ij is rounded once to the type of q, k and v for its product with v; all sums are
    fp32.  A query that sees nothing gives 0.  Rows of q in no sequence: a given `out` keeps them, a new
    one holds 0.  Returns out [N, H, D], with return_lse (out, lse fp32 [N, H]): the log of every row's sum of
    exponentials, the sink's among them (-inf for rows in no sequence)."""
    shape, dtype, ks = q.shape, q.dtype, k.shape
    if len(shape) != 3 or len(ks) != 3 or v.shape != ks or ks[2] != shape[2]:
        raise RuntimeError(f"prompt_attention expects q [N, H, D] and k, v [M, kv_heads, D], got {tuple(shape)}, "
                           f"{tuple(ks)} and {tuple(v.shape)}")
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype is not dtype or v.dtype is not dtype:
        raise RuntimeError(f"q, k and v must be bfloat16 or float16 alike, got {dtype}, {k.dtype} and {v.dtype}")
    N, H, D = shape
    M, hk, _ = ks
    if hk < 1 or H % hk:
        raise RuntimeError(f"{H} query heads are no multiple of {hk} KV heads")
    if cu_seqlens.dim() != 1 or cu_seqlens.size(0) < 2:
        raise RuntimeError(f"cu_seqlens must be int32 [B + 1], got {tuple(cu_seqlens.shape)}")
    B = cu_seqlens.size(0) - 1
    _lib.require_device("q", q)
    dev = q.device
    _one_device(q.get_device(), k, v, cu_seqlens, cu_seqlens_k, sink, workspace, out)
    cq = _counts("cu_seqlens", cu_seqlens, B + 1)
    if cu_seqlens_k is None:
        if M != N:
            raise RuntimeError(f"{N} queries and {M} keys: cu_seqlens_k is needed")
        ck = cq
    else:
        ck = _counts("cu_seqlens_k", cu_seqlens_k, B + 1)
    q, (qt, qh, _) = _rows(q)
    k, (kt, kh, _) = _rows(k)
    v, (vt, vh, _) = _rows(v)
    sk = None if sink is None else _sink_f32(sink, H)
    clear = 0
    if out is None:
        out, clear = torch.empty(shape, dtype=dtype, device=dev), 1
    else:
        _check_out("out", out, dtype, q.numel(), dev)
    lse = torch.empty((N, H), dtype=torch.float32, device=dev) if return_lse else None
    need = _lib.prompt_ws_bytes(B, N, M, H, hk, D) if workspace is None else 0
    with _lib.on_device(dev):
        stream = _lib.raw_stream(dev)
        ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream) if need else None
        rc = _lib.hot("aekv_prompt_attention")(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _TYPES[dtype], qt, qh, kt, kh, vt, vh, cq.data_ptr(),
            ck.data_ptr(), B, N, M, H, hk, D, None if sk is None else sk.data_ptr(), float(softmax_scale), out.data_ptr(),
            None if lse is None else lse.data_ptr(), clear, None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel(), stream)
    if rc:
        _lib.check(rc, "aekv_prompt_attention")
    out = out if out.dim() == 3 else out.view(shape)
    return (out, lse) if return_lse else out
