"""A paged per-head KV cache held in TurboQuant codes: filled, attended and kept within a budget in place.

PolarQuant codes K and V entries of any attention (one vector per token and KV head); here they live in pages that
sequences share through page tables, and nothing is ever decoded to memory:

  append_tokens     codes the K and V of new tokens straight into their slots (bit for bit PolarQuant.encode)
  paged_attention   the newest tokens' attention over their sequence's slots, heads grouped over KV heads, optionally
                    adding every slot's attention weight to a tracker
  evict_by_weight   brings sequences back to a budget of slots by accumulated weight

A PagedKVCache is one layer's pool; page table int32 [B, max_pages], lengths and the like int32 [B] are shared by the
layers and only read here: after a step the caller adds the new tokens to `lengths`, after an eviction of every layer it
clamps them to `keep`.  Slot p of sequence b is row p % page_size of page table[b, p // page_size].  The tables and counts
are device data that no host check can see, so a slot outside the table or a page outside the pool is skipped, never
accessed.  Pages may be shared between sequences as long as nothing writes to them: append_tokens and evict_by_weight
write to the pages of the slots they fill.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .decode import _check_out, _i32, _sink_f32
from .turbo_quant import PolarQuant


class PagedKVCache:
    """One layer's pool of pages: codes [pages, kv_heads, page_size, row] and fp32 scales [pages, kv_heads, page_size],
    for K and for V.  head dim 64 or 128, page_size a power of two from 16 to 4096."""

    def __init__(self, quant: PolarQuant, pages: int, kv_heads: int, dim: int, *, page_size: int = 64,
                 device: Optional[torch.device] = None):
        if dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head dim must be 64 or 128, got {dim}")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size must be a power of two from 16 to 4096, got {page_size}")
        if pages < 1 or kv_heads < 1:
            raise ValueError(f"PagedKVCache needs pages, kv_heads >= 1, got {pages}, {kv_heads}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        rows = (int(pages), int(kv_heads), int(page_size))
        dtype = torch.int8 if quant.bits == 8 else torch.uint8
        row = dim * quant.bits // 8
        tensors = [torch.zeros(rows + (row,), dtype=dtype, device=dev) if i % 2 == 0 else
                   torch.zeros(rows, dtype=torch.float32, device=dev) for i in range(4)]
        _lib.require_device("PagedKVCache", *tensors)  # (the calls compare their tensors' device with the cache's)
        self._set(quant, *tensors)
        self._diag = quant._diag(self.dim, self.device)  # (here: a first call may be captured, which a copy from the host may not)

    def _set(self, quant, k_codes, k_scale, v_codes, v_scale) -> None:
        self.quant, self.bits = quant, quant.bits
        self._tensors = (k_codes, k_scale, v_codes, v_scale)
        self._ptrs = tuple(t.data_ptr() for t in self._tensors)  # (the cache owns its tensors: they stay where they are)
        self.pages, self.kv_heads, self.page_size = k_scale.shape
        self.dim = k_codes.size(3) * (1 if quant.bits == 8 else 2)
        self.device, self._index = k_codes.device, k_codes.get_device()

    k_codes = property(lambda self: self._tensors[0])
    k_scale = property(lambda self: self._tensors[1])
    v_codes = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    @classmethod
    def from_tensors(cls, quant: PolarQuant, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor,
                     v_scale: torch.Tensor) -> "PagedKVCache":
        """A cache over existing pools (used in place: contiguous, on one device)."""
        _lib.require_device("k_codes", k_codes, k_scale, v_codes, v_scale)
        want = torch.int8 if quant.bits == 8 else torch.uint8
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape:
            raise RuntimeError(f"codes must be [pages, kv_heads, page_size, row], got {tuple(k_codes.shape)} and "
                               f"{tuple(v_codes.shape)}")
        if k_codes.dtype != want or v_codes.dtype != want:
            raise RuntimeError(f"{quant.bits}-bit codes must be {want}, got {k_codes.dtype} and {v_codes.dtype}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or t.shape != k_codes.shape[:3]:
                raise RuntimeError(f"{name} must be float32 {tuple(k_codes.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
        for t in (k_codes, k_scale, v_codes, v_scale):
            if not t.is_contiguous() or t.data_ptr() % 16 or t.device != k_codes.device:
                raise RuntimeError("codes and scales must be contiguous, 16-byte aligned and on one device")
        self = cls.__new__(cls)
        self._set(quant, k_codes, k_scale, v_codes, v_scale)
        if self.dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head dim must be 64 or 128, got {self.dim}")
        if self.page_size < 16 or self.page_size > 4096 or self.page_size & (self.page_size - 1):
            raise ValueError(f"PagedKVCache: page_size must be a power of two from 16 to 4096, got {self.page_size}")
        self._diag = quant._diag(self.dim, self.device)
        return self

    def decode(self, page_table: torch.Tensor, length: int, out_dtype: torch.dtype = torch.bfloat16):
        """(K, V) [kv_heads, length, dim] of one sequence's first slots, decoded (page_table [max_pages]); 0 for the slots of
        a page outside the pool."""
        _one_device(self._index, page_table)
        if page_table.dim() != 1 or page_table.is_floating_point():
            raise RuntimeError(f"page_table must be int32 [max_pages], got {page_table.dtype} {tuple(page_table.shape)}")
        length, slots = int(length), page_table.size(0) * self.page_size
        if not 0 <= length <= slots:
            raise RuntimeError(f"decode of {length} slots: page_table has {slots} slots")
        if not self.pages:
            return tuple(torch.zeros((self.kv_heads, length, self.dim), dtype=out_dtype, device=self.device) for _ in range(2))
        slot = torch.arange(length, device=self.device)
        page, row = page_table.long()[slot // self.page_size], slot % self.page_size
        none = (page < 0) | (page >= self.pages)
        page = page.masked_fill(none, 0)
        return tuple(self.quant.decode(c[page, :, row], s[page, :, row].masked_fill(none[:, None], 0.0).unsqueeze(-1), out_dtype).transpose(0, 1)
                     for c, s in ((self.k_codes, self.k_scale), (self.v_codes, self.v_scale)))


class SlotTracker:
    """Per sequence, KV head and slot of one layer: `weights` fp32, the attention weight accumulated since the slot was
    filled, and `tokens` int32, the token index that it holds ([B, kv_heads, capacity], views of one int32 tensor).

    Give it the table's slots (max_pages * page_size), or as many as its sequences ever fill: the calls with a tracker end a
    sequence at its capacity.  What lies behind is not seen by a tracked attention, as its weight could not be counted, and
    lost to an eviction."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, *, device: Optional[torch.device] = None):
        if batch < 1 or kv_heads < 1 or capacity < 1:
            raise ValueError(f"SlotTracker needs batch, kv_heads, capacity >= 1, got {batch}, {kv_heads}, {capacity}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        storage = torch.zeros((2, int(batch), int(kv_heads), int(capacity)), dtype=torch.int32, device=dev)
        _lib.require_device("SlotTracker", storage)
        self._set(storage)

    def _set(self, storage: torch.Tensor) -> None:
        self._storage, self._weights, self._tokens = storage, storage[0].view(torch.float32), storage[1]
        self.batch, self.kv_heads, self.capacity = storage.shape[1:]

    storage = property(lambda self: self._storage)
    weights = property(lambda self: self._weights)
    tokens = property(lambda self: self._tokens)

    @classmethod
    def from_tensor(cls, storage: torch.Tensor) -> "SlotTracker":
        """A tracker over an existing int32 [2, B, kv_heads, capacity] (used in place)."""
        _lib.require_device("storage", storage)
        if storage.dtype != torch.int32 or storage.dim() != 4 or storage.size(0) != 2 or not storage.is_contiguous() \
                or storage.data_ptr() % 16:
            raise RuntimeError(f"storage must be contiguous, 16-byte aligned int32 [2, B, kv_heads, capacity], got {storage.dtype} "
                               f"{tuple(storage.shape)}")
        self = cls.__new__(cls)
        self._set(storage)
        return self


# The calls below are made once per layer and token, so their host cost counts: every tensor method costs some 0.1 us, a
# new view or conversion several times that, so what is already in the kernels' form is passed as it is.
_INT32 = torch.int32
_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


def _counts(name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    """A per-sequence count as contiguous int32 [n]."""
    if t.shape != (n,) or t.is_floating_point():
        raise RuntimeError(f"{name} must be int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t if t.dtype is _INT32 and t.is_contiguous() else _i32(t)


def _table(page_table: torch.Tensor) -> torch.Tensor:
    if page_table.dim() != 2 or page_table.is_floating_point():
        raise RuntimeError(f"page_table must be int32 [B, max_pages], got {page_table.dtype} {tuple(page_table.shape)}")
    return page_table if page_table.dtype is _INT32 and page_table.is_contiguous() else _i32(page_table)


def _one_device(index: int, *tensors: Optional[torch.Tensor]) -> None:
    """The kernels get raw pointers: every tensor of a call must be on the device `index`."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"every tensor of the call must be on the HIP device {index}, got one on {t.device}")


def _given(workspace: torch.Tensor) -> torch.Tensor:
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise RuntimeError(f"workspace must be contiguous uint8, got {workspace.dtype} {tuple(workspace.shape)}")
    return workspace


def _check_tracker(tracker: SlotTracker, cache: PagedKVCache, B: int) -> None:
    if tracker.batch != B or tracker.kv_heads != cache.kv_heads:
        raise RuntimeError(f"tracker of {tracker.batch} sequences x {tracker.kv_heads} heads does not match {B} x "
                           f"{cache.kv_heads}")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, ...]]:
    """t [.., heads, D] with rows the kernels can read in place (contiguous in D, 16-byte aligned; else a copy), and its
    strides."""
    st = t.stride()
    e = 8 if t.dtype is not torch.float32 else 4
    if st[-1] == 1 and not t.data_ptr() % 16:
        for s in st[:-1]:
            if s % e:
                break
        else:
            return t, st
    t = _lib.aligned(t, 16)
    return t, t.stride()


def _token_rows(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """[B, T, heads, D] as B * T tokens: the tensor (or a copy), the stride of a token and of a head."""
    t, st = _rows(t)
    B, T = t.size(0), t.size(1)
    if T == 1:
        return t, st[0], st[2]
    if B == 1 or st[0] == T * st[1]:
        return t, st[1], st[2]
    t = t.contiguous()
    return t, t.stride(1), t.stride(2)


def append_tokens(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                  start: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                  tracker: Optional[SlotTracker] = None, token: Optional[torch.Tensor] = None) -> None:
    """Code the K and V of new tokens into slots start[b], start[b] + 1, ... of their sequences.

    k, v [B, T, kv_heads, D] (T tokens of every sequence), or packed [N, kv_heads, D] with cu_seqlens int32 [B + 1]
    (sequence b's tokens are cu_seqlens[b] .. cu_seqlens[b + 1]; rows outside are skipped); bf16, fp16 or fp32, strided
    views are read in place.  The codes are PolarQuant.encode's, bit for bit.  With a tracker, the slots' weights start at
    0 and their token indices at token[b] (int32 [B]: the sequence's tokens before this call); slots past its capacity get
    codes alone."""
    B = page_table.size(0)
    shape, dtype = k.shape, k.dtype
    if len(shape) != (4 if cu_seqlens is None else 3) or v.shape != shape or shape[-2] != cache.kv_heads or shape[-1] != cache.dim:
        want = "[B, T" if cu_seqlens is None else "[N"
        raise RuntimeError(f"append_tokens expects k and v {want}, {cache.kv_heads}, {cache.dim}], got {tuple(shape)} "
                           f"and {tuple(v.shape)}")
    code = _TYPES.get(dtype)
    if code is None or v.dtype is not dtype:
        raise RuntimeError(f"k and v must be bfloat16, float16 or float32 alike, got {dtype} and {v.dtype}")
    if (tracker is None) != (token is None):
        raise RuntimeError("append_tokens: a tracker and the sequences' token counts come together")
    _one_device(cache._index, k, v, page_table, start, cu_seqlens, token, None if tracker is None else tracker._storage)
    table, start = _table(page_table), _counts("start", start, B)
    if cu_seqlens is None:
        if shape[0] != B:
            raise RuntimeError(f"k holds {shape[0]} sequences, page_table {B}")
        cu, n = None, B * shape[1]
        k, kt, kh = _token_rows(k)
        v, vt, vh = _token_rows(v)
    else:
        cu, n = _counts("cu_seqlens", cu_seqlens, B + 1), shape[0]
        k, (kt, kh, _) = _rows(k)
        v, (vt, vh, _) = _rows(v)
    weights = tokens = first = None
    capacity = 0
    if tracker is not None:
        _check_tracker(tracker, cache, B)
        token = _counts("token", token, B)
        weights, tokens, first, capacity = tracker._weights.data_ptr(), tracker._tokens.data_ptr(), token.data_ptr(), tracker.capacity
    kc, ks, vc, vs = cache._ptrs
    dev = cache.device
    with _lib.on_device(dev):
        rc = _lib.hot("aekv_kv_append")(
            k.data_ptr(), v.data_ptr(), code, kt, kh, vt, vh, n, None if cu is None else cu.data_ptr(), B,
            start.data_ptr(), cache.dim, cache.bits, cache._diag.data_ptr(), kc, ks, vc, vs, cache.pages, cache.kv_heads,
            cache.page_size, table.data_ptr(), table.size(1), weights, tokens, capacity, first, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "aekv_kv_append")


def paged_attention_workspace(B: int, T: int, H: int, kv_heads: int, dim: int, slots: int, device, *,
                              tracked: bool = False) -> torch.Tensor:
    """Workspace of paged_attention; slots = page_table.size(1) * page_size."""
    if H < 1 or kv_heads < 1 or H % kv_heads:
        raise RuntimeError(f"{H} query heads are no multiple of {kv_heads} KV heads")
    n = _lib.paged_ws_bytes(int(B), int(T), int(H), int(kv_heads), int(dim), int(slots), int(tracked))
    return torch.empty(n, dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                    softmax_scale: float, *, sink: Optional[torch.Tensor] = None,
                    tracker: Optional[SlotTracker] = None, workspace: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest T tokens of every sequence, its last T slots, over its slots [0, lengths[b]).

    q [B, T, H, D] bf16 or fp16 (strided views are read in place), H a multiple of the cache's KV heads: query head h
    reads KV head h // (H // kv_heads).  Token t sees slots j < lengths[b] - T + 1 + t, as far as the table has them, and
    with a tracker as far as its capacity goes.  sink [H] (or a scalar): a logit counted once in the normaliser.  A row that sees nothing gives 0.  With a tracker, weights[b, kv head, j] grows by
    the attention weight of slot j, summed over the group's heads and the T tokens.  Returns [B, T, H, D] like q."""
    shape, dtype = q.shape, q.dtype
    if len(shape) != 4 or shape[3] != cache.dim:
        raise RuntimeError(f"q must be [B, T, H, {cache.dim}], got {tuple(shape)}")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise RuntimeError(f"q must be bfloat16 or float16, got {dtype}")
    B, T, H, D = shape
    heads = cache.kv_heads
    if H % heads:
        raise RuntimeError(f"{H} query heads are no multiple of {heads} KV heads")
    _one_device(cache._index, q, page_table, lengths, sink, workspace, out, None if tracker is None else tracker._storage)
    table, lengths = _table(page_table), _counts("lengths", lengths, B)
    table_rows, max_pages = table.shape
    if table_rows != B:
        raise RuntimeError(f"q holds {B} sequences, page_table {table_rows}")
    q, st = _rows(q)
    sk = None if sink is None else _sink_f32(sink, H)
    dev = cache.device
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    else:
        _check_out("out", out, dtype, q.numel(), dev)
    weights, capacity, tracked = None, 0, 0
    if tracker is not None:
        _check_tracker(tracker, cache, B)
        weights, capacity, tracked = tracker._weights.data_ptr(), tracker.capacity, 1
    kc, ks, vc, vs = cache._ptrs
    need = _lib.paged_ws_bytes(B, T, H, heads, D, max_pages * cache.page_size, tracked) if workspace is None else 0
    with _lib.on_device(dev):
        stream = _lib.raw_stream(dev)
        ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream) if need else None
        rc = _lib.hot("aekv_paged_attention")(
            q.data_ptr(), _TYPES[dtype], st[0], st[1], st[2], B, T, H, D, cache.bits, cache._diag.data_ptr(), kc, ks, vc, vs,
            cache.pages, heads, cache.page_size, table.data_ptr(), max_pages, lengths.data_ptr(),
            None if sk is None else sk.data_ptr(), weights, capacity, float(softmax_scale),
            None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), out.data_ptr(), stream)
    if rc:
        _lib.check(rc, "aekv_paged_attention")
    return out if out.dim() == 4 else out.view(shape)


def evict_workspace(B: int, kv_heads: int, keep: int, slots: int, device) -> torch.Tensor:
    """Workspace of evict_by_weight; slots = min(page_table.size(1) * page_size, tracker.capacity)."""
    return torch.empty(_lib.evict_ws_bytes(int(B), int(kv_heads), int(keep), int(slots)), dtype=torch.uint8, device=device)


def evict_by_weight(cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, tracker: SlotTracker,
                    seen: torch.Tensor, keep: int, *, first: int = 0, recent: int = 0,
                    workspace: Optional[torch.Tensor] = None) -> None:
    """Bring every (sequence, KV head) with more than `keep` slots back to `keep`, in place.

    The slots that stay are those of the first `first` tokens and of the last `recent` of the seen[b] tokens (by the
    tracker's token indices), then the ones with the largest accumulated weight (equal ones: the lower slot; NaN above
    every number).  Kept slots below `keep` stay where they are; the evicted ones below `keep`, in order, take the kept
    slots from `keep` on, in order, with their weight and token index: cached keys carry their rotation, so attention
    does not depend on the order of the slots.  A sequence ends at the tracker's capacity: slots behind it are not among
    those that can stay.  `lengths` is only read: clamp it to `keep` once every layer is done."""
    B, max_pages = page_table.shape
    _one_device(cache._index, page_table, lengths, seen, workspace, tracker._storage)
    table, lengths, seen = _table(page_table), _counts("lengths", lengths, B), _counts("seen", seen, B)
    _check_tracker(tracker, cache, B)
    keep, first, recent = int(keep), int(first), int(recent)
    dev = cache.device
    kc, ks, vc, vs = cache._ptrs
    need = _lib.evict_ws_bytes(B, cache.kv_heads, keep, min(max_pages * cache.page_size, tracker.capacity)) if workspace is None else 0
    with _lib.on_device(dev):
        stream = _lib.raw_stream(dev)
        ws = _given(workspace) if workspace is not None else _lib.workspace(need, dev, stream) if need else None
        rc = _lib.hot("aekv_kv_evict")(
            cache.dim, cache.bits, kc, ks, vc, vs, cache.pages, cache.kv_heads, cache.page_size, table.data_ptr(), max_pages,
            B, lengths.data_ptr(), tracker._weights.data_ptr(), tracker._tokens.data_ptr(), tracker.capacity,
            seen.data_ptr(), keep, first, recent, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
            stream)
    if rc:
        _lib.check(rc, "aekv_kv_evict")
