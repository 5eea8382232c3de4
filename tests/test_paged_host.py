"""Paged cache and prompt attention: host-side logic — refusals of the C entries and of the Python calls, workspace sizes,
and where slots lie (bad pages among them), checked on the CPU."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess
import sys

import pytest
import torch

import aetherkv._lib as L
from conftest import PKG_DIR, ROOT

FAKE, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001)


@pytest.fixture(scope="module")
def lib():
    if not L.available():
        pytest.fail("libaetherkv.so is not built (run __graft_entry__.build())")
    return L.lib()


def _pool(**kw):
    a = dict(k_codes=FAKE, k_scale=FAKE, v_codes=FAKE, v_scale=FAKE, pages=8, heads=2, page_size=16, table=FAKE, max_pages=4)
    a.update(kw)
    return a


def _append(lib, dtype=L.BF16, kt=256, kh=128, vt=256, vh=128, n=6, cu=None, B=3, start=FAKE, d=128, bits=4, k=FAKE, v=FAKE, diag=FAKE, weights=None,
            tokens=None, cap=0, token=None, **kw):
    p = _pool(**kw)
    return lib.aekv_kv_append(k, v, dtype, kt, kh, vt, vh, n, cu, B, start, d, bits, diag, p["k_codes"], p["k_scale"], p["v_codes"], p["v_scale"],
                              p["pages"], p["heads"], p["page_size"], p["table"], p["max_pages"], weights, tokens, cap, token, None)


def _attend(lib, q=FAKE, dtype=L.BF16, qb=512, qt=512, qh=128, B=3, T=1, H=4, d=128, bits=4, diag=FAKE, lengths=FAKE, sink=None, weights=None, cap=0, ws=FAKE,
            wsb=1 << 30, out=FAKE, **kw):
    p = _pool(**kw)
    return lib.aekv_paged_attention(q, dtype, qb, qt, qh, B, T, H, d, bits, diag, p["k_codes"], p["k_scale"], p["v_codes"], p["v_scale"], p["pages"],
                                    p["heads"], p["page_size"], p["table"], p["max_pages"], lengths, sink, weights, cap, 0.1, ws, wsb, out, None)


def _evict(lib, d=128, bits=4, B=3, lengths=FAKE, weights=FAKE, tokens=FAKE, cap=64, seen=FAKE, keep=16, first=0, recent=0, ws=FAKE, wsb=1 << 30, **kw):
    p = _pool(**kw)
    return lib.aekv_kv_evict(d, bits, p["k_codes"], p["k_scale"], p["v_codes"], p["v_scale"], p["pages"], p["heads"], p["page_size"], p["table"],
                             p["max_pages"], B, lengths, weights, tokens, cap, seen, keep, first, recent, ws, wsb, None)


def _prompt(lib, q=FAKE, k=FAKE, v=FAKE, dtype=L.BF16, st=(512, 128, 256, 128, 256, 128), cq=FAKE, ck=FAKE, B=2, nq=10, nk=10, H=4, hk=2, d=128, out=FAKE, ws=FAKE, wsb=1 << 30):
    return lib.aekv_prompt_attention(q, k, v, dtype, *st, cq, ck, B, nq, nk, H, hk, d, None, 0.1, out, None, 0, ws, wsb, None)


@pytest.mark.parametrize("call", [_append, _attend, _evict])
def test_pool_refusals(lib, call):
    assert call(lib, bits=5) == L.ERR_VALUE and "bits must be 4 or 8" in lib.aekv_last_error().decode()
    assert call(lib, d=96) == L.ERR_UNSUPPORTED
    assert call(lib, d=256) == L.ERR_UNSUPPORTED
    for ps in (0, 8, 24, 8192):
        assert call(lib, page_size=ps) == L.ERR_VALUE
    assert call(lib, heads=0) == L.ERR_SHAPE
    assert call(lib, pages=-1) == L.ERR_SHAPE
    assert call(lib, max_pages=1 << 28) == L.ERR_UNSUPPORTED
    assert call(lib, k_codes=ODD) == L.ERR_ALIGN
    assert call(lib, v_scale=ctypes.c_void_p(0x10004)) == L.ERR_ALIGN
    assert call(lib, v_codes=None) == L.ERR_VALUE
    assert call(lib, table=None) == L.ERR_VALUE


def test_append_refusals(lib):
    assert _append(lib, dtype=L.I32) == L.ERR_DTYPE
    assert _append(lib, n=7) == L.ERR_SHAPE  # no whole number of tokens for each of 3 sequences
    assert _append(lib, k=ODD) == L.ERR_ALIGN
    assert _append(lib, kt=255) == L.ERR_ALIGN
    assert _append(lib, start=None) == L.ERR_VALUE
    assert _append(lib, weights=FAKE) == L.ERR_VALUE  # without tokens
    assert _append(lib, n=1 << 31, cu=FAKE) == L.ERR_UNSUPPORTED
    assert _append(lib, n=0) == L.OK and _append(lib, B=0) == L.OK and _append(lib, max_pages=0, table=None) == L.OK


def test_attention_refusals(lib):
    assert _attend(lib, dtype=L.F32) == L.ERR_DTYPE
    assert _attend(lib, H=3) == L.ERR_SHAPE  # no multiple of 2 KV heads
    assert _attend(lib, q=ODD) == L.ERR_ALIGN
    assert _attend(lib, qh=100) == L.ERR_ALIGN
    assert _attend(lib, out=None) == L.ERR_VALUE
    assert _attend(lib, weights=FAKE, cap=-1) == L.ERR_SHAPE
    need = lib.aekv_paged_attention_workspace_size(3, 1, 4, 2, 128, 64, 1)
    assert need > 0
    assert _attend(lib, weights=FAKE, cap=64, wsb=need - 1) == L.ERR_WORKSPACE
    assert _attend(lib, weights=FAKE, cap=64, ws=None, wsb=need) == L.ERR_WORKSPACE
    assert _attend(lib, B=0) == L.OK and _attend(lib, T=0) == L.OK
    assert lib.aekv_paged_attention_workspace_size(0, 1, 4, 2, 128, 64, 1) == 0


def test_evict_refusals(lib):
    assert _evict(lib, keep=-1) == L.ERR_VALUE
    assert _evict(lib, keep=16, first=10, recent=7) == L.ERR_VALUE
    assert _evict(lib, first=-1) == L.ERR_VALUE
    assert _evict(lib, weights=None) == L.ERR_VALUE
    need = lib.aekv_kv_evict_workspace_size(3, 2, 16, 64)
    assert need >= 3 * 2 * 16 * 8
    assert _evict(lib, wsb=need - 1) == L.ERR_WORKSPACE
    assert _evict(lib, keep=64, ws=None, wsb=0) == L.OK  # no sequence can hold more
    assert _evict(lib, B=0) == L.OK
    assert lib.aekv_kv_evict_workspace_size(3, 2, 64, 64) == 0


def test_prompt_refusals(lib):
    assert _prompt(lib, dtype=L.F32) == L.ERR_DTYPE
    assert _prompt(lib, d=256) == L.ERR_UNSUPPORTED
    assert _prompt(lib, H=3) == L.ERR_SHAPE
    assert _prompt(lib, k=None) == L.ERR_VALUE
    assert _prompt(lib, cq=None) == L.ERR_VALUE
    assert _prompt(lib, v=ODD) == L.ERR_ALIGN
    assert _prompt(lib, st=(512, 128, 252, 128, 256, 128)) == L.ERR_ALIGN
    assert _prompt(lib, B=0) == L.ERR_SHAPE
    assert _prompt(lib, nq=0) == L.OK
    need = lib.aekv_prompt_attention_workspace_size(2, 10, 100000, 4, 2, 128)
    assert need > 0 and _prompt(lib, nk=100000, wsb=need - 1) == L.ERR_WORKSPACE
    assert _prompt(lib, nk=100000, ws=ctypes.c_void_p(0x10008), wsb=need) == L.ERR_ALIGN
    assert lib.aekv_prompt_attention_workspace_size(2, 10, 10, 4, 2, 128) == 0


def test_python_calls_refuse_cpu_tensors_and_wrong_arguments():
    from aetherkv import PolarQuant
    from aetherkv.paged import PagedKVCache, SlotTracker
    from aetherkv.prompt import prompt_attention

    pq = PolarQuant(4)
    with pytest.raises(ValueError):
        PagedKVCache(pq, 4, 2, 96, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(pq, 4, 2, 128, page_size=48, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(pq, 0, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        SlotTracker(1, 0, 16, device="cpu")
    codes, scale = torch.zeros(4, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="device"):
        PagedKVCache.from_tensors(pq, codes, scale, codes.clone(), scale.clone())
    with pytest.raises(RuntimeError, match="device"):
        SlotTracker.from_tensor(torch.zeros(2, 1, 2, 16, dtype=torch.int32))
    q, kv, cu = torch.zeros(8, 4, 128, dtype=torch.bfloat16), torch.zeros(8, 2, 128, dtype=torch.bfloat16), torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="device"):
        prompt_attention(q, kv, kv, cu, 0.1)
    with pytest.raises(RuntimeError):
        prompt_attention(q.float(), kv, kv, cu, 0.1)
    with pytest.raises(RuntimeError):
        prompt_attention(q, kv, kv[:7], cu, 0.1)


def test_where_slots_lie(tmp_path):
    """cache_row over good and bad tables: the row of a slot in the pool, -1 for slots outside the table and pages
    outside the pool, and offsets past 31 bits."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    src = tmp_path / "slot.cpp"
    src.write_text('#define __device__\n#define __forceinline__ inline\n#include "paged_slot.h"\n'
                   'extern "C" long long row(const int* table, int pages, int max_pages, int heads, int shift, long long b, int h, long long p) {\n'
                   '  aekv::PagePool c{nullptr, nullptr, nullptr, nullptr, table, pages, max_pages, heads, shift};\n'
                   '  return aekv::cache_row(c, b, h, p);\n}\n')
    so = tmp_path / "slot.so"
    subprocess.run([gxx, "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{PKG_DIR / 'csrc'}", str(src), "-o", str(so)], check=True)
    fn = ctypes.CDLL(str(so)).row
    fn.restype = ctypes.c_longlong
    fn.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4 + [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong]
    table = torch.tensor([[3, -1, 5, 7], [6, 100, 0, 0x7fffffff]], dtype=torch.int32)

    def row(b, h, p, pages=7, heads=2, shift=4, t=table):
        return fn(t.data_ptr(), pages, t.size(1), heads, shift, b, h, p)

    assert row(0, 1, 5) == (3 * 2 + 1) * 16 + 5
    assert row(1, 0, 15) == 6 * 2 * 16 + 15
    assert row(0, 0, 16) == -1 and row(1, 0, 16) == -1 and row(0, 0, 48) == -1 and row(1, 1, 63) == -1  # bad pages
    assert row(0, 0, -1) == -1 and row(0, 0, 64) == -1 and row(0, 0, 1 << 40) == -1
    big = torch.tensor([[0x7ffffffe]], dtype=torch.int32)
    assert row(0, 11, 4095, pages=0x7fffffff, heads=12, shift=12, t=big) == (0x7ffffffe * 12 + 11) * 4096 + 4095


def test_attention_workspace_holds_logits_for_few_rows_and_up_to_2_gib(lib):
    size = lambda B, T, slots, tracked: lib.aekv_paged_attention_workspace_size(B, T, 8, 2, 128, slots, tracked)  # noqa: E731
    lse = lambda B, T: 4 * B * T * 8  # noqa: E731
    # 64 sequences x 2 heads x 4 rows x 2^20 slots are 2 GiB, with 32 more slots beyond it
    assert size(64, 1, (1 << 20) - 32, 1) - size(64, 1, (1 << 20) - 32, 0) == lse(64, 1) + 64 * 2 * 4 * ((1 << 20) - 32) * 4
    assert size(64, 1, 1 << 20, 1) - size(64, 1, 1 << 20, 0) == lse(64, 1)
    assert size(1, 4, 1024, 1) - size(1, 4, 1024, 0) == lse(1, 4) + 2 * 16 * 1024 * 4
    assert size(1, 5, 1024, 1) - size(1, 5, 1024, 0) == lse(1, 5)  # 20 rows: scored again


def test_caches_and_trackers_are_on_a_device():
    """A cache in host memory would hand the kernels host pointers: it cannot be made."""
    from aetherkv import PolarQuant
    from aetherkv.paged import PagedKVCache, SlotTracker

    with pytest.raises(RuntimeError, match="device"):
        PagedKVCache(PolarQuant(4), 4, 2, 128, page_size=16, device="cpu")
    with pytest.raises(RuntimeError, match="device"):
        SlotTracker(1, 2, 64, device="cpu")


def test_workspace_sizes_of_refused_arguments():
    """Sizes are asked for before the call that refuses: whatever the arguments, an answer comes back (in a process of its own,
    as a division by zero would end it), and the Python calls raise."""
    from aetherkv.paged import paged_attention_workspace

    code = ("import itertools, random\nimport aetherkv._lib as L\nlib = L.lib()\n"
            "assert lib.aekv_paged_attention_workspace_size(1, 1, 2, 4, 128, 4096, 0) == 0\n"
            "assert lib.aekv_paged_attention_workspace_size(1, 1, 6, 4, 128, 4096, 1) == 0\n"
            "v = (-1, 0, 1, 2, 3, 7, 64, 65536, 2 ** 31, 2 ** 40)\nr = random.Random(0)\n"
            "for _ in range(20000):\n"
            "    a = [r.choice(v) for _ in range(6)]\n"
            "    d = r.choice((-1, 0, 64, 96, 128))\n"
            "    lib.aekv_paged_attention_workspace_size(*a[:4], d, a[4], r.randint(0, 1))\n"
            "    lib.aekv_kv_evict_workspace_size(*a[:4])\n"
            "    lib.aekv_prompt_attention_workspace_size(*a[:5], d)\n"
            "print('done')\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": str(PKG_DIR)})
    assert done.returncode == 0 and done.stdout.endswith("done\n"), (done.returncode, done.stderr[-500:])
    for H, heads in ((2, 4), (6, 4), (0, 2), (4, 0)):
        with pytest.raises(RuntimeError, match="multiple"):
            paged_attention_workspace(1, 1, H, heads, 128, 4096, "cpu")
