"""Rotary positions, attention over an encoder's states and a pool's pages: refusals of the C entries and of the Python calls,
and workspace sizes, checked on the CPU."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

import pytest
import torch

import aetherkv._lib as L
from conftest import PKG_DIR

FAKE, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001)


@pytest.fixture(scope="module")
def lib():
    if not L.available():
        pytest.fail("libaetherkv.so is not built (run __graft_entry__.build())")
    return L.lib()


def _cross(lib, q=FAKE, k=FAKE, v=FAKE, dtype=L.BF16, st=(512, 128, 256, 128, 256, 128), cq=FAKE, ck=FAKE, states=FAKE, B=2, E=3, nq=10, nk=10, H=4, hk=2, d=128, out=FAKE,
           ws=FAKE, wsb=1 << 30):
    return lib.aekv_cross_attention(q, k, v, dtype, *st, cq, ck, states, B, E, nq, nk, H, hk, d, None, 0.1, out, None, 0, ws, wsb, None)


def _rotate(lib, q=FAKE, k=FAKE, dtype=L.BF16, n=4, H=4, hk=2, d=128, st=(512, 128, 256, 128), pos=FAKE, pdt=L.I32, axes=3, freq=FAKE, axis=FAKE, pairs=64, first=0, halves=0, qo=FAKE,
            ko=FAKE, so=(512, 128, 256, 128)):
    return lib.aekv_rotate_axes(q, k, dtype, n, H, hk, d, *st, pos, pdt, axes, n, 1, freq, axis, pairs, first, halves, 0, qo, ko, *so, None)


def _reserve(lib, table=FAKE, B=3, W=4, filled=FAKE, wanted=FAKE, first=None, size=16, refs=FAKE, marks=FAKE, lacking=FAKE, pages=8, segs=FAKE, n=4, ws=FAKE, wsb=1 << 30):
    return lib.aekv_pool_reserve(table, B, W, filled, wanted, first, size, refs, marks, lacking, pages, segs, n, ws, wsb, None)


def _release(lib, table=FAKE, B=3, W=4, keep=FAKE, size=16, refs=FAKE, pages=8):
    return lib.aekv_pool_release(table, B, W, keep, size, refs, pages, None)


def _fork(lib, table=FAKE, B=3, W=4, filled=FAKE, source=FAKE, target=FAKE, n=2, size=16, refs=FAKE, pages=8, ws=FAKE, wsb=1 << 30):
    return lib.aekv_pool_fork(table, B, W, filled, source, target, n, size, refs, pages, ws, wsb, None)


def _compact(lib, table=FAKE, entries=12, refs=FAKE, pages=8, segs=FAKE, n=4, ws=FAKE, wsb=1 << 30):
    return lib.aekv_pool_compact(table, entries, refs, pages, segs, n, ws, wsb, None)


def test_cross_refusals(lib):
    assert _cross(lib, dtype=L.F32) == L.ERR_DTYPE
    assert _cross(lib, d=256) == L.ERR_UNSUPPORTED
    assert _cross(lib, H=3) == L.ERR_SHAPE and _cross(lib, hk=0) == L.ERR_SHAPE and _cross(lib, E=-1) == L.ERR_SHAPE
    assert _cross(lib, B=0) == L.ERR_SHAPE
    assert _cross(lib, cq=None) == L.ERR_SHAPE and "one query" in lib.aekv_last_error().decode()
    assert _cross(lib, states=None) == L.ERR_SHAPE and "list" in lib.aekv_last_error().decode()
    assert _cross(lib, k=None) == L.ERR_VALUE and _cross(lib, ck=None) == L.ERR_VALUE and _cross(lib, out=None) == L.ERR_VALUE
    assert _cross(lib, v=ODD) == L.ERR_ALIGN and _cross(lib, st=(512, 128, 252, 128, 256, 128)) == L.ERR_ALIGN
    assert _cross(lib, st=(512, 128, -256, 128, 256, 128)) == L.ERR_UNSUPPORTED and _cross(lib, st=(512, 128, 1 << 30, 128, 256, 128)) == L.ERR_UNSUPPORTED
    assert _cross(lib, nq=1 << 31) == L.ERR_UNSUPPORTED and _cross(lib, nk=1 << 31) == L.ERR_UNSUPPORTED and _cross(lib, H=1 << 17, hk=1) == L.ERR_UNSUPPORTED
    assert _cross(lib, nq=0) == L.OK
    for nq, nk in ((10, 1000), (1000, 100000)):
        need = lib.aekv_cross_attention_workspace_size(2, 3, nq, nk, 4, 2, 128)
        assert need > 0 and _cross(lib, nq=nq, nk=nk, wsb=need - 1) == L.ERR_WORKSPACE and _cross(lib, nq=nq, nk=nk, ws=None) == L.ERR_WORKSPACE
        assert _cross(lib, nq=nq, nk=nk, ws=ctypes.c_void_p(0x10008)) == L.ERR_ALIGN


def test_cross_partial_rows_are_aligned(lib):
    """The workspace holds a descriptor per workgroup and behind them partial rows of 16-byte vectors, each (d + 4) fp32: the size
    is whole 16 bytes for every number of workgroups only if the rows begin on 16 bytes."""
    for d in (64, 128):
        for B, E in ((1, 1), (2, 3), (7, 7), (64, 8), (300, 300)):
            for nq in (B, 3 * B, 200 * B):
                for H, hk in ((1, 1), (12, 4), (16, 16), (10, 2)):
                    for nk in (0, 1, 128, 300, 700, 1500, 9001):
                        assert lib.aekv_cross_attention_workspace_size(B, E, nq, nk, H, hk, d) % 16 == 0, (B, E, nq, nk, H, hk, d)


def test_cross_rows_that_overlap_are_refused(lib):
    for st in ((512, 128, 120, 128, 256, 128), (512, 128, 256, 128, 0, 128)):
        assert _cross(lib, nk=2, st=st, ws=None) == L.ERR_UNSUPPORTED and "strides" in lib.aekv_last_error().decode()


def test_cross_strides_that_no_second_row_needs(lib):
    """One row of keys has no token stride: whatever stands there, the call goes on to its next check."""
    for st in ((512, 128, 1 << 30, 128, 1 << 30, 128), (512, 128, -256, 128, 256, 128)):
        assert _cross(lib, nk=2, st=st, ws=None) == L.ERR_UNSUPPORTED
        assert _cross(lib, nk=1, st=st, ws=None) == L.ERR_WORKSPACE and _cross(lib, nk=0, st=st, ws=None) == L.ERR_WORKSPACE


def test_rotate_refusals(lib):
    assert _rotate(lib, dtype=L.I32) == L.ERR_DTYPE and _rotate(lib, pdt=L.F32) == L.ERR_DTYPE
    assert _rotate(lib, n=-1) == L.ERR_SHAPE and _rotate(lib, H=0, hk=0) == L.ERR_SHAPE and _rotate(lib, H=-1) == L.ERR_SHAPE and _rotate(lib, axes=0) == L.ERR_SHAPE
    assert _rotate(lib, H=65535, hk=1) == L.ERR_SHAPE
    assert _rotate(lib, d=127) == L.ERR_UNSUPPORTED and _rotate(lib, d=0) == L.ERR_UNSUPPORTED and _rotate(lib, d=1026) == L.ERR_UNSUPPORTED
    assert _rotate(lib, pairs=0) == L.ERR_VALUE and _rotate(lib, pairs=65) == L.ERR_VALUE and _rotate(lib, first=2) == L.ERR_VALUE
    assert _rotate(lib, pairs=3, first=1) == L.ERR_VALUE and _rotate(lib, pairs=3, halves=1) == L.ERR_VALUE and _rotate(lib, first=-2, pairs=4) == L.ERR_VALUE
    assert _rotate(lib, q=ODD) == L.ERR_ALIGN and _rotate(lib, ko=ctypes.c_void_p(0x10002)) == L.ERR_ALIGN and _rotate(lib, st=(511, 128, 256, 128)) == L.ERR_ALIGN
    assert _rotate(lib, pos=None) == L.ERR_VALUE and _rotate(lib, axis=None) == L.ERR_VALUE and _rotate(lib, qo=None) == L.ERR_VALUE and _rotate(lib, k=None) == L.ERR_VALUE
    assert _rotate(lib, n=0, q=None) == L.OK


def test_pool_refusals(lib):
    for call in (_reserve, _release, _fork):
        for size in (0, 8, 24, 8192, -16):
            assert call(lib, size=size) == L.ERR_VALUE
        assert call(lib, B=-1) == L.ERR_SHAPE and call(lib, W=-1) == L.ERR_SHAPE and call(lib, pages=-1) == L.ERR_SHAPE
        assert call(lib, B=4097) == L.ERR_UNSUPPORTED and call(lib, W=1 << 29) == L.ERR_UNSUPPORTED and call(lib, pages=1 << 30) == L.ERR_UNSUPPORTED
        assert call(lib, table=None) == L.ERR_VALUE and call(lib, refs=None) == L.ERR_VALUE
        assert call(lib, B=0, table=None) == L.OK and call(lib, W=0, table=None) == L.OK
    for name in ("filled", "wanted", "marks", "lacking"):
        assert _reserve(lib, **{name: None}) == L.ERR_VALUE
    assert _reserve(lib, segs=None) == L.ERR_VALUE and _reserve(lib, segs=ODD) == L.ERR_VALUE and _reserve(lib, n=-1) == L.ERR_SHAPE
    assert _release(lib, keep=None) == L.ERR_VALUE
    assert _fork(lib, source=None) == L.ERR_VALUE and _fork(lib, n=-1) == L.ERR_SHAPE and _fork(lib, n=0, source=None) == L.OK and _fork(lib, n=1 << 30) == L.ERR_SHAPE
    assert _compact(lib, pages=-1) == L.ERR_SHAPE and _compact(lib, entries=-1) == L.ERR_SHAPE and _compact(lib, table=None) == L.ERR_VALUE and _compact(lib, refs=None) == L.ERR_VALUE and _compact(lib, segs=None) == L.ERR_VALUE
    size = lib.aekv_pool_workspace_size
    for call, need in ((_reserve, size(3, 4, 0, 0)), (_fork, size(0, 4, 2, 0)), (_compact, size(0, 0, 0, 8))):
        assert need > 0 and call(lib, wsb=need - 1) == L.ERR_WORKSPACE and call(lib, ws=None) == L.ERR_WORKSPACE and call(lib, ws=ctypes.c_void_p(0x10008)) == L.ERR_ALIGN
    assert lib.aekv_pool_renumber(FAKE, 4, 8, FAKE, size(0, 0, 0, 8) - 1, None) == L.ERR_WORKSPACE
    assert lib.aekv_pool_renumber(None, 4, 8, FAKE, 1 << 20, None) == L.ERR_VALUE and lib.aekv_pool_renumber(None, 0, 8, FAKE, 1 << 20, None) == L.OK


def test_workspace_sizes_of_refused_arguments():
    """Sizes are asked for before the call that refuses: whatever the arguments, an answer comes back (in a process of its own, as
    a division by zero would end it)."""
    code = ("import random\nimport aetherkv._lib as L\nlib = L.lib()\n"
            "v = (-1, 0, 1, 2, 3, 7, 64, 65536, 2 ** 31, 2 ** 40)\nr = random.Random(0)\n"
            "for _ in range(30000):\n"
            "    a = [r.choice(v) for _ in range(6)]\n"
            "    lib.aekv_cross_attention_workspace_size(*a, r.choice((-1, 0, 64, 96, 128)))\n"
            "    lib.aekv_pool_workspace_size(*a[:4])\n"
            "print('done')\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": str(PKG_DIR)})
    assert done.returncode == 0 and done.stdout.endswith("done\n"), (done.returncode, done.stderr[-500:])


def test_axis_sections():
    from aetherkv.rotary import axis_sections

    assert axis_sections([2, 1, 3]) == [0, 0, 1, 2, 2, 2]
    assert axis_sections([2, 1, 3], interleaved=True) == [0, 1, 2, 0, 2, 2]
    assert axis_sections([4]) == [0] * 4
    for bad in ([], [0, 0], [2, -1]):
        with pytest.raises(ValueError):
            axis_sections(bad)


def test_python_calls_refuse_cpu_tensors_and_wrong_arguments():
    from aetherkv.cross import cross_attention
    from aetherkv.pages import PagePool
    from aetherkv.rotary import AxisRotary

    with pytest.raises(RuntimeError, match="device"):
        AxisRotary(torch.ones(64), [0] * 64, 128)
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 2, 4, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="device"):
        cross_attention(q, k, k, cu, 0.1)
    with pytest.raises(RuntimeError, match="alike"):
        cross_attention(q, k.half(), k, cu, 0.1)
    with pytest.raises(RuntimeError, match="multiple"):
        cross_attention(q[:, :3], k, k, cu, 0.1)
    with pytest.raises(RuntimeError, match="cu_seqlens_k"):
        cross_attention(q, k, k, cu[None], 0.1)
    with pytest.raises(RuntimeError, match="cu_seqlens must"):
        cross_attention(q, k, k, cu, 0.1, cu_seqlens=cu[:1])
    with pytest.raises(ValueError):
        PagePool([])
