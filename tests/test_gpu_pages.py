"""The life of a pool's pages on the GPU against a model of lists (caches_ref.PoolRef), and the operators of a per-head cache
together as a serving loop uses them."""
from __future__ import annotations

import random

import pytest
import torch

import caches_ref as C
import paged_ref as R
from aetherkv import PolarQuant
from aetherkv.cache import rope_inv_freq
from aetherkv.cross import cross_attention
from aetherkv.paged import PagedKVCache, SlotTracker, append_tokens, evict_by_weight, paged_attention
from aetherkv.pages import PagePool
from aetherkv.prompt import prompt_attention
from aetherkv.rotary import AxisRotary, axis_sections, rotate_axes

pytestmark = pytest.mark.gpu


def _t(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Both:
    """The pool and its model side by side; every page's bytes are checked by where they came from."""

    def __init__(self, dev, pages, size, rows, width, layers=2, bits=4, heads=2, dim=64):
        self.dev, self.size = dev, size
        self.caches = [PagedKVCache(PolarQuant(bits), pages, heads, dim, page_size=size, device=dev) for _ in range(layers)]
        gen = torch.Generator(device=dev).manual_seed(pages)
        for c in self.caches:
            for t in c._tensors:
                t.copy_(torch.randint(0, 100, t.shape, device=dev, generator=gen))
        self.pool = PagePool(self.caches)
        self.model = C.PoolRef([0] * pages, size)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.rows = [[-1] * width for _ in range(rows)]
        self.bytes = [[t.cpu().clone() for t in c._tensors] for c in self.caches]

    def check(self):
        assert self.table.tolist() == self.rows
        assert self.pool.refs.tolist() == self.model.refs
        assert self.pool.lacking.item() == self.model.lacking
        assert int(self.pool.unused()) == sum(r <= 0 for r in self.model.refs)
        assert not self.pool._marks.any()
        for a, b in self.model.copies:
            for layer in self.bytes:
                for t in layer:
                    t[b] = t[a]
        self.model.copies.clear()
        for c, layer in zip(self.caches, self.bytes):
            for t, want in zip(c._tensors, layer):
                assert torch.equal(t.cpu(), want)

    def reserve(self, filled, wanted, first=None):
        self.pool.reserve(self.table, _t(filled, self.dev), _t(wanted, self.dev), first=None if first is None else _t(first, self.dev))
        self.model.reserve(self.rows, filled, wanted, first)
        self.check()

    def release(self, keep):
        self.pool.release(self.table, _t(keep, self.dev))
        self.model.release(self.rows, keep)
        self.check()

    def fork(self, filled, source, target):
        self.pool.fork(self.table, _t(filled, self.dev), _t(source, self.dev), _t(target, self.dev))
        self.model.fork(self.rows, filled, source, target)
        self.check()

    def compact(self):
        self.pool.compact(self.table)
        self.model.compact(self.rows)
        self.check()


@pytest.mark.parametrize("size,layers,bits,heads,dim", [(16, 1, 4, 1, 64), (64, 3, 8, 2, 128), (16, 2, 4, 3, 64), (512, 1, 8, 2, 128)])
def test_one_of_each(dev, size, layers, bits, heads, dim):
    b = Both(dev, 40, size, 5, 8, layers, bits, heads, dim)
    n = [3 * size + 1, size, 0, 5, 2 * size - 1]
    b.reserve([0] * 5, n)
    b.reserve(n, [x + 1 for x in n])
    n = [x + 1 for x in n]
    b.fork(n, [0, 0], [2, 1])  # two more answers to the first
    n = [n[0], n[0], n[0], n[3], n[4]]
    b.reserve(n, [x + 1 for x in n])  # the last of the three keeps the shared page
    n = [x + 1 for x in n]
    b.reserve(n, [x + size for x in n], first=[0] * 5)  # all pages their own, as before an eviction
    b.release([0, n[1], size, -3, 1 << 30])
    b.compact()
    b.release([0] * 5)
    b.compact()
    assert not b.pool.refs.any()


def test_beams_change_places(dev):
    b = Both(dev, 60, 16, 6, 9)
    n = [35] * 6
    b.reserve([0] * 6, n)
    for source in ([1, 0, 3, 2, 5, 4], [0, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5], [5, 5, 1, 1, 0, 0]):
        b.fork(n, source, list(range(6)))
        b.reserve(n, [x + 1 for x in n])
        n = [x + 1 for x in n]


def test_the_same_row_twice_and_rows_outside(dev):
    b = Both(dev, 30, 16, 4, 5)
    n = [40, 17, 16, 1]
    b.reserve([0] * 4, n)
    b.fork(n, [0, 1, 2], [3, 3, 3])  # the last counts
    b.fork(n, [3, 0, -1, 1, 4, 2 ** 31 - 1, 0], [3, 4, 1, -1, 0, 0, -2 ** 31])  # to itself; outside
    b.fork(n, [0, 3], [3, 3])  # the last says: stay
    b.fork(n, [], [])


def test_rows_that_write_nothing(dev):
    """A row without slots to write takes no page, and keeps what it shares, where the pool is out of pages too."""
    b = Both(dev, 4, 16, 3, 3)
    b.reserve([0] * 3, [40, 0, 0])
    b.fork([40, 0, 0], [0, 0], [1, 2])
    b.reserve([40] * 3, [40, 41, 40])  # one copy: the others write nothing
    assert b.rows == [[0, 1, 2], [0, 1, 3], [0, 1, 2]] and b.pool.lacking.item() == 0
    b.reserve([40, 41, 40], [40, 41, 39], first=[40, 47, 100])
    b.reserve([0, 0, 0], [0, 0, 0])
    assert b.rows == [[0, 1, 2], [0, 1, 3], [0, 1, 2]]


def test_more_than_the_pool_has(dev):
    b = Both(dev, 5, 16, 3, 4)
    b.reserve([0, 0, 0], [40, 40, 40])
    assert b.pool.lacking.item() == 4
    b.release([0, 16, 40])
    b.fork([0, 16, 0], [1], [0])
    b.reserve([16, 16, 0], [16 + 33, 17, 0], first=[0, 0, 0])
    b.release([0, 0, 0])
    b.compact()


def test_what_a_short_pool_loses_and_what_waits(dev):
    """A row that shares a filled page and gets none loses it, and a later reserve gives an empty page; rows that wait until the unused
    pages cover the call's entries lose nothing."""
    shared = [[0, 1, 2]] * 3
    b = Both(dev, 4, 16, 3, 3)
    b.reserve([0] * 3, [40, 0, 0])
    b.fork([40, 0, 0], [0, 0], [1, 2])
    assert b.rows == shared
    b.reserve([40] * 3, [41] * 3)  # three entries, one unused page: the last keeps the shared one, the second has none
    assert b.rows == [[0, 1, 3], [0, 1, -1], [0, 1, 2]] and b.pool.lacking.item() == 1 and b.pool.refs.tolist() == [3, 3, 1, 1]
    b.release([0, 40, 41])
    b.reserve([0, 40, 41], [0, 41, 42])
    assert b.rows == [[-1] * 3, [0, 1, 3], [0, 1, 2]] and not b.model.copies  # (no copy of page 2: its tokens are not there)

    b = Both(dev, 4, 16, 3, 3)
    b.reserve([0] * 3, [40, 0, 0])
    b.fork([40, 0, 0], [0, 0], [1, 2])
    assert int(b.pool.unused()) == 1  # covers one entry: the others wait
    b.reserve([40] * 3, [41, 40, 40])
    assert b.rows == [[0, 1, 3], [0, 1, 2], [0, 1, 2]]
    b.release([0, 40, 40])
    assert int(b.pool.unused()) == 1
    b.reserve([0, 40, 40], [0, 41, 40])
    assert b.rows == [[-1] * 3, [0, 1, 3], [0, 1, 2]] and b.pool.lacking.item() == 0
    b.release([0, 0, 40])
    b.reserve([0, 0, 40], [0, 0, 0], first=[0] * 3)  # before an eviction: wanted at or below first waits as well
    assert b.rows[2] == [0, 1, 2]


def test_entries_outside_the_pool_and_odd_counts(dev):
    b = Both(dev, 20, 16, 3, 6)
    b.reserve([0, 0, 0], [50, 20, 96])
    b.rows[0][1], b.rows[1][1], b.rows[1][3] = 20, 2 ** 31 - 1, -7  # (page 20 is the first outside)
    b.model.refs[b.table[0, 1].item()] -= 1
    b.model.refs[b.table[1, 1].item()] -= 1
    b.table.copy_(_t(b.rows, dev))
    b.pool.refs.copy_(_t(b.model.refs, dev))
    b.compact()
    b.fork([50, 20, 96], [0], [1])
    b.reserve([50, 50, 96], [1 << 30, 60, -5], first=[0, -100, 3])
    b.reserve([50, 50, 96], [60, 60, 1 << 30], first=[2 ** 31 - 1, 60, 96])
    b.release([-1, 17, 2 ** 31 - 1])


@pytest.mark.parametrize("seed", range(6))
def test_long_lives(dev, seed):
    """Many calls in turn, on a pool that runs short at times."""
    rng = random.Random(seed)
    size, rows, width = rng.choice([16, 32]), rng.choice([3, 17, 70]), rng.choice([4, 33])
    b = Both(dev, int(rows * width * rng.uniform(0.3, 1.1)) + 1, size, rows, width, layers=1, heads=1)
    n = [0] * rows
    for _ in range(12):
        kind = rng.choice(["grow", "grow", "step", "fork", "own", "release", "compact"])
        if kind in ("grow", "step", "own"):
            to = [min(width * size, x + (1 if kind == "step" else rng.randint(0, 3 * size) * (rng.random() < 0.5))) for x in n]
            b.reserve(n, to, first=[0] * rows if kind == "own" else None)
            n = to
        elif kind == "fork":
            k = rng.randint(1, rows)
            source, target = [rng.randrange(rows) for _ in range(k)], [rng.randrange(rows) for _ in range(k)]
            b.fork(n, source, target)
            old = list(n)
            for s, t in zip(source, target):
                n[t] = old[s]
        elif kind == "release":
            n = [rng.choice([0, x, rng.randint(0, x)]) for x in n]
            b.release(n)
        else:
            b.compact()


@pytest.mark.parametrize("pages,rows,width", [(5000, 1500, 3), (3000, 2, 1400), (40000, 64, 500), (1023, 33, 31), (1024, 32, 32), (1025, 1025, 1), (9000, 128, 32), (9000, 241, 17)])
def test_large_tables(dev, pages, rows, width):
    b = Both(dev, pages, 16, rows, width, layers=1, heads=1)
    rng = random.Random(pages)
    n = [rng.randint(0, width * 16) for _ in range(rows)]
    b.reserve([0] * rows, n)
    b.fork(n, [i // 2 for i in range(rows)], list(range(rows)))
    n = [n[i // 2] for i in range(rows)]
    b.reserve(n, [min(width * 16, x + 5) for x in n])
    b.reserve(n, n, first=[0] * rows)
    b.release([x if i % 3 else 0 for i, x in enumerate(n)])
    b.compact()


def test_every_entry_shares_its_page(dev):
    """All entries of a call share pages, up to and past the number that the kernel keeps: 64 rows over one prompt, in calls that
    write some of them or all."""
    for width in (1, 63, 64, 65):
        b = Both(dev, 64 * width + 70, 16, 64, width, layers=1, heads=1)
        n = [width * 16 - 3] + [0] * 63
        b.reserve([0] * 64, n)
        b.fork(n, [0] * 63, list(range(1, 64)))
        n = [n[0]] * 64
        b.reserve(n, [x + 2 if i % 3 else 0 for i, x in enumerate(n)])  # every third row writes nothing
        b.reserve(n, n, first=[0] * 64)


def test_many_tables_hold_one_pool(dev):
    b = Both(dev, 30, 16, 4, 4)
    kept = torch.full((2, 3), -1, dtype=torch.int32, device=dev)  # prefixes kept aside
    b.reserve([0] * 4, [60, 30, 10, 64])
    rows = [[-1] * 3 for _ in range(2)]
    b.pool.reserve(kept, _t([0, 0], dev), _t([48, 20], dev))
    b.model.reserve(rows, [0, 0], [48, 20])
    assert kept.tolist() == rows
    b.release([0, 30, 0, 64])
    b.pool.compact(b.table, kept)
    b.model.compact(b.rows, rows)
    assert kept.tolist() == rows
    b.check()


def test_captured_and_replayed(dev):
    """reserve, fork and release in one graph, replayed with other counts, eager calls between."""
    b = Both(dev, 64, 16, 4, 8)
    filled, wanted, keep, source, target = _t([0] * 4, dev), _t([20] * 4, dev), _t([200] * 4, dev), _t([0, 1], dev), _t([1, 0], dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def calls():
        b.pool.release(b.table, keep)
        b.pool.fork(b.table, filled, source, target)
        b.pool.reserve(b.table, filled, wanted)

    def model():
        b.model.release(b.rows, keep.tolist())
        b.model.fork(b.rows, filled.tolist(), source.tolist(), target.tolist())
        b.model.reserve(b.rows, filled.tolist(), wanted.tolist())

    with torch.cuda.stream(side):
        calls()
    side.synchronize()
    model()
    b.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        calls()
        with pytest.raises(RuntimeError, match="captured"):
            b.pool.unused()
    torch.cuda.synchronize()
    b.check()
    for step, (f, w, k, s) in enumerate([([20, 20, 20, 20], [33, 21, 20, 60], [20] * 4, [3, 0]), ([33, 21, 20, 60], [34] * 4, [33, 0, 20, 60], [1, 1]), ([34, 21, 30, 34], [40, 40, 128, 35], [34, 20, 10, 34], [2, 3])]):
        for t, x in ((filled, f), (wanted, w), (keep, k), (source, s)):
            t.copy_(_t(x, dev))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        model()
        b.check()
        if step == 1:
            b.compact()


def test_caches_of_several_forms_and_sizes(dev):
    """One pool over caches of other widths, heads and dims: every tensor's pages move alike."""
    caches = [PagedKVCache(PolarQuant(bits), 24, heads, dim, page_size=32, device=dev) for bits, heads, dim in ((4, 1, 64), (8, 3, 128), (8, 1, 64), (4, 5, 128))]
    gen = torch.Generator(device=dev).manual_seed(0)
    for c in caches:
        for t in c._tensors:
            t.copy_(torch.randint(1, 100, t.shape, device=dev, generator=gen))
    before = [t.clone() for c in caches for t in c._tensors]
    pool, table, n = PagePool(caches), torch.full((2, 4), -1, dtype=torch.int32, device=dev), _t([100, 0], dev)
    pool.reserve(table, _t([0, 0], dev), n)
    pool.fork(table, n, _t([0], dev), _t([1], dev))
    pool.reserve(table, _t([100, 100], dev), _t([100, 101], dev), first=_t([100, 0], dev))  # copies of all four pages
    assert table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]]
    for t, was in zip((t for c in caches for t in c._tensors), before):
        assert torch.equal(t[4:8], was[:4]) and torch.equal(t[:4], was[:4]) and torch.equal(t[8:], was[8:])
    pool.release(table, _t([0, 100], dev))
    pool.compact(table)
    assert table.tolist() == [[-1] * 4, [0, 1, 2, 3]]


def test_pages_past_32_bits(dev):
    """Tensors of 4.7 GB: copies from and to their last pages."""
    pages = 9000
    cache = PagedKVCache(PolarQuant(8), pages, 8, 128, page_size=512, device=dev)
    gen = torch.Generator(device=dev).manual_seed(0)
    some = [8999, 8998, 5]
    for t in cache._tensors:
        t[some] = torch.randint(-100, 100, t[some].shape, device=dev, generator=gen).to(t.dtype)
    before = [t[some].clone() for t in cache._tensors]
    refs = torch.ones(pages, dtype=torch.int32, device=dev)
    refs[[3, 4, 8997]] = 0
    pool = PagePool([cache], refs=refs)
    table = _t([some, [-1] * 3], dev)
    n = _t([3 * 512, 0], dev)
    pool.fork(table, n, _t([0], dev), _t([1], dev))
    assert pool.refs[some].tolist() == [2, 2, 2]
    pool.reserve(table, _t([3 * 512] * 2, dev), _t([0, 3 * 512], dev), first=_t([0, 0], dev))
    assert table.tolist() == [some, [3, 4, 8997]]
    for t, was in zip(cache._tensors, before):
        assert torch.equal(t[some], was) and torch.equal(t[[3, 4, 8997]], was)
    pool.release(table, _t([0, 3 * 512], dev))
    refs.zero_()
    refs[[3, 4, 8997]] = 1
    pool.compact(table)
    assert table.tolist() == [[-1] * 3, [0, 1, 2]] and refs[:3].tolist() == [1, 1, 1] and not refs[3:].any()
    for t, was in zip(cache._tensors, before):
        assert torch.equal(t[table[1].long()], was)


def test_two_pools_on_two_streams(dev):
    """Each stream has its own pool and workspace; calls of both lie between each other's."""
    both, streams = [Both(dev, 400, 16, 32, 10, layers=1, heads=1) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    n = [[0] * 32 for _ in range(2)]
    rng = random.Random(5)
    for _ in range(5):
        more = [[min(160, x + rng.randint(0, 20)) for x in row] for row in n]
        source = [[rng.randrange(32) for _ in range(6)] for _ in range(2)]
        args = [[_t(x, dev) for x in (n[i], more[i], source[i], list(range(6)))] for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both[i].pool.reserve(both[i].table, args[i][0], args[i][1])
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both[i].pool.fork(both[i].table, args[i][1], args[i][2], args[i][3])
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both[i].pool.compact(both[i].table)
        torch.cuda.synchronize()
        for i, b in enumerate(both):
            b.model.reserve(b.rows, n[i], more[i], None)
            b.model.fork(b.rows, more[i], source[i], list(range(6)))
            b.model.compact(b.rows)
            b.check()
            n[i] = [more[i][source[i][j]] if j < 6 else x for j, x in enumerate(more[i])]


def test_a_captured_compaction_of_several_tables(dev):
    b = Both(dev, 40, 16, 4, 4)
    kept, rows = torch.full((2, 3), -1, dtype=torch.int32, device=dev), [[-1] * 3 for _ in range(2)]
    want, side = _t([0, 0], dev), torch.cuda.Stream()
    b.pool.compact(b.table, kept)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.pool.compact(b.table, kept)
    torch.cuda.synchronize()
    b.check()
    for n, m, keep in (([60, 30, 10, 64], [48, 20], [0, 30, 0, 64]), ([64] * 4, [48, 48], [64, 0, 20, 3]), ([0] * 4, [0, 0], [0] * 4)):
        b.reserve([0] * 4, n)
        b.pool.reserve(kept, want, _t(m, dev))
        b.model.reserve(rows, [0, 0], m)
        b.release(keep)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        b.model.compact(b.rows, rows)
        assert kept.tolist() == rows
        b.check()


def test_serving_loop(dev):
    """Prompts with image positions, two answers each, attention over an encoder, an eviction, an end, a compaction: every
    answer's attention equals that of a sequence that never shared or moved a page."""
    H, hk, D, size, layers = 4, 2, 64, 16, 2
    gen = torch.Generator(device=dev).manual_seed(7)
    rotary = AxisRotary(rope_inv_freq(D, 10000.0, dev), axis_sections([8, 12, 12]), D)
    quant = PolarQuant(8)
    lens, budget, steps = [37, 20], 32, 14
    B, width = 4, 8
    caches = [PagedKVCache(quant, 80, hk, D, page_size=size, device=dev) for _ in range(layers)]
    alone = [PagedKVCache(quant, B * width, hk, D, page_size=size, device=dev) for _ in range(layers)]
    pool = PagePool(caches)
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    own = torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width)
    trackers = [[SlotTracker(B, hk, width * size, device=dev) for _ in range(layers)] for _ in range(2)]
    zero, n = torch.zeros(B, dtype=torch.int32, device=dev), _t([lens[0], 0, lens[1], 0], dev)
    cu = _t([0, lens[0], lens[0], sum(lens), sum(lens)], dev)
    # the prompts: rows 0 and 2, then forked to rows 1 and 3
    pool.reserve(table, zero, n)
    N = sum(lens)
    pos = torch.randint(0, 40, (3, N), device=dev, generator=gen)
    k_enc, v_enc = (torch.randn(90, hk, D, device=dev, generator=gen).bfloat16() for _ in range(2))
    cu_enc = _t([0, 50, 90], dev)
    for layer in range(layers):
        qkv = torch.randn(N, H + 2 * hk, D, device=dev, generator=gen).bfloat16()
        q, k = rotate_axes(qkv[:, :H], qkv[:, H:H + hk], pos, rotary, out_q=qkv[:, :H], out_k=qkv[:, H:H + hk])
        v = qkv[:, H + hk:]
        out = prompt_attention(q, k, v, cu, 0.125)
        want, bound, _, _ = R.prompt_attention_ref(q.cpu(), k.cpu(), v.cpu(), cu.tolist(), cu.tolist(), 0.125)
        R.within(out, want, bound, "prompt")
        out = cross_attention(q, k_enc, v_enc, cu_enc, 0.125, cu_seqlens=cu, states=_t([0, 0, 1, 1], dev))
        want, bound, _, _ = C.cross_attention_ref(q.cpu(), k_enc.cpu(), v_enc.cpu(), cu.tolist(), cu_enc.tolist(), [0, 0, 1, 1], 0.125)
        R.within(out, want, bound, "cross")
        append_tokens(caches[layer], k, v, table, zero, cu_seqlens=cu, tracker=trackers[0][layer], token=zero)
        # the sequences that share nothing: both answers hold the prompt
        twice = torch.cat([torch.arange(lens[0]), torch.arange(lens[0]), torch.arange(lens[0], N), torch.arange(lens[0], N)]).to(dev)
        append_tokens(alone[layer], k[twice], v[twice], own, zero, cu_seqlens=_t([0, lens[0], 2 * lens[0], 2 * lens[0] + lens[1], 2 * N], dev), tracker=trackers[1][layer], token=zero)
    pool.fork(table, n, _t([0, 2], dev), _t([1, 3], dev))
    for tr in trackers[0]:
        tr.storage[:, [1, 3]] = tr.storage[:, [0, 2]]
    n = _t([lens[0], lens[0], lens[1], lens[1]], dev)
    seen = n.clone()
    assert pool.refs.max() == 2
    active = list(range(B))
    for step in range(steps):
        pool.reserve(table, n, n + 1)
        pos = torch.randint(0, 60, (3, B), device=dev, generator=gen)
        for layer in range(layers):
            qkv = torch.randn(B, H + 2 * hk, D, device=dev, generator=gen).bfloat16()
            q, k = rotate_axes(qkv[:, :H], qkv[:, H:H + hk], pos, rotary)
            v = qkv[:, H + hk:]
            outs = []
            for cache, tab, tr in ((caches[layer], table, trackers[0][layer]), (alone[layer], own, trackers[1][layer])):
                append_tokens(cache, k[:, None], v[:, None], tab, n, tracker=tr, token=seen)
                outs.append(paged_attention(q[:, None], cache, tab, n + 1, 0.125, tracker=tr))
            assert torch.equal(outs[0][active], outs[1][active])
            out = cross_attention(q, k_enc, v_enc, cu_enc, 0.125, states=_t([0, 0, 1, 1], dev))
            want, bound, _, _ = C.cross_attention_ref(q.cpu(), k_enc.cpu(), v_enc.cpu(), list(range(B + 1)), cu_enc.tolist(), [0, 0, 1, 1], 0.125)
            R.within(out, want, bound, "cross")
        n, seen = n + 1, seen + 1
        if step == 5:  # the first two are past their budget: pages of their own, evict, give back
            pool.reserve(table, n, n, first=zero)
            assert pool.refs.max() == 1
            for layer in range(layers):
                for cache, tab, tr in ((caches[layer], table, trackers[0][layer]), (alone[layer], own, trackers[1][layer])):
                    evict_by_weight(cache, tab, n, tr, seen, budget, first=2, recent=8)
            n = n.clamp(max=budget)
            pool.release(table, n)
        if step == 8:  # the third ends; what is left moves together
            active.remove(2)
            n[2] = 0
            pool.release(table, n)
            pool.compact(table)
            used = int((pool.refs > 0).sum())
            assert not pool.refs[used:].any() and int(table.max()) < used
    assert pool.lacking.item() == 0


def test_refusals(dev):
    a, b = (PagedKVCache(PolarQuant(4), n, 2, 64, page_size=16, device=dev) for n in (8, 9))
    with pytest.raises(RuntimeError, match="same pages"):
        PagePool([a, b])
    none = PagedKVCache.from_tensors(PolarQuant(4), *(torch.empty((0, 2, 16, 32) if i % 2 == 0 else (0, 2, 16), dtype=torch.uint8 if i % 2 == 0 else torch.float32, device=dev) for i in range(4)))
    with pytest.raises(ValueError, match="pages"):
        PagePool([none])
    with pytest.raises(RuntimeError, match="refs"):
        PagePool([a], refs=torch.zeros(9, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="refs"):
        PagePool([a], refs=torch.zeros(8, dtype=torch.int32))
    pool, table, n = PagePool([a]), torch.full((3, 4), -1, dtype=torch.int32, device=dev), _t([0, 0, 0], dev)
    for bad in (table.long(), table.t(), table[0], table[:, :2]):
        for call in (lambda t: pool.reserve(t, n, n), lambda t: pool.release(t, n), lambda t: pool.fork(t, n, n, n), lambda t: pool.compact(t)):
            with pytest.raises(RuntimeError, match="page_table"):
                call(bad)
    for call in (lambda: pool.reserve(table, n[:2], n), lambda: pool.reserve(table, n, n.float()), lambda: pool.reserve(table, n, n, first=n[:1]), lambda: pool.release(table, n.cpu()),
                 lambda: pool.fork(table, n, n, n[:2]), lambda: pool.fork(table, n, n[None], n[None]), lambda: pool.compact(), lambda: pool.compact(table.cpu()),
                 lambda: pool.reserve(table, n, n, workspace=torch.empty(8, dtype=torch.uint8, device=dev))):
        with pytest.raises(RuntimeError):
            call()
