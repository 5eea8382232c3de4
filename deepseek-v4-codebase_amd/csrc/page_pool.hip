// The life of a cache's pages: which are in use (refs[p]: entries of page tables that hold page p), given to sequences,
// shared by forks, copied before they are written, released, moved together.  One pool serves the caches of all layers, whose
// tables are one: a page's bytes lie in several tensors.
//
//   reserve  every table entry of the slots that are about to be written gets a page of its own: a fresh one where it has none,
//            and a fresh copy where it shares one with entries that the call does not write (the last of a page's holders, if
//            the call writes them all, keeps it).  Fresh pages are the lowest unused ones, in the entries' order.
//   release  entries past the kept slots let go of their pages.
//   fork     rows take over other rows' pages, all read before any is written.
//   compact  the k-th unused page below the number of pages in use takes the k-th page in use from there on.
//
// Tables and counts are device data: entries outside the pool count as none, rows outside the table are skipped.  What decides is
// a few thousand whole numbers, which one workgroup reads in some memory rounds: bound by latency.  (Unused pages are looked for
// from the lowest on, 4096 counts to a round, and a compaction reads 1024: in a pool of 200000 pages that are in use 64 rows'
// reserve takes 68 us, and a compaction 172.)  What moves is a page's bytes in every tensor, by a second launch that reads the
// number of copies from memory.
#include "aekv_common.h"

namespace aekv {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxRows = 4096;    // rows of a table (what is known of them lies in LDS)
constexpr int kOwn = 4;           // entries that a thread keeps in registers
constexpr int kSlots = 2 * kOwn * kThreads;  // of the shared pages' table
constexpr int kSegment = 4096;    // bytes that a wave copies at a time
constexpr int kHeader = 16;       // ints before the lists in the workspace: copies

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

struct Segment {
  uint64_t base;  // of a page's part in one tensor, page 0
  uint64_t page;  // bytes from a page to the next
  uint64_t bytes; // at most kSegment, a multiple of 16
};

struct PoolArgs {
  int32_t* table;  // [B, W]
  int32_t B, W, shift;
  const int32_t* filled;
  const int32_t* wanted;
  const int32_t* first;
  int32_t* refs;     // [pages]
  int32_t* marks;    // [2, pages]: writers of a shared page, the last of them + 1; 0 between calls
  int32_t* lacking;  // [1]: pages that could not be given
  int32_t pages;
  int32_t* ws;
};

__device__ __forceinline__ int32_t load_now(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void add(int32_t* p, int32_t v) { __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Sums over the threads before this one, and over all: of any v, or of v < 8 from its bits.  s: 2 kWaves ints, of which the calls
// take one half in turn, so that one barrier to a call is enough.
struct Scan {
  int32_t* s;
  int turn;
  __device__ __forceinline__ int32_t join(int32_t before, int32_t wave_sum, int32_t* total) {
    int32_t* const w = s + kWaves * turn;
    turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) w[wave] = wave_sum;
    __syncthreads();
    int32_t all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const int32_t n = w[i];
      before += i < wave ? n : 0;
      all += n;
    }
    *total = all;
    return before;
  }
  __device__ __forceinline__ int32_t any(int32_t v, int32_t* total) {
    const int lane = threadIdx.x & 63;
    int32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t o = __shfl_up(x, d);
      if (lane >= d) x += o;
    }
    return join(x - v, x, total);
  }
  template <int kBits>
  __device__ __forceinline__ int32_t small(int32_t v, int32_t* total) {
    const uint64_t below = (1ull << (threadIdx.x & 63)) - 1;
    int32_t before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kBits; ++i) {
      const uint64_t with = __builtin_amdgcn_ballot_w64(v >> i & 1);
      before += __popcll(with & below) << i, sum += __popcll(with) << i;
    }
    return join(before, sum, total);
  }
};

// The counts of pages p0 + 4 tid .., 1 (not unused) for those past the last.
__device__ __forceinline__ int4 load_refs(const PoolArgs& a, int32_t p0) {
  const int32_t p = p0 + 4 * static_cast<int32_t>(threadIdx.x);
  int4 r = make_int4(1, 1, 1, 1);
  if (p < a.pages) r.x = a.refs[p];
  if (p + 1 < a.pages) r.y = a.refs[p + 1];
  if (p + 2 < a.pages) r.z = a.refs[p + 2];
  if (p + 3 < a.pages) r.w = a.refs[p + 3];
  return r;
}

// Pages that slots [0, n) lie in, as far as the table has them.
__device__ __forceinline__ int32_t pages_of(const PoolArgs& a, int32_t n) {
  const int32_t p = n <= 0 ? 0 : ((n - 1) >> a.shift) + 1;
  return p < a.W ? p : a.W;
}

struct Rows {
  int32_t offs[kMaxRows + 1];  // where a row's entries start among the call's
  int32_t from[kMaxRows];      // its first entry
  int32_t filled[kMaxRows];
};
struct Entry {
  int32_t row, i, p, r;  // table[row, i] = p, which has r holders; r = -1: no page
};

// The call's shared pages, where its entries are kept: a table by page, open to the next slot.
// (Aligned as it is cleared, four slots to a store.)
struct alignas(16) Shared {
  int32_t page[kSlots], count[kSlots], last[kSlots];  // -1: free; the page's entries in the call, and the last of them
};

// The call's `entries` entries.  kKept: they are at most kOwn to a thread, which reads them once; else every pass reads them.  (A step
// of 64 sequences: 6.2 us, 11.6 with every pass reading.)
template <bool kKept>
__device__ __forceinline__ void reserve_entries(const PoolArgs& a, const Rows& s, int32_t entries, Scan& scan, Shared& sh, int32_t* s_copies, const int4& refs0) {
  const int tid = threadIdx.x;
  auto place = [&](int32_t e, Entry* x) {
    int32_t lo = 0, hi = a.B;  // offs[lo] <= e < offs[hi]
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (s.offs[mid] <= e) lo = mid;
      else hi = mid;
    }
    x->row = lo, x->i = s.from[lo] + e - s.offs[lo];
  };
  auto look = [&](Entry* x) {
    x->p = a.table[static_cast<int64_t>(x->row) * a.W + x->i];
    const bool has = x->p >= 0 && x->p < a.pages;
    const int32_t r = a.pages > 0 ? a.refs[has ? x->p : 0] : 0;
    x->r = has ? max(r, 0) : -1;
  };
  Entry own[kOwn];
  if constexpr (kKept) {
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      own[j].r = 0;
      if (tid + j * kThreads < entries) place(tid + j * kThreads, &own[j]);
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (tid + j * kThreads < entries) look(&own[j]);
  }
  auto each = [&](auto f) __attribute__((always_inline)) {  // f(e, entry, place among the thread's)
    if constexpr (kKept) {
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
        if (j * kThreads < entries) f(tid + j * kThreads, own[j], j);
    } else {
      for (int32_t e0 = 0; e0 < entries; e0 += kThreads) {
        Entry x{0, 0, 0, 0};
        if (e0 + tid < entries) place(e0 + tid, &x), look(&x);
        f(e0 + tid, x, 0);
      }
    }
  };
  // a shared page's entries in the call: how many, and which is the last
  int32_t slot_of[kOwn];
  each([&](int32_t e, const Entry& x, int j) {
    if (e >= entries || x.r <= 1) return;
    if constexpr (kKept) {
      uint32_t h = static_cast<uint32_t>(x.p) * 2654435761u >> 19;
      for (;;) {  // (at most half of the slots are taken)
        const int32_t was = atomicCAS(sh.page + h, -1, x.p);
        if (was == -1 || was == x.p) break;
        h = (h + 1) % kSlots;
      }
      atomicAdd(sh.count + h, 1);
      atomicMax(sh.last + h, e);
      slot_of[j] = static_cast<int32_t>(h);
    } else {
      add(a.marks + x.p, 1);
      __hip_atomic_fetch_max(a.marks + a.pages + x.p, e + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  });
  if constexpr (!kKept) __threadfence();
  __syncthreads();
  auto keeps = [&](int32_t e, const Entry& x, int j) {  // the last of all the page's holders
    if constexpr (kKept) return sh.count[slot_of[j]] == x.r && sh.last[slot_of[j]] == e;
    else return load_now(a.marks + x.p) == x.r && load_now(a.marks + a.pages + x.p) == e + 1;
  };
  int32_t* const rank_of = a.ws + kHeader;                           // [entries]: the entry's number among those that take a page, or -1
  int32_t* const fresh = kKept ? sh.page : rank_of + static_cast<int64_t>(a.B) * a.W;  // [entries] (kept: the table has been read)
  int32_t* const copies = rank_of + 2 * static_cast<int64_t>(a.B) * a.W;  // [entries][2]
  int32_t takes = 0, ranks[kOwn];
  each([&](int32_t e, const Entry& x, int j) {
    bool take = e < entries && x.r < 0;
    if (e < entries && x.r > 1) take = !keeps(e, x, j);
    int32_t all;
    const int32_t rank = takes + scan.small<1>(take, &all);
    if constexpr (kKept) ranks[j] = take ? rank : -1;
    else if (e < entries) rank_of[e] = take ? rank : -1;
    takes += all;
  });
  __syncthreads();
  int32_t found = 0;  // the lowest unused pages, four to a thread
  for (int32_t p0 = 0; p0 < a.pages && found < takes; p0 += 4 * kThreads) {
    int4 r = refs0;
    if (p0) r = load_refs(a, p0);
    const bool u0 = r.x <= 0, u1 = r.y <= 0, u2 = r.z <= 0, u3 = r.w <= 0;
    int32_t all;
    int32_t at = found + scan.small<3>(u0 + u1 + u2 + u3, &all);
    const int32_t p = p0 + 4 * tid;
    if (u0 && at < takes) fresh[at] = p;
    at += u0;
    if (u1 && at < takes) fresh[at] = p + 1;
    at += u1;
    if (u2 && at < takes) fresh[at] = p + 2;
    at += u2;
    if (u3 && at < takes) fresh[at] = p + 3;
    found += all;
  }
  __syncthreads();
  each([&](int32_t e, const Entry& x, int j) {
    if (e >= entries) return;
    // (read again, r may have sunk: others of the page's entries let go of it meanwhile)
    if (!kKept && x.r >= 0) a.marks[x.p] = 0, a.marks[a.pages + x.p] = 0;
    const int32_t rank = kKept ? ranks[j] : rank_of[e];
    if (rank < 0) return;
    const int32_t to = rank < found ? fresh[rank] : -1;
    a.table[static_cast<int64_t>(x.row) * a.W + x.i] = to;
    if (x.r >= 0) add(a.refs + x.p, -1);
    if (to < 0) return;
    a.refs[to] = 1;
    if (x.r >= 0 && (static_cast<int64_t>(x.i) << a.shift) < s.filled[x.row]) {
      const int32_t c = atomicAdd(s_copies, 1);
      copies[2 * c] = x.p, copies[2 * c + 1] = to;
    }
  });
  __syncthreads();
  if (tid == 0) {
    a.ws[0] = *s_copies;
    if (found < takes) *a.lacking += takes - found;
  }
}

__global__ __launch_bounds__(kThreads) void pool_reserve_kernel(PoolArgs a) {
  __shared__ Rows s;
  __shared__ Shared sh;
  __shared__ int32_t s_scan[2 * kWaves];
  __shared__ int32_t s_copies;
  static_assert(alignof(Shared) >= sizeof(int4) && kSlots % 4 == 0, "its arrays are cleared by int4");
  static_assert(kSlots == 1 << 13 && (kSlots / 4) % kThreads == 0, "the hash's bits; whole rounds of four slots");
  Scan scan{s_scan, 0};
  const int tid = threadIdx.x;
  if (tid == 0) s_copies = 0;
  const int4 refs0 = load_refs(a, 0);  // (here, so that it arrives with the rows' counts)
#pragma unroll
  for (int i = 0; i < kSlots / 4 / kThreads; ++i) {
    const int at = 4 * (i * kThreads + tid);
    *reinterpret_cast<int4*>(sh.page + at) = *reinterpret_cast<int4*>(sh.last + at) = make_int4(-1, -1, -1, -1);
    *reinterpret_cast<int4*>(sh.count + at) = make_int4(0, 0, 0, 0);
  }
  int32_t entries = 0;
  for (int32_t b0 = 0; b0 < a.B; b0 += kThreads) {
    const int32_t b = b0 + tid;
    int32_t n = 0, from = 0, filled = 0;
    if (b < a.B) {
      const int32_t w = a.wanted[b];
      filled = a.filled[b];
      const int32_t f = max(a.first ? a.first[b] : filled, 0);
      from = f >> a.shift;
      n = w > f ? max(pages_of(a, w) - from, 0) : 0;  // (no slots: no pages, within a page too)
    }
    int32_t all;
    const int32_t before = scan.any(n, &all);
    if (b < a.B) s.offs[b] = entries + before, s.from[b] = from, s.filled[b] = filled;
    entries += all;  // (at most B W, which fits 30 bits)
  }
  if (tid == 0) s.offs[a.B] = entries;
  __syncthreads();
  if (entries <= kOwn * kThreads) reserve_entries<true>(a, s, entries, scan, sh, &s_copies, refs0);
  else reserve_entries<false>(a, s, entries, scan, sh, &s_copies, refs0);
}

__global__ __launch_bounds__(256) void pool_release_kernel(PoolArgs a) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<int64_t>(a.B) * a.W) return;
  const int32_t row = static_cast<int32_t>(at / a.W), i = static_cast<int32_t>(at - static_cast<int64_t>(row) * a.W);
  if (i < pages_of(a, a.wanted[row])) return;
  const int32_t p = a.table[at];
  if (p >= 0 && p < a.pages) add(a.refs + p, -1);
  if (p != -1) a.table[at] = -1;
}

// A workgroup has kColumns columns of the table, so that it reads all rows' old entries before it writes any.
constexpr int kColumns = 16;
__global__ __launch_bounds__(256) void pool_fork_kernel(PoolArgs a, const int32_t* source, const int32_t* target, int32_t n) {
  extern __shared__ int32_t owner[];  // [B]: the last fork to a row + 1
  for (int32_t b = threadIdx.x; b < a.B; b += 256) owner[b] = 0;
  __syncthreads();
  for (int32_t j = threadIdx.x; j < n; j += 256) {
    const int32_t s = source[j], t = target[j];
    if (s >= 0 && s < a.B && t >= 0 && t < a.B) atomicMax(owner + t, j + 1);
  }
  const int32_t i = blockIdx.x * kColumns + threadIdx.x % kColumns;
  int32_t* const old = a.ws + kHeader;
  const bool in = i < a.W;
  for (int32_t j = threadIdx.x / kColumns; in && j < n; j += 256 / kColumns) {
    const int32_t s = source[j];
    if (s < 0 || s >= a.B) continue;
    old[static_cast<int64_t>(j) * a.W + i] = i < pages_of(a, a.filled[s]) ? a.table[static_cast<int64_t>(s) * a.W + i] : -1;
  }
  __syncthreads();
  for (int32_t j = threadIdx.x / kColumns; in && j < n; j += 256 / kColumns) {
    const int32_t s = source[j], t = target[j];
    if (s < 0 || s >= a.B || t < 0 || t >= a.B || s == t || owner[t] != j + 1) continue;
    int32_t* const entry = a.table + static_cast<int64_t>(t) * a.W + i;
    const int32_t was = *entry, now = old[static_cast<int64_t>(j) * a.W + i];
    if (was == now) continue;
    if (was >= 0 && was < a.pages) add(a.refs + was, -1);
    if (now >= 0 && now < a.pages) add(a.refs + now, 1);
    *entry = now;
  }
}

__global__ __launch_bounds__(kThreads) void pool_compact_kernel(PoolArgs a) {
  __shared__ int32_t s_scan[2 * kWaves];
  Scan scan{s_scan, 0};
  const int tid = threadIdx.x;
  int32_t* const to = a.ws + kHeader;  // [pages]: where a page from `live` on goes, or -1
  int32_t* const moves = to + a.pages; // [moves][2]
  int32_t mine = 0, live;
  for (int32_t p = tid; p < a.pages; p += kThreads) mine += a.refs[p] > 0;
  scan.any(mine, &live);
  int32_t holes = 0, movers = 0;
  for (int32_t p0 = 0; p0 < a.pages; p0 += kThreads) {
    const int32_t p = p0 + tid;
    const bool used = p < a.pages && a.refs[p] > 0;
    const bool hole = p < live && !used, mover = p >= live && used;
    int32_t all;
    const int32_t before = scan.any((hole ? 1 : 0) + (mover ? 1 << 16 : 0), &all);
    if (hole) moves[2 * (holes + (before & 0xFFFF)) + 1] = p;
    if (mover) moves[2 * (movers + (before >> 16))] = p;
    if (p >= live && p < a.pages && !used) to[p] = -1;
    holes += all & 0xFFFF, movers += all >> 16;
  }
  __syncthreads();
  for (int32_t k = tid; k < holes; k += kThreads) {  // (as many movers)
    const int32_t p = moves[2 * k], q = moves[2 * k + 1];
    to[p] = q;
    a.refs[q] = a.refs[p];
    a.refs[p] = 0;
  }
  if (tid == 0) a.ws[0] = holes, a.ws[1] = live;
}

// Entries of a table after a compaction.
__device__ __forceinline__ void renumber(int32_t* table, int64_t at, int32_t pages, const int32_t* ws) {
  const int32_t p = table[at];
  if (p >= ws[1] && p < pages) table[at] = ws[kHeader + p];
}
__global__ __launch_bounds__(256) void pool_renumber_kernel(int32_t* table, int64_t n, int32_t pages, const int32_t* ws) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at < n) renumber(table, at, pages, ws);
}

// Copies of pages: a wave takes a segment of one copy at a time.  Written past the caches, where the reads of what lies far apart
// have the room (513 of 1218 pages, 28 layers of 35 KB: 107 us, 5.5 TB/s; with plain stores 123).  With a table: a compaction's,
// whose entries are renumbered by the way.
__global__ __launch_bounds__(256) void pool_copy_kernel(const int32_t* ws, const int32_t* copies, const Segment* segs, int32_t n_segs, int32_t* table, int64_t entries, int32_t pages) {
  const int32_t* const count = ws;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < entries; at += static_cast<int64_t>(gridDim.x) * 256) renumber(table, at, pages, ws);
  const int lane = threadIdx.x & 63;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t items = static_cast<int64_t>(*count) * n_segs;
  for (int64_t it = wave; it < items; it += static_cast<int64_t>(gridDim.x) * 4) {
    const int32_t c = static_cast<int32_t>(it / n_segs), s = static_cast<int32_t>(it - static_cast<int64_t>(c) * n_segs);
    const Segment g = segs[s];
    const uint64_t src = g.base + g.page * static_cast<uint32_t>(copies[2 * c]), dst = g.base + g.page * static_cast<uint32_t>(copies[2 * c + 1]);
    u32x4_t w[kSegment / 1024];
#pragma unroll
    for (int i = 0; i < kSegment / 1024; ++i) {
      const uint32_t at = 1024 * i + 16 * lane;
      w[i] = at < g.bytes ? *reinterpret_cast<const u32x4_t*>(src + at) : u32x4_t{};
    }
#pragma unroll
    for (int i = 0; i < kSegment / 1024; ++i) {
      const uint32_t at = 1024 * i + 16 * lane;
      if (at < g.bytes) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4_t*>(dst + at));
    }
  }
}

int check_table(const char* who, const int32_t* table, int64_t B, int64_t W, int64_t pages, const int32_t* refs) {
  if (B < 0 || W < 0 || pages < 0) return fail(AEKV_ERR_SHAPE, "%s: B=%lld max_pages=%lld pages=%lld", who, (long long)B, (long long)W, (long long)pages);
  if (B > kMaxRows) return fail(AEKV_ERR_UNSUPPORTED, "%s: a table of %lld rows (%d supported)", who, (long long)B, kMaxRows);
  if (W > 0x7fffffff || B * W > 0x3fffffff || pages > 0x3fffffff)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld max_pages=%lld pages=%lld exceed 30 bits", who, (long long)B, (long long)W, (long long)pages);
  if (B * W > 0 && (!table || !refs)) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  return AEKV_OK;
}
int page_shift(int32_t page_size) { return is_pow2(page_size) && page_size >= 16 && page_size <= 4096 ? __builtin_ctz(page_size) : -1; }

int check_segments(const char* who, const void* segs, int64_t n) {
  if (n < 0 || n > 0x7fffffff) return fail(AEKV_ERR_SHAPE, "%s: %lld segments", who, (long long)n);
  if (n && (!segs || !is_aligned(segs, 8))) return fail(AEKV_ERR_VALUE, "%s: null or unaligned segments", who);
  return AEKV_OK;
}

int launch_copies(const char* who, const int32_t* ws, const int32_t* copies, int64_t most, const void* segs, int64_t n, int32_t* table, int64_t entries, int64_t pages,
                  hipStream_t st) {
  int64_t blocks = ceil_div(most * n, static_cast<int64_t>(4));
  if (blocks < ceil_div(entries, 256)) blocks = ceil_div(entries, 256);
  if (!blocks) return AEKV_OK;
  hipLaunchKernelGGL(pool_copy_kernel, dim3(static_cast<uint32_t>(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, ws, copies,
                     static_cast<const Segment*>(segs), static_cast<int32_t>(n), table, entries, static_cast<int32_t>(pages));
  return check_launch(who);
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" size_t aekv_pool_workspace_size(int64_t B, int64_t max_pages, int64_t n_forks, int64_t pages) {
  if (B < 0 || max_pages < 0 || n_forks < 0 || pages < 0 || B > kMaxRows || max_pages > 0x7fffffff || B * max_pages > 0x3fffffff || n_forks > 0x3fffffff || pages > 0x3fffffff) return 0;
  const int64_t reserve = 4 * B * max_pages, fork = n_forks * max_pages, compact = 3 * pages;
  const int64_t most = reserve > fork ? reserve : fork;
  return static_cast<size_t>(kHeader + (most > compact ? most : compact)) * 4;
}

extern "C" int aekv_pool_reserve(int32_t* table, int64_t B, int64_t max_pages, const int32_t* filled, const int32_t* wanted,
                                 const int32_t* first, int32_t page_size, int32_t* refs, int32_t* marks, int32_t* lacking,
                                 int64_t pages, const void* segments, int64_t n_segments, void* ws, size_t ws_bytes,
                                 void* stream) {
  const char* who = "aekv_pool_reserve";
  if (const int rc = check_table(who, table, B, max_pages, pages, refs)) return rc;
  if (const int rc = check_segments(who, segments, n_segments)) return rc;
  const int shift = page_shift(page_size);
  if (shift < 0) return fail(AEKV_ERR_VALUE, "%s: page_size must be a power of two from 16 to 4096, got %d", who, page_size);
  if (B * max_pages == 0) return AEKV_OK;
  if (!filled || !wanted || !marks || !lacking) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  const size_t want = aekv_pool_workspace_size(B, max_pages, 0, 0);
  if (!ws || ws_bytes < want) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  PoolArgs a{};
  a.table = table, a.B = static_cast<int32_t>(B), a.W = static_cast<int32_t>(max_pages), a.shift = shift, a.filled = filled, a.wanted = wanted, a.first = first;
  a.refs = refs, a.marks = marks, a.lacking = lacking, a.pages = static_cast<int32_t>(pages), a.ws = static_cast<int32_t*>(ws);
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(pool_reserve_kernel, dim3(1), dim3(kThreads), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  return launch_copies(who, a.ws, a.ws + kHeader + 2 * B * max_pages, B * max_pages, segments, n_segments, nullptr, 0, 0, st);
}

extern "C" int aekv_pool_release(int32_t* table, int64_t B, int64_t max_pages, const int32_t* keep, int32_t page_size,
                                 int32_t* refs, int64_t pages, void* stream) {
  const char* who = "aekv_pool_release";
  if (const int rc = check_table(who, table, B, max_pages, pages, refs)) return rc;
  const int shift = page_shift(page_size);
  if (shift < 0) return fail(AEKV_ERR_VALUE, "%s: page_size must be a power of two from 16 to 4096, got %d", who, page_size);
  if (B * max_pages == 0) return AEKV_OK;
  if (!keep) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  PoolArgs a{};
  a.table = table, a.B = static_cast<int32_t>(B), a.W = static_cast<int32_t>(max_pages), a.shift = shift, a.wanted = keep, a.refs = refs, a.pages = static_cast<int32_t>(pages);
  hipLaunchKernelGGL(pool_release_kernel, dim3(static_cast<uint32_t>(ceil_div(B * max_pages, 256))), dim3(256), 0, as_stream(stream), a);
  return check_launch(who);
}

extern "C" int aekv_pool_fork(int32_t* table, int64_t B, int64_t max_pages, const int32_t* filled, const int32_t* source,
                              const int32_t* target, int64_t n, int32_t page_size, int32_t* refs, int64_t pages, void* ws,
                              size_t ws_bytes, void* stream) {
  const char* who = "aekv_pool_fork";
  if (const int rc = check_table(who, table, B, max_pages, pages, refs)) return rc;
  const int shift = page_shift(page_size);
  if (shift < 0) return fail(AEKV_ERR_VALUE, "%s: page_size must be a power of two from 16 to 4096, got %d", who, page_size);
  if (n < 0 || n > 0x3fffffff || n * max_pages > 0x3fffffff) return fail(AEKV_ERR_SHAPE, "%s: %lld forks of %lld pages", who, (long long)n, (long long)max_pages);
  if (B * max_pages == 0 || n == 0) return AEKV_OK;
  if (!filled || !source || !target) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  const size_t want = aekv_pool_workspace_size(0, max_pages, n, 0);
  if (!ws || ws_bytes < want) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  PoolArgs a{};
  a.table = table, a.B = static_cast<int32_t>(B), a.W = static_cast<int32_t>(max_pages), a.shift = shift, a.filled = filled, a.refs = refs;
  a.pages = static_cast<int32_t>(pages), a.ws = static_cast<int32_t*>(ws);
  hipLaunchKernelGGL(pool_fork_kernel, dim3(static_cast<uint32_t>(ceil_div(max_pages, kColumns))), dim3(256), B * sizeof(int32_t), as_stream(stream), a, source, target,
                     static_cast<int32_t>(n));
  return check_launch(who);
}

extern "C" int aekv_pool_compact(int32_t* table, int64_t n, int32_t* refs, int64_t pages, const void* segments, int64_t n_segments, void* ws, size_t ws_bytes,
                                 void* stream) {
  const char* who = "aekv_pool_compact";
  if (n < 0 || pages < 0 || pages > 0x3fffffff || n > 0x3fffffff) return fail(AEKV_ERR_SHAPE, "%s: %lld entries of %lld pages", who, (long long)n, (long long)pages);
  if (const int rc = check_segments(who, segments, n_segments)) return rc;
  const size_t want = aekv_pool_workspace_size(0, 0, 0, pages);
  if (!ws || ws_bytes < want) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  if ((pages && !refs) || (n && !table)) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  PoolArgs a{};
  a.refs = refs, a.pages = static_cast<int32_t>(pages), a.ws = static_cast<int32_t*>(ws);
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(pool_compact_kernel, dim3(1), dim3(kThreads), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  return launch_copies(who, a.ws, a.ws + kHeader + pages, ceil_div(pages, static_cast<int64_t>(2)), segments, n_segments, table, n, pages, st);
}

extern "C" int aekv_pool_renumber(int32_t* table, int64_t n, int64_t pages, const void* ws, size_t ws_bytes, void* stream) {
  const char* who = "aekv_pool_renumber";
  if (n < 0 || pages < 0 || pages > 0x3fffffff || n > 0x3fffffff) return fail(AEKV_ERR_SHAPE, "%s: %lld entries of %lld pages", who, (long long)n, (long long)pages);
  if (n == 0) return AEKV_OK;
  if (!table) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (!ws || ws_bytes < aekv_pool_workspace_size(0, 0, 0, pages)) return fail(AEKV_ERR_WORKSPACE, "%s: the workspace of aekv_pool_compact is needed", who);
  hipLaunchKernelGGL(pool_renumber_kernel, dim3(static_cast<uint32_t>(ceil_div(n, 256))), dim3(256), 0, as_stream(stream), table, n, static_cast<int32_t>(pages),
                     static_cast<const int32_t*>(ws));
  return check_launch(who);
}
