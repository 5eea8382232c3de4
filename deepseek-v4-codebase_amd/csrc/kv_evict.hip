// Eviction from a paged per-head cache by accumulated attention weight, in place.
//
// For every (sequence, KV head) with n = lengths[b] > keep slots, the `keep` highest ranked slots stay: first those whose
// token is protected (token < first, or token >= seen[b] - recent), then by weight, larger first (NaN above every number),
// equal ranks by slot, lower first.  Cached keys carry their rotation and the softmax does not depend on the order of its
// terms, so a kept slot below `keep` stays where it is; the holes (evicted slots below `keep`), in increasing order, take
// the kept slots from `keep` on, in increasing order.  Sources and destinations are disjoint: the rows move in place, in
// parallel, and only as many as there are holes.
//
// One workgroup per (sequence, head) selects and lists the moves; it makes them itself where they are few, and the whole
// chip makes them in a second launch where they can be many.
#include "paged_cache.h"

namespace aekv {
namespace {

struct EvictArgs {
  PagePool pool;
  const int32_t* lengths;  // [B]
  float* weights;          // [B, heads, capacity]
  int32_t* tokens;         // [B, heads, capacity]
  const int32_t* seen;     // [B]
  int32_t* counts;         // [B * heads]: moves
  int2* moves;             // [B * heads, most]: (source, destination)
  int64_t capacity;
  int32_t keep, first, recent, most;
};

// Order key of a slot: protected slots first, then weights by size (-0 and +0 alike), NaN above every number.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t token, int32_t first, int64_t recent_from) {
  if (token < first || token >= recent_from) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  return order_key(w + 0.0f);
}

// 16 lanes move one slot: its code rows, scales, weight and token.  (In a launch of its own, bound by the reads and writes:
// 96 rows of 16384 slots to 4096, 8 bits, dim 128, 33 us.)  kMoves slots at a time, so that their dependent loads
// (the move, the pages, the rows) overlap: those of the `count` listed moves from `first` on, every `step`.
constexpr int kMoves = 4;

template <int ROW>
__device__ __forceinline__ void move_slots(const EvictArgs& a, int64_t bh, int64_t b, const int2* moves, int count, int first, int step) {
  constexpr int NB = ROW / 16;
  struct alignas(NB) W { uint8_t x[NB]; };
  const int32_t h = static_cast<int32_t>(bh - b * a.pool.heads);
  const int sub = threadIdx.x & 15;
  for (; first < count; first += step) {
    int2 mv[kMoves];
    int64_t src[kMoves], dst[kMoves];
    W kc[kMoves], vc[kMoves];
    uint32_t extra[kMoves];
#pragma unroll
    for (int i = 0; i < kMoves; ++i) mv[i] = moves[min(first + i, count - 1)];  // (the last again past the end: not stored)
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      src[i] = cache_row(a.pool, b, h, mv[i].x);
      dst[i] = cache_row(a.pool, b, h, mv[i].y);
    }
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int64_t r = src[i] < 0 ? 0 : src[i];  // (a pool has a first row)
      kc[i] = *reinterpret_cast<const W*>(a.pool.k_codes + r * ROW + sub * NB);
      vc[i] = *reinterpret_cast<const W*>(a.pool.v_codes + r * ROW + sub * NB);
      // lanes 0 .. 3: K scale, V scale, weight, token
      const int64_t slot = bh * a.capacity + mv[i].x;
      const uint32_t* from = sub == 0   ? reinterpret_cast<const uint32_t*>(a.pool.k_scale) + r
                             : sub == 1 ? reinterpret_cast<const uint32_t*>(a.pool.v_scale) + r
                             : sub == 2 ? reinterpret_cast<const uint32_t*>(a.weights) + slot
                                        : reinterpret_cast<const uint32_t*>(a.tokens) + slot;
      extra[i] = *from;
    }
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      if (first + i >= count) break;
      const bool there = src[i] >= 0 && dst[i] >= 0;
      if (there) {
        *reinterpret_cast<W*>(a.pool.k_codes + dst[i] * ROW + sub * NB) = kc[i];
        *reinterpret_cast<W*>(a.pool.v_codes + dst[i] * ROW + sub * NB) = vc[i];
      }
      const int64_t slot = bh * a.capacity + mv[i].y;
      if (sub == 0 && there) reinterpret_cast<uint32_t*>(a.pool.k_scale)[dst[i]] = extra[i];
      if (sub == 1 && there) reinterpret_cast<uint32_t*>(a.pool.v_scale)[dst[i]] = extra[i];
      if (sub == 2) reinterpret_cast<uint32_t*>(a.weights)[slot] = extra[i];
      if (sub == 3) a.tokens[slot] = static_cast<int32_t>(extra[i]);
    }
  }
}

// One workgroup per (sequence, head).  Its waves own consecutive runs of slots, 64 kRegRows or fewer each, whose keys stay in
// registers while the threshold is found; longer rows go through in rounds of kRound slots, read again for each pass.
//
// The threshold: the keep-th largest key by 11, 11 and 10 bits from the top, each level a histogram in LDS of the keys that
// share the bits above, searched from its largest bin by all waves.  A level whose bin is kept whole ends it.
// The order: ballots rank a wave's ties, holes and movers by slot; one word per wave carries the counts between waves.
//
// Bound by its barriers and the chain of its loads: 1088 slots with up to 64 moves made here 10 us (16 sequences x 4 heads;
// with the moves in a launch of their own 2 us more), 16384 slots 27 us (96 rows).
constexpr int kRegRows = 16, kBins = 2048;

// The waves' counts before this one's, and their total, for two counters (the first below 2^32, packed with the second).
template <int kWaves>
__device__ __forceinline__ uint64_t wave_prefix(uint64_t mine, uint64_t* part, int lane, int wave, uint64_t* total) {
  __syncthreads();  // the readers of the call before are done
  if (lane == 0) part[wave] = mine;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t p = part[w];
    before += w < wave ? p : 0;
    all += p;
  }
  *total = all;
  return before;
}

// ROW: 0 lists the moves for the launch that makes them; else a row's moves are at most kOwnMoves, and the workgroup makes
// them itself, from a list in LDS.
constexpr int kOwnMoves = 256;

template <int ROW, int kSelThreads>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  constexpr int kWaves = kSelThreads / 64, kRound = kSelThreads * kRegRows, kPer = kBins / kSelThreads;
  __shared__ int2 s_moves[ROW ? kOwnMoves : 1];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t s_sum[kWaves];
  __shared__ uint64_t s_part[kWaves];
  __shared__ int s_found[3];  // bin, keys of it that stay, keys in it
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / a.pool.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t cap = static_cast<int32_t>(min<int64_t>(table_slots(a.pool), a.capacity));
  const int32_t n = min(a.lengths[b], cap);
  const int64_t recent_from = static_cast<int64_t>(a.seen[b]) - a.recent;
  if (n <= a.keep) {  // (the whole workgroup)
    if (ROW == 0 && tid == 0) a.counts[bh] = 0;
    return;
  }
  const float* w = a.weights + bh * a.capacity;
  const int32_t* tok = a.tokens + bh * a.capacity;
  // the waves' runs in a round that starts at `base`: `rows` rows of 64 slots each
  uint32_t key[kRegRows];
  int rows = 0, run = 0;
  auto load_round = [&](int base) __attribute__((always_inline)) {
    const int left = min(n - base, kRound);
    rows = __builtin_amdgcn_readfirstlane((left + kSelThreads - 1) / kSelThreads);
    run = base + wave * rows * 64;
    float wt[kRegRows];
    int32_t tk[kRegRows];
#pragma unroll
    for (int r = 0; r < kRegRows; ++r) {
      if (r >= rows) break;
      const int i = min(run + 64 * r + lane, n - 1);
      wt[r] = w[i], tk[r] = tok[i];
    }
#pragma unroll
    for (int r = 0; r < kRegRows; ++r) {
      if (r >= rows) break;
      key[r] = evict_key(wt[r], tk[r], a.first, recent_from);
    }
  };
  const bool one_round = n <= kRound;
  if (one_round) load_round(0);
  uint32_t prefix = 0;
  int need = a.keep, shift = 21;
  for (;;) {
    const int width = shift == 0 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int base = 0; base < n; base += kRound) {
      if (!one_round) load_round(base);
#pragma unroll
      for (int r = 0; r < kRegRows; ++r) {
        if (r >= rows) break;
        if (run + 64 * r + lane < n && (shift == 21 || (key[r] >> (shift + width)) == (prefix >> (shift + width))))
          atomicAdd(&hist[(key[r] >> shift) & ((1u << width) - 1)], 1u);
      }
    }
    __syncthreads();
    // bins from the top: thread t holds the kPer from 2047 - kPer t down
    uint32_t h[kPer], own = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) own += h[i] = hist[kBins - 1 - kPer * tid - i];
    uint32_t s = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(s, d);
      if (lane >= d) s += o;
    }
    if (lane == 63) s_sum[wave] = s;
    __syncthreads();
    uint32_t above = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) above += v < wave ? s_sum[v] : 0;
    above += s - own;  // keys in higher bins than this thread's
    const uint32_t want = static_cast<uint32_t>(need);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (above < want && above + h[i] >= want) s_found[0] = kBins - 1 - kPer * tid - i, s_found[1] = want - above, s_found[2] = h[i];
      above += h[i];
    }
    if (need == 0 && tid == 0) s_found[0] = kBins - 1, s_found[1] = 0, s_found[2] = -1;
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_found[0]) << shift;
    need = s_found[1];
    if (need == s_found[2] || shift == 0 || a.keep == 0) break;
    shift = shift == 21 ? 10 : 0;
  }
  // in slot order: of the keys that share the threshold's bits the first `need` stay; holes and movers by their ranks
  uint64_t ties = 0, moved = 0;  // of the rounds before; holes low, movers high
  int2* const mv = ROW ? s_moves : a.moves + bh * a.most;
  const uint32_t room = ROW ? kOwnMoves : static_cast<uint32_t>(a.most);
  const uint64_t below = (1ull << lane) - 1;
  for (int base = 0; base < n; base += kRound) {
    if (!one_round) load_round(base);
    uint64_t mine = 0, total;
#pragma unroll
    for (int r = 0; r < kRegRows; ++r) {
      if (r >= rows) break;
      const bool in = run + 64 * r + lane < n;
      mine += __popcll(__builtin_amdgcn_ballot_w64(in && (key[r] >> shift) == (prefix >> shift)));
    }
    uint64_t rank = ties + wave_prefix<kWaves>(mine, s_part, lane, wave, &total);
    ties += total;
    uint32_t hole = 0, mover = 0;  // bit r: the slot of row r
    uint64_t count = 0;
#pragma unroll
    for (int r = 0; r < kRegRows; ++r) {
      if (r >= rows) break;
      const int i = run + 64 * r + lane;
      const bool in = i < n;
      const bool tie = in && (key[r] >> shift) == (prefix >> shift);
      const uint64_t tm = __builtin_amdgcn_ballot_w64(tie);
      const bool kept = in && ((key[r] >> shift) > (prefix >> shift) || (tie && rank + __popcll(tm & below) < static_cast<uint64_t>(need)));
      rank += __popcll(tm);
      const bool h = in && !kept && i < a.keep, m = kept && i >= a.keep;
      hole |= (h ? 1u : 0u) << r;
      mover |= (m ? 1u : 0u) << r;
      count += __popcll(__builtin_amdgcn_ballot_w64(h)) + (static_cast<uint64_t>(__popcll(__builtin_amdgcn_ballot_w64(m))) << 32);
    }
    uint64_t at = moved + wave_prefix<kWaves>(count, s_part, lane, wave, &total);
    moved += total;
#pragma unroll
    for (int r = 0; r < kRegRows; ++r) {
      if (r >= rows) break;
      const int i = run + 64 * r + lane;
      const bool h = (hole >> r) & 1u, m = (mover >> r) & 1u;
      const uint64_t hm = __builtin_amdgcn_ballot_w64(h), mm = __builtin_amdgcn_ballot_w64(m);
      const uint32_t to = static_cast<uint32_t>(at) + __popcll(hm & below), from = static_cast<uint32_t>(at >> 32) + __popcll(mm & below);
      if (h && to < room) mv[to].y = i;
      if (m && from < room) mv[from].x = i;
      at += __popcll(hm) + (static_cast<uint64_t>(__popcll(mm)) << 32);
    }
  }
  // as many holes as movers, `room` at most: keep slots stay.  (Weights that another stream changes meanwhile, which a long
  // row reads again for every pass, break that; no move may then go anywhere else.)
  const int count = static_cast<int>(min(min(static_cast<uint32_t>(moved), static_cast<uint32_t>(moved >> 32)), room));
  if constexpr (ROW == 0) {
    if (tid == 0) a.counts[bh] = count;
  } else {
    __syncthreads();
    move_slots<ROW>(a, bh, b, s_moves, count, (tid >> 4) * kMoves, kSelThreads / 16 * kMoves);
  }
}

template <int ROW>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, uint32_t per) {  // `per` workgroups to a row
  const uint32_t row = blockIdx.x / per;
  const int64_t bh = row;
  move_slots<ROW>(a, bh, bh / a.pool.heads, a.moves + bh * a.most, a.counts[bh],
                  static_cast<int>((blockIdx.x - row * per) * 16 + (threadIdx.x >> 4)) * kMoves, static_cast<int>(per) * 16 * kMoves);
}

using evict_fn = void (*)(EvictArgs);
template <int THREADS>
evict_fn pick_select(int row) {
  return row == 0 ? evict_select_kernel<0, THREADS> : row == 32 ? evict_select_kernel<32, THREADS>
       : row == 64 ? evict_select_kernel<64, THREADS> : evict_select_kernel<128, THREADS>;
}
// Slots of a row up to which eight waves select, whose keys they hold in registers; beyond, sixteen.  More waves shorten the
// passes and make each barrier longer; sixteen fill half a CU.  8 / 16 waves (256 threads: 4), with a copy of the weights
// before each call, 3 to 5 us: 16 sequences x 4 heads of 1088 slots to 1024 12.3 / 16.6 us (12.5), 256 x 8 42 / 87 (35), 16 x 4
// of 4000 to 3900 16.1 / 18.4 (4096: 23.3), 64 x 8 of 8000 to 7900 40 / 51, 8 x 12 of 16384 to 4096 70.6 / 60.1.
constexpr int64_t kSmallRow = 8192;

int64_t evict_most(int64_t keep, int64_t slots) { return keep >= slots ? 0 : (keep < slots - keep ? keep : slots - keep); }

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" size_t aekv_kv_evict_workspace_size(int64_t B, int64_t heads, int64_t keep, int64_t slots) {
  if (B <= 0 || heads <= 0 || keep < 0 || slots <= keep) return 0;
  return align_up(static_cast<size_t>(B * heads) * 4, 16) + static_cast<size_t>(B * heads * evict_most(keep, slots)) * 8;
}

extern "C" int aekv_kv_evict(int32_t d, int32_t bits, void* k_codes, float* k_scale, void* v_codes, float* v_scale,
                             int64_t pages, int64_t heads, int32_t page_size, const int32_t* page_table,
                             int64_t max_pages, int64_t B, const int32_t* lengths, float* weights, int32_t* tokens,
                             int64_t capacity, const int32_t* seen, int64_t keep, int64_t first, int64_t recent,
                             void* ws, size_t ws_bytes, void* stream) {
  const char* who = "aekv_kv_evict";
  EvictArgs a{};
  if (const int rc = check_pool(who, k_codes, k_scale, v_codes, v_scale, pages, heads, page_size, d, bits, page_table,
                                max_pages, B, &a.pool))
    return rc;
  if (capacity < 0) return fail(AEKV_ERR_SHAPE, "%s: capacity=%lld", who, (long long)capacity);
  if (keep < 0 || first < 0 || recent < 0 || first + recent > keep)
    return fail(AEKV_ERR_VALUE, "%s: keep=%lld must hold the %lld first and %lld recent tokens", who, (long long)keep,
                (long long)first, (long long)recent);
  const int64_t slots = max_pages * page_size < capacity ? max_pages * page_size : capacity;
  if (B == 0 || keep >= slots) return AEKV_OK;  // no sequence can be longer than that
  if (!lengths || !weights || !tokens || !seen) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  const size_t want = aekv_kv_evict_workspace_size(B, heads, keep, slots);
  if (!ws || ws_bytes < want) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16) || !is_aligned(weights, 4) || !is_aligned(tokens, 4))
    return fail(AEKV_ERR_ALIGN, "%s: misaligned pointer", who);
  if (pages == 0) return AEKV_OK;  // nothing is there
  if (B * heads > kMaxGridThreads / 1024) return fail(AEKV_ERR_UNSUPPORTED, "%s: %lld (sequence, head) rows exceed the grid", who, (long long)(B * heads));
  a.lengths = lengths;
  a.weights = weights;
  a.tokens = tokens;
  a.seen = seen;
  a.counts = static_cast<int32_t*>(ws);
  a.moves = reinterpret_cast<int2*>(static_cast<uint8_t*>(ws) + align_up(static_cast<size_t>(B * heads) * 4, 16));
  a.capacity = capacity;
  a.keep = static_cast<int32_t>(keep);
  a.first = static_cast<int32_t>(first);
  a.recent = static_cast<int32_t>(recent);
  a.most = static_cast<int32_t>(evict_most(keep, slots));
  const hipStream_t st = as_stream(stream);
  const int row = d * bits / 8;
  const bool own = a.most > 0 && a.most <= kOwnMoves;
  auto sel = slots <= kSmallRow ? pick_select<512>(own ? row : 0) : pick_select<1024>(own ? row : 0);
  hipLaunchKernelGGL(sel, dim3(static_cast<uint32_t>(B * heads)), dim3(slots <= kSmallRow ? 512 : 1024), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  if (own || a.most == 0) return AEKV_OK;  // (keep = 0: nothing stays, nothing moves)
  const int64_t all = ceil_div(a.most, 16 * kMoves), per = all < 64 ? all : 64, fit = kMaxGridThreads / 256 / (B * heads);  // (fit >= 4)
  const uint32_t each = static_cast<uint32_t>(per < fit ? per : fit);
  auto fn = row == 32 ? evict_move_kernel<32> : row == 64 ? evict_move_kernel<64> : evict_move_kernel<128>;
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(B * heads) * each), dim3(256), 0, st, a, each);
  return check_launch(who);
}
