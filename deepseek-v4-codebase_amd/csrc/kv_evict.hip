// Eviction from a paged per-head cache by accumulated attention weight, in place.
//
// For every (sequence, KV head) with n = lengths[b] > keep slots, the `keep` highest ranked slots stay: first those whose
// token is protected (token < first, or token >= seen[b] - recent), then by weight, larger first (NaN above every number),
// equal ranks by slot, lower first.  Cached keys carry their rotation and the softmax does not depend on the order of its
// terms, so a kept slot below `keep` stays where it is; the holes (evicted slots below `keep`), in increasing order, take
// the kept slots from `keep` on, in increasing order.  Sources and destinations are disjoint: the rows move in place, in
// parallel, and only as many as there are holes.
//
// Two launches: one workgroup per (sequence, head) selects and lists the moves, then the whole chip moves the rows.
#include "paged_cache.h"

namespace aekv {
namespace {

constexpr int kSelThreads = 1024;

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

// Exclusive sum of v over the workgroup's threads in order; *total its whole.  `part`: one word per wave.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();  // part's readers of the call before are done
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelThreads / 64; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  *total = all;
  return before + s - v;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ int part[kSelThreads / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / a.pool.heads;
  const int32_t cap = static_cast<int32_t>(min<int64_t>(table_slots(a.pool), a.capacity));
  const int32_t n = min(a.lengths[b], cap);
  const int tid = threadIdx.x;
  if (n <= a.keep) {  // (the whole workgroup)
    if (tid == 0) a.counts[bh] = 0;
    return;
  }
  const float* w = a.weights + bh * a.capacity;
  const int32_t* tok = a.tokens + bh * a.capacity;
  const int64_t recent_from = static_cast<int64_t>(a.seen[b]) - a.recent;
  // the keep-th largest key, 8 bits at a time: `prefix` its leading bits, `need` how many of the keys with that prefix stay
  uint32_t prefix = 0;
  int need = a.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t key = evict_key(w[i], tok[i], a.first, recent_from);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, bin = 255;
      while (bin > 0 && left > static_cast<int>(hist[bin])) left -= static_cast<int>(hist[bin--]);
      s_prefix = prefix | (static_cast<uint32_t>(bin) << shift);
      s_need = left;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // in slot order: the first `need` of the keys equal to the threshold stay; holes and movers by their ranks
  int ties = 0, holes = 0, movers = 0;
  int2* mv = a.moves + bh * a.most;
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + tid;
    const uint32_t key = i < n ? evict_key(w[i], tok[i], a.first, recent_from) : 0u;
    const bool tie = i < n && key == prefix;
    int total;
    const int rank = ties + block_scan(tie, part, &total);
    ties += total;
    const bool kept = i < n && (key > prefix || (tie && rank < need));
    const bool hole = i < n && !kept && i < a.keep, mover = kept && i >= a.keep;
    const int hr = holes + block_scan(hole, part, &total);
    holes += total;
    const int mr = movers + block_scan(mover, part, &total);
    movers += total;
    if (hole) mv[hr].y = i;
    if (mover) mv[mr].x = i;
  }
  if (tid == 0) a.counts[bh] = holes;  // (as many movers: keep slots stay)
}

// 16 lanes move one slot: its code rows, scales, weight and token.
template <int ROW>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  const int64_t bh = blockIdx.y;
  const int64_t b = bh / a.pool.heads;
  const int32_t h = static_cast<int32_t>(bh - b * a.pool.heads);
  const int count = a.counts[bh];
  const int sub = threadIdx.x & 15;
  for (int m = blockIdx.x * 16 + (threadIdx.x >> 4); m < count; m += gridDim.x * 16) {
    const int2 mv = a.moves[bh * a.most + m];
    const int64_t src = cache_row(a.pool, b, h, mv.x), dst = cache_row(a.pool, b, h, mv.y);
    if (src >= 0 && dst >= 0) {
      constexpr int NB = ROW / 16;
      struct alignas(NB) W { uint8_t x[NB]; };
      const W kc = *reinterpret_cast<const W*>(a.pool.k_codes + src * ROW + sub * NB);
      const W vc = *reinterpret_cast<const W*>(a.pool.v_codes + src * ROW + sub * NB);
      *reinterpret_cast<W*>(a.pool.k_codes + dst * ROW + sub * NB) = kc;
      *reinterpret_cast<W*>(a.pool.v_codes + dst * ROW + sub * NB) = vc;
      if (sub == 0) {
        a.pool.k_scale[dst] = a.pool.k_scale[src];
        a.pool.v_scale[dst] = a.pool.v_scale[src];
      }
    }
    if (sub == 1) {
      a.weights[bh * a.capacity + mv.y] = a.weights[bh * a.capacity + mv.x];
      a.tokens[bh * a.capacity + mv.y] = a.tokens[bh * a.capacity + mv.x];
    }
  }
}

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
  if (B * heads > 65535) return fail(AEKV_ERR_UNSUPPORTED, "%s: %lld (sequence, head) rows exceed the grid", who, (long long)(B * heads));
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
  hipLaunchKernelGGL(evict_select_kernel, dim3(static_cast<uint32_t>(B * heads)), dim3(kSelThreads), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  if (a.most == 0) return AEKV_OK;  // keep = 0: nothing stays, nothing moves
  const int64_t per = ceil_div(a.most, 16);
  const dim3 grid(static_cast<uint32_t>(per < 64 ? per : 64), static_cast<uint32_t>(B * heads));
  const int row = d * bits / 8;
  auto fn = row == 32 ? evict_move_kernel<32> : row == 64 ? evict_move_kernel<64> : evict_move_kernel<128>;
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, st, a);
  return check_launch(who);
}
