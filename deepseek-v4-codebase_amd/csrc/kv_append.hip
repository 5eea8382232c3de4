// New tokens into a paged per-head cache: every K and V vector is coded (PolarQuant.encode, bit for bit) straight into
// its slot's row, and the slot's tracker entries, where there are any, are started.
//
// Reference: the encode is aether_2b/turbo_quant.py:127-166; the reference engine appends coded blocks with torch.cat
// (aether_2b/serving.py:327-346).
//
// Two layouts, bit for bit alike.  Small calls (and fp32): D / 8 lanes hold one vector, 8 elements each, so that a decode
// step's few vectors spread over many waves; bound by the chain of a wave (load, exchanges, divisions, store): 64 tokens x
// 4 heads 3.9 us.  Large calls: 32 elements to a lane (tq_fast_lane.h), a wave taking VPW consecutive tokens of one head of
// K or V, so that it reads whole rows and writes its codes contiguously; bound by its vector instructions (some 500 a wave,
// the codec's own 435 among them) with the reads and writes close behind: 8 prompts of up to
// 8192 tokens x 12 heads, 334 MB, 75 us, 4.4 TB/s of a copy's 5.0 (81 with a search in 64 bits in every lane).  fp32 keeps the
// first at every size, as the other's registers hold packed 16-bit words: 40000 tokens x 12 heads, 557 MB, 157 us.
#include "paged_cache.h"
#include "tq_fast_lane.h"

namespace aekv {
namespace {

struct AppendArgs {
  PagePool pool;
  const void* k;
  const void* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* cu;      // [B + 1] or null: token n belongs to sequence n / per_seq
  const int32_t* start;   // [B]: slots in use before the call
  const float* diag;
  float* weights;         // [B, heads, capacity] or null
  int32_t* tokens;        // [B, heads, capacity], with weights
  const int32_t* token;   // [B]: token index of each sequence's first new one
  int64_t n_tokens, B, per_seq, capacity;
  float wscale;
};

// The sequence of packed token n: the last b with cu[b] <= n, or -1 where no sequence holds it.
__device__ __forceinline__ int64_t packed_sequence(const int32_t* cu, int64_t B, int64_t n) {
  int64_t lo = 0, hi = B;  // cu[lo] <= n < cu[hi], if the ends hold
  if (n < cu[0] || n >= cu[B]) return -1;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (cu[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  constexpr int EPL = 8, LPV = D / EPL, NB = BITS == 8 ? EPL : EPL / 2;
  const int sub = threadIdx.x % LPV;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LPV;
  const int32_t heads = a.pool.heads;
  const int64_t total = a.n_tokens * 2 * heads;
  const bool in = i < total;
  const int64_t n = in ? i / (2 * heads) : 0;
  const int32_t kh = in ? static_cast<int32_t>(i - n * 2 * heads) : 0;
  const bool is_v = kh >= heads;
  const int32_t h = is_v ? kh - heads : kh;
  float x[EPL];
  load_elems<DT, EPL>(is_v ? a.v : a.k, is_v ? n * a.v_token + h * a.v_head + sub * EPL : n * a.k_token + h * a.k_head + sub * EPL, in, x);
#pragma unroll
  for (int e = 0; e < EPL; ++e) x[e] *= a.diag[sub * EPL + e];
  int64_t b = -1, at = 0;
  if (in) {
    b = a.cu ? packed_sequence(a.cu, a.B, n) : n / a.per_seq;
    if (b >= 0) at = a.cu ? n - a.cu[b] : n - b * a.per_seq;
  }
  const int64_t slot = b >= 0 ? a.start[b] + at : -1;
  const int64_t row = b >= 0 ? cache_row(a.pool, b, h, slot) : -1;
  float m;
  const Bytes<NB> w = encode_lane<BITS, D, true>(x, sub, a.wscale, &m);  // (every lane takes part in the exchanges)
  if (row >= 0) {
    *reinterpret_cast<Bytes<NB>*>((is_v ? a.pool.v_codes : a.pool.k_codes) + row * (D * BITS / 8) + sub * NB) = w;
    if (sub == 0) (is_v ? a.pool.v_scale : a.pool.k_scale)[row] = m / (BITS == 8 ? 127.0f : 7.0f);
    if (sub == 0 && !is_v && a.weights && slot < a.capacity) {
      const int64_t t = (b * heads + h) * a.capacity + slot;
      a.weights[t] = 0.0f;
      a.tokens[t] = a.token[b] + static_cast<int32_t>(at);
    }
  }
}

constexpr int kTableThreads = 256;

// Token n's sequence, its place among that sequence's new tokens, and its slot.
__device__ __forceinline__ int64_t token_slot(const AppendArgs& a, int64_t n, int64_t* b, int64_t* at) {
  *b = a.cu ? packed_sequence(a.cu, a.B, n) : n / a.per_seq;
  if (*b < 0) return -1;
  *at = a.cu ? n - a.cu[*b] : n - *b * a.per_seq;
  return a.start[*b] + *at;
}

// The same for a wave's tokens n0 + v (n0 uniform, fewer than `span` of them): n0's sequence is found once, with scalar
// loads, and lanes step on from it only where the span leaves it.
__device__ __forceinline__ int64_t token_slot_near(const AppendArgs& a, uint32_t n0, uint32_t v, uint32_t span, int32_t* b, int32_t* at) {
  const int32_t n = static_cast<int32_t>(n0 + v), B = static_cast<int32_t>(a.B);
  if (a.cu) {
    int32_t lo = -1, hi = B + 1;  // cu[lo] <= n0 < cu[hi], as if cu[-1] were lowest and cu[B + 1] highest
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (a.cu[mid] <= static_cast<int32_t>(n0)) lo = mid;
      else hi = mid;
    }
    int32_t own = lo;
    if (lo < B && a.cu[lo + 1] < static_cast<int64_t>(n0) + span)
      while (own < B && a.cu[own + 1] <= n) ++own;
    if (own < 0 || own >= B) {
      *b = -1, *at = 0;
      return -1;
    }
    *b = own, *at = n - a.cu[own];
  } else {
    const uint32_t per = static_cast<uint32_t>(a.per_seq), first = n0 / per;
    uint32_t own = first, place = n0 - first * per + v;
    while (place >= per) place -= per, ++own;
    *b = static_cast<int32_t>(own), *at = static_cast<int32_t>(place);
  }
  return static_cast<int64_t>(a.start[*b]) + *at;
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(kTableThreads, 4) void kv_append_rows_kernel(AppendArgs a, float cq) {
  using F = FastEnc<BITS, D>;
  constexpr int LPV = F::LPV, VPW = F::VPW, NW = F::LB / 4;
  const int lane = threadIdx.x & 63;
  const int v = lane / LPV, g = lane % LPV;
  __shared__ uint4 dm_tab[LPV][4];  // diag sign masks of a lane part's 16 packed words
  if (threadIdx.x < 16 * LPV) {
    const int gg = threadIdx.x >> 4, k = threadIdx.x & 15;
    reinterpret_cast<uint32_t*>(dm_tab[gg])[k] = (a.diag[32 * gg + 2 * k] < 0.0f ? 0x8000u : 0u) |
                                                (a.diag[32 * gg + 2 * k + 1] < 0.0f ? 0x80000000u : 0u);
  }
  __syncthreads();
  // the wave's tokens, head, and K or V (neighbouring waves take neighbouring heads: whole token rows are read together)
  const uint32_t heads = static_cast<uint32_t>(a.pool.heads);
  const uint32_t grp = blockIdx.x * (kTableThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile = grp / (2 * heads), kh = grp - tile * 2 * heads;
  const bool is_v = kh >= heads;
  const int32_t h = static_cast<int32_t>(is_v ? kh - heads : kh);
  const int64_t n0 = static_cast<int64_t>(tile) * VPW;
  if (n0 >= a.n_tokens) return;
  const uint8_t* x = static_cast<const uint8_t*>(is_v ? a.v : a.k) + (is_v ? h * a.v_head : h * a.k_head) * 2;
  const int64_t stride = (is_v ? a.v_token : a.k_token) * 2;
  uint8_t* codes = is_v ? a.pool.v_codes : a.pool.k_codes;
  float* scale = is_v ? a.pool.v_scale : a.pool.k_scale;
  const uint32_t last = static_cast<uint32_t>(a.n_tokens - 1 - n0), vn = min(static_cast<uint32_t>(v), last);  // (spare lanes of the last tile read its last token)
  uint32_t w[16];
  {
    const uint4* p = reinterpret_cast<const uint4*>(x + n0 * stride + vn * stride + 64 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 t = p[i];
      w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
    }
  }
  int32_t b = -1, at = 0;
  const int64_t slot = token_slot_near(a, static_cast<uint32_t>(n0), vn, VPW, &b, &at);
  const int64_t row = static_cast<uint32_t>(v) <= last && b >= 0 ? cache_row(a.pool, b, h, slot) : -1;
  if (row >= 0 && g == 0 && !is_v && a.weights && slot < a.capacity) {
    const int64_t t = (static_cast<int64_t>(b) * heads + h) * a.capacity + slot;
    a.weights[t] = 0.0f;
    a.tokens[t] = a.token[b] + at;
  }
  uint32_t dm[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 d = dm_tab[g][i];
    dm[4 * i] = d.x, dm[4 * i + 1] = d.y, dm[4 * i + 2] = d.z, dm[4 * i + 3] = d.w;
  }
  auto exact = [&] {  // the wave's vectors by the other layout, read again
    constexpr int EPL = 8, LPV8 = D / EPL, NB = BITS == 8 ? EPL : EPL / 2;
    const int sub = lane % LPV8;
#pragma unroll 1
    for (int i = lane / LPV8; i < VPW; i += 64 / LPV8) {
      const bool in = n0 + i < a.n_tokens;
      float e[EPL], m;
      load_elems<DT, EPL>(x + (n0 + i) * stride, sub * EPL, in, e);
#pragma unroll
      for (int j = 0; j < EPL; ++j) e[j] *= a.diag[sub * EPL + j];
      const Bytes<NB> c = encode_lane<BITS, D, false>(e, sub, a.wscale, &m);
      int64_t bb = -1, aa = 0;
      const int64_t s = in ? token_slot(a, n0 + i, &bb, &aa) : -1;
      const int64_t r = bb >= 0 ? cache_row(a.pool, bb, h, s) : -1;
      if (r >= 0) {
        *reinterpret_cast<Bytes<NB>*>(codes + r * F::RB + sub * NB) = c;
        if (sub == 0) scale[r] = m / F::Q;
      }
    }
  };
  auto store = [&](const uint32_t (&o)[NW], float m) {
    if (row < 0) return;
    uint4* p = reinterpret_cast<uint4*>(codes + row * F::RB + g * F::LB);
#pragma unroll
    for (int i = 0; i < NW / 4; ++i) p[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    if (g == 0) scale[row] = m / F::Q;
  };
  fast_encode_lane<DT, BITS, D>(w, dm, g, a.wscale, cq, exact, store);
}

// Elements of K and V together from which a call takes the second layout (4-bit D = 128 / 8-bit D = 64, first against
// second: 524288 elements 3.7 / 3.5 and 4.4 / 4.7 us, 1048576 4.0 / 3.9 and 4.8 / 4.7, 2097152 4.9 / 4.8 and 4.8 / 5.0;
// a prompt batch of 98 M elements, 334 MB, 176 and 75 us).
constexpr int64_t kRowsElements = int64_t(1) << 21;

using append_fn = void (*)(AppendArgs);
using rows_fn = void (*)(AppendArgs, float);

template <int DT>
append_fn pick_append(int d, int bits) {
  if (d == 64) return bits == 8 ? kv_append_kernel<DT, 64, 8> : kv_append_kernel<DT, 64, 4>;
  return bits == 8 ? kv_append_kernel<DT, 128, 8> : kv_append_kernel<DT, 128, 4>;
}

template <int DT>
rows_fn pick_rows(int d, int bits) {
  if (d == 64) return bits == 8 ? kv_append_rows_kernel<DT, 64, 8> : kv_append_rows_kernel<DT, 64, 4>;
  return bits == 8 ? kv_append_rows_kernel<DT, 128, 8> : kv_append_rows_kernel<DT, 128, 4>;
}

}  // namespace

int check_pool(const char* who, void* k_codes, float* k_scale, void* v_codes, float* v_scale, int64_t pages,
               int64_t heads, int32_t page_size, int32_t d, int32_t bits, const int32_t* table, int64_t max_pages,
               int64_t B, PagePool* out) {
  if (bits != 4 && bits != 8) return fail(AEKV_ERR_VALUE, "bits must be 4 or 8, got %d", bits);
  if (d != 64 && d != 128) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128 supported)", who, d);
  if (page_size < 16 || page_size > 4096 || !is_pow2(page_size))
    return fail(AEKV_ERR_VALUE, "%s: page_size %d must be a power of two from 16 to 4096", who, page_size);
  if (B < 0 || heads < 1 || pages < 0 || max_pages < 0)
    return fail(AEKV_ERR_SHAPE, "%s: B=%lld heads=%lld pages=%lld max_pages=%lld", who, (long long)B, (long long)heads,
                (long long)pages, (long long)max_pages);
  if (pages > 0x7fffffff || heads > 65535 || max_pages * page_size > 0x7fff0000 || B > 0x7fffffff)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: pages=%lld heads=%lld slots=%lld B=%lld exceed 31 bits (65535 heads)", who,
                (long long)pages, (long long)heads, (long long)(max_pages * page_size), (long long)B);
  if (pages > 0 && (!k_codes || !k_scale || !v_codes || !v_scale)) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (B > 0 && max_pages > 0 && !table) return fail(AEKV_ERR_VALUE, "%s: null page table", who);
  if (!is_aligned(k_codes, 16) || !is_aligned(v_codes, 16) || !is_aligned(k_scale, 16) || !is_aligned(v_scale, 16) ||
      !is_aligned(table, 4))
    return fail(AEKV_ERR_ALIGN, "%s: codes and scales must be 16-byte aligned", who);
  out->k_codes = static_cast<uint8_t*>(k_codes);
  out->k_scale = k_scale;
  out->v_codes = static_cast<uint8_t*>(v_codes);
  out->v_scale = v_scale;
  out->table = table;
  out->pages = static_cast<int32_t>(pages);
  out->max_pages = static_cast<int32_t>(max_pages);
  out->heads = static_cast<int32_t>(heads);
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  out->page_shift = shift;
  return AEKV_OK;
}

}  // namespace aekv

using namespace aekv;

extern "C" int aekv_kv_append(const void* k, const void* v, int32_t dtype, int64_t k_token_stride,
                              int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int64_t n_tokens,
                              const int32_t* cu_seqlens, int64_t B, const int32_t* start, int32_t d, int32_t bits,
                              const float* diag, void* k_codes, float* k_scale, void* v_codes, float* v_scale,
                              int64_t pages, int64_t heads, int32_t page_size, const int32_t* page_table,
                              int64_t max_pages, float* weights, int32_t* tokens, int64_t capacity,
                              const int32_t* token, void* stream) {
  const char* who = "aekv_kv_append";
  AppendArgs a{};
  if (const int rc = check_pool(who, k_codes, k_scale, v_codes, v_scale, pages, heads, page_size, d, bits, page_table,
                                max_pages, B, &a.pool))
    return rc;
  if (!is_float_dtype(dtype)) return fail(AEKV_ERR_DTYPE, "%s: K and V must be F32, F16 or BF16", who);
  if (n_tokens < 0) return fail(AEKV_ERR_SHAPE, "%s: n_tokens=%lld", who, (long long)n_tokens);
  if (!cu_seqlens && B > 0 && n_tokens % B)
    return fail(AEKV_ERR_SHAPE, "%s: %lld tokens are no whole number for each of %lld sequences", who,
                (long long)n_tokens, (long long)B);
  if (weights && (!tokens || !token || capacity < 0)) return fail(AEKV_ERR_VALUE, "%s: weights need tokens and token", who);
  if (B == 0 || n_tokens == 0 || pages == 0 || max_pages == 0) return AEKV_OK;
  if (!k || !v || !start || !diag) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  const size_t na = dtype == AEKV_F32 ? 16 : static_cast<size_t>(8 * es);
  if (!is_aligned(k, na) || !is_aligned(v, na) || (k_token_stride * es) % 16 || (k_head_stride * es) % 16 ||
      (v_token_stride * es) % 16 || (v_head_stride * es) % 16)
    return fail(AEKV_ERR_ALIGN, "%s: K and V rows must be 16-byte aligned", who);
  const int64_t lanes = n_tokens * 2 * heads * (d / 8);
  if (n_tokens > 0x7fffffff || lanes > kMaxGridThreads - 256)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: %lld tokens exceed the grid", who, (long long)n_tokens);
  a.k = k;
  a.v = v;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.cu = cu_seqlens;
  a.start = start;
  a.diag = diag;
  a.weights = weights;
  a.tokens = tokens;
  a.token = token;
  a.n_tokens = n_tokens;
  a.B = B;
  a.per_seq = n_tokens / B;
  a.capacity = capacity;
  a.wscale = wht_scale(d);
  const hipStream_t st = as_stream(stream);
  if (dtype != AEKV_F32 && n_tokens * 2 * heads * d >= kRowsElements) {
    const int64_t groups = ceil_div(n_tokens, static_cast<int64_t>(64 / (d / 32))) * 2 * heads;
    auto fn = dtype == AEKV_F16 ? pick_rows<AEKV_F16>(d, bits) : pick_rows<AEKV_BF16>(d, bits);
    hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(ceil_div(groups, kTableThreads / 64))), dim3(kTableThreads), 0, st, a,
                       (bits == 8 ? 127.0f : 7.0f) * a.wscale);
    return check_launch(who);
  }
  auto fn = dtype == AEKV_F32 ? pick_append<AEKV_F32>(d, bits)
            : dtype == AEKV_F16 ? pick_append<AEKV_F16>(d, bits) : pick_append<AEKV_BF16>(d, bits);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(ceil_div(lanes, 256))), dim3(256), 0, st, a);
  return check_launch(who);
}
