// New tokens into a paged per-head cache: every K and V vector is coded (PolarQuant.encode, bit for bit) straight into
// its slot's row, and the slot's tracker entries, where there are any, are started.
//
// Reference: the encode is aether_2b/turbo_quant.py:127-166; the reference engine appends coded blocks with torch.cat
// (aether_2b/serving.py:327-346).
//
// D / 8 lanes hold one vector, 8 elements each (one 16-byte load of a 16-bit type); the lanes of a vector store its codes
// contiguously.
#include "paged_cache.h"
#include "tq_device.h"

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

template <int DT>
using append_fn = void (*)(AppendArgs);

template <int DT>
append_fn<DT> pick_append(int d, int bits) {
  if (d == 64) return bits == 8 ? kv_append_kernel<DT, 64, 8> : kv_append_kernel<DT, 64, 4>;
  return bits == 8 ? kv_append_kernel<DT, 128, 8> : kv_append_kernel<DT, 128, 4>;
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
  const dim3 grid(static_cast<uint32_t>(ceil_div(lanes, 256)));
  auto fn = dtype == AEKV_F32 ? pick_append<AEKV_F32>(d, bits)
            : dtype == AEKV_F16 ? pick_append<AEKV_F16>(d, bits) : pick_append<AEKV_BF16>(d, bits);
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, as_stream(stream), a);
  return check_launch(who);
}
