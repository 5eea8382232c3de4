// Attention of a sequence's newest tokens over its paged per-head cache in TurboQuant codes.
//
// Token t (of T, the last T slots of each sequence) of query head h sees slots j < lengths[b] - T + 1 + t of KV head
// h / (H / heads):  l_j = scale q . K_j,  p_j = exp(l_j) / (sum exp(l) + exp(sink_h)),  out = sum_j p_j V_j.
// With the codec's orthogonal rotation R = c Had diag (K_j = s_j R^T codes_j) both products stay in the rotated domain:
//   q . K_j = s_j (R q) . codes_j        sum_j p_j V_j = R^T sum_j p_j s_j codes_j
// so a query is rotated once, an output is rotated back once, and a cached row costs its codes and one scale.
// weights[b, KV head, j] += the sum of p_j over the group's heads and the T tokens.
#include "paged_cache.h"
#include "tq_device.h"

namespace aekv {
namespace {

constexpr float kNegInf = -__builtin_inff();

struct PagedArgs {
  PagePool pool;
  const void* q;
  int64_t q_batch, q_token, q_head;  // strides in elements
  const int32_t* lengths;            // [B]
  const float* diag;
  const float* sink;                 // [H] or null
  float* weights;                    // [B, heads, capacity] or null
  float* rot;                        // [B, T, H, D]: rotated queries (with weights)
  float* lse;                        // [B, T, H] (with weights)
  void* out;                         // [B, T, H, D]
  int64_t capacity;
  int32_t T, H;
  float scale, wscale;
};

template <int BITS>
__device__ __forceinline__ float code_at(const uint8_t* row, int d) {
  if constexpr (BITS == 8) return static_cast<float>(static_cast<int8_t>(row[d]));
  const int x = (row[d >> 1] >> (4 * (d & 1))) & 15;
  return static_cast<float>((x ^ 8) - 8);
}

__device__ __forceinline__ int32_t visible_slots(const PagedArgs& a, int64_t b, int32_t t) {
  const int64_t cap = a.weights ? min<int64_t>(table_slots(a.pool), a.capacity) : table_slots(a.pool);
  const int64_t n = min<int64_t>(a.lengths[b], cap);
  return static_cast<int32_t>(max<int64_t>(n - a.T + 1 + t, 0));
}

// y[d] = c sum_e (-1)^popcount(d & e) x[e]
template <int D>
__device__ __forceinline__ float wht_at(const float* x, int d, float c) {
  float s = 0.0f;
  for (int e = 0; e < D; ++e) s += (__popc(d & e) & 1) ? -x[e] : x[e];
  return s * c;
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedArgs a) {
  __shared__ float xs[D], qr[D], ps[4][64], acc[4][D], ml[4][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t h = blockIdx.x, t = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int32_t kh = h / (a.H / a.pool.heads);
  if (tid < D) {
    const int64_t at = b * a.q_batch + t * a.q_token + h * a.q_head + tid;
    const uint16_t u = static_cast<const uint16_t*>(a.q)[at];
    xs[tid] = (DT == AEKV_BF16 ? bf16_to_f32(u) : f16_to_f32(u)) * a.diag[tid];
  }
  __syncthreads();
  if (tid < D) qr[tid] = wht_at<D>(xs, tid, a.wscale);
  __syncthreads();
  const int64_t orow = (b * a.T + t) * a.H + h;
  if (a.weights && tid < D) a.rot[orow * D + tid] = qr[tid];
  const int32_t n = visible_slots(a, b, t);
  float m = kNegInf, l = 0.0f, o[D / 64];
  for (int i = 0; i < D / 64; ++i) o[i] = 0.0f;
  for (int base = 64 * wave; base < n; base += 256) {
    const int j = base + lane;
    const int64_t row = j < n ? cache_row(a.pool, b, kh, j) : -1;
    float s = kNegInf, vs = 0.0f;
    if (row >= 0) {
      const uint8_t* kr = a.pool.k_codes + row * (D * BITS / 8);
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot += qr[d] * code_at<BITS>(kr, d);
      s = dot * a.pool.k_scale[row] * a.scale;
      vs = a.pool.v_scale[row];
    }
    const float m2 = fmaxf(m, wave_max(s));
    const float r = m2 == kNegInf ? 1.0f : expf(m - m2);
    const float p = s == kNegInf ? 0.0f : expf(s - m2);
    l = l * r + wave_sum(p);
    m = m2;
    ps[wave][lane] = row >= 0 ? p * vs : 0.0f;
    __builtin_amdgcn_wave_barrier();
    for (int i = 0; i < D / 64; ++i) o[i] *= r;
    for (int k = 0; k < 64; ++k) {
      const int64_t vrow = __shfl(row, k);
      if (vrow < 0) continue;
      for (int i = 0; i < D / 64; ++i) o[i] += ps[wave][k] * code_at<BITS>(a.pool.v_codes + vrow * (D * BITS / 8), lane + 64 * i);
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int i = 0; i < D / 64; ++i) acc[wave][lane + 64 * i] = o[i];
  if (lane == 0) ml[wave][0] = m, ml[wave][1] = l;
  __syncthreads();
  float M = a.sink ? a.sink[h] : kNegInf, L = M == kNegInf ? 0.0f : 1.0f;
  float x = 0.0f;
  for (int w = 0; w < 4; ++w) {
    if (ml[w][1] == 0.0f) continue;  // (NaN alone leaves a maximum of -inf, and a sum that says so)
    const float M2 = fmaxf(M, ml[w][0]);
    const float r = M == kNegInf ? 0.0f : expf(M - M2), f = expf(ml[w][0] - M2);
    L = L * r + ml[w][1] * f;
    x = x * r + (tid < D ? acc[w][tid] : 0.0f) * f;
    M = M2;
  }
  __syncthreads();
  if (tid < D) xs[tid] = L > 0.0f ? x / L : (L == 0.0f ? 0.0f : L);
  __syncthreads();
  if (tid < D) {
    const float y = wht_at<D>(xs, tid, a.wscale) * a.diag[tid];
    static_cast<uint16_t*>(a.out)[orow * D + tid] = DT == AEKV_BF16 ? static_cast<uint16_t>(pack_bf16x2(y, 0.0f)) : static_cast<uint16_t>(f32_to_f16_bits(y));
  }
  if (a.weights && tid == 0) a.lse[orow] = M + logf(L);
}

template <int D, int BITS>
__global__ __launch_bounds__(256) void paged_weights_kernel(PagedArgs a) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int32_t kh = blockIdx.y, g = a.H / a.pool.heads;
  const int64_t b = blockIdx.z;
  if (j >= visible_slots(a, b, a.T - 1)) return;
  const int64_t row = cache_row(a.pool, b, kh, j);
  if (row < 0) return;
  const uint8_t* kr = a.pool.k_codes + row * (D * BITS / 8);
  float sum = 0.0f;
  for (int32_t t = 0; t < a.T; ++t) {
    if (j >= visible_slots(a, b, t)) continue;
    for (int32_t i = 0; i < g; ++i) {
      const int64_t orow = (b * a.T + t) * a.H + kh * g + i;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot += a.rot[orow * D + d] * code_at<BITS>(kr, d);
      sum += expf(dot * a.pool.k_scale[row] * a.scale - a.lse[orow]);
    }
  }
  a.weights[(b * a.pool.heads + kh) * a.capacity + j] += sum;
}

using paged_fn = void (*)(PagedArgs);

template <int DT>
paged_fn pick_paged(int d, int bits) {
  if (d == 64) return bits == 8 ? paged_attention_kernel<DT, 64, 8> : paged_attention_kernel<DT, 64, 4>;
  return bits == 8 ? paged_attention_kernel<DT, 128, 8> : paged_attention_kernel<DT, 128, 4>;
}

paged_fn pick_weights(int d, int bits) {
  if (d == 64) return bits == 8 ? paged_weights_kernel<64, 8> : paged_weights_kernel<64, 4>;
  return bits == 8 ? paged_weights_kernel<128, 8> : paged_weights_kernel<128, 4>;
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" size_t aekv_paged_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t heads, int32_t d,
                                                      int64_t slots, int32_t tracked) {
  if (B <= 0 || T <= 0 || H <= 0 || heads <= 0 || d <= 0 || slots <= 0 || !tracked) return 0;
  return align_up(static_cast<size_t>(B * T * H) * 4, 16) + static_cast<size_t>(B * T * H) * d * 4;
}

extern "C" int aekv_paged_attention(const void* q, int32_t dtype, int64_t q_batch_stride, int64_t q_token_stride,
                                    int64_t q_head_stride, int64_t B, int64_t T, int64_t H, int32_t d, int32_t bits,
                                    const float* diag, const void* k_codes, const float* k_scale, const void* v_codes,
                                    const float* v_scale, int64_t pages, int64_t heads, int32_t page_size,
                                    const int32_t* page_table, int64_t max_pages, const int32_t* lengths,
                                    const float* sink, float* weights, int64_t capacity, float softmax_scale, void* ws,
                                    size_t ws_bytes, void* out, void* stream) {
  const char* who = "aekv_paged_attention";
  PagedArgs a{};
  if (const int rc = check_pool(who, const_cast<void*>(k_codes), const_cast<float*>(k_scale), const_cast<void*>(v_codes),
                                const_cast<float*>(v_scale), pages, heads, page_size, d, bits, page_table, max_pages, B,
                                &a.pool))
    return rc;
  if (dtype != AEKV_F16 && dtype != AEKV_BF16) return fail(AEKV_ERR_DTYPE, "%s: q must be F16 or BF16", who);
  if (T < 0 || H < 1 || H % heads)
    return fail(AEKV_ERR_SHAPE, "%s: T=%lld, and %lld query heads are no multiple of %lld KV heads", who, (long long)T,
                (long long)H, (long long)heads);
  if (weights && capacity < 0) return fail(AEKV_ERR_SHAPE, "%s: capacity=%lld", who, (long long)capacity);
  if (B == 0 || T == 0) return AEKV_OK;
  if (!q || !lengths || !diag || !out) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (!is_aligned(q, 16) || !is_aligned(out, 16) || !is_aligned(ws, 16) || (q_batch_stride % 8) || (q_token_stride % 8) ||
      (q_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q rows, out and workspace must be 16-byte aligned", who);
  if (B > 65535 || T > 65535 || H > 65535) return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld T=%lld H=%lld exceed the grid", who, (long long)B, (long long)T, (long long)H);
  const int64_t slots = max_pages * page_size;
  const size_t want = aekv_paged_attention_workspace_size(B, T, H, heads, d, slots, weights != nullptr);
  if (want && (!ws || ws_bytes < want)) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  a.q = q;
  a.q_batch = q_batch_stride;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.lengths = lengths;
  a.diag = diag;
  a.sink = sink;
  a.weights = slots > 0 ? weights : nullptr;
  a.lse = static_cast<float*>(ws);
  a.rot = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + align_up(static_cast<size_t>(B * T * H) * 4, 16));
  a.out = out;
  a.capacity = capacity;
  a.T = static_cast<int32_t>(T);
  a.H = static_cast<int32_t>(H);
  a.scale = softmax_scale;
  a.wscale = wht_scale(d);
  const hipStream_t st = as_stream(stream);
  auto fn = dtype == AEKV_F16 ? pick_paged<AEKV_F16>(d, bits) : pick_paged<AEKV_BF16>(d, bits);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(H), static_cast<uint32_t>(T), static_cast<uint32_t>(B)), dim3(256), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  if (!a.weights) return AEKV_OK;
  const int64_t reach = slots < capacity ? slots : capacity;
  if (reach == 0) return AEKV_OK;
  hipLaunchKernelGGL(pick_weights(d, bits), dim3(static_cast<uint32_t>(ceil_div(reach, 256)), static_cast<uint32_t>(heads), static_cast<uint32_t>(B)), dim3(256), 0, st, a);
  return check_launch(who);
}
