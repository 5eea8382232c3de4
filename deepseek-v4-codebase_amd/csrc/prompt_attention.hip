// Causal attention over whole prompts: packed sequences of different lengths, grouped heads.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] and keys cu_k[b] .. cu_k[b + 1]; its i-th query sees its keys
// j <= i + (keys - queries), so that the last query sees every key (a chunk of a prompt comes with the keys before it).
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / (sum exp(scale q_i . k) + exp(sink)),  lse_i = log of that sum.
// A query that sees nothing gives 0 and a log sum of the sink's, or -inf.
#include "aekv_common.h"

namespace aekv {
namespace {

constexpr float kNegInf = -__builtin_inff();

struct PromptArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* cu_q;  // [B + 1]
  const int32_t* cu_k;  // [B + 1]
  const float* sink;    // [H] or null
  void* out;            // [n_q, H, D]
  float* lse;           // [n_q, H] or null
  int32_t n_q, n_k, B, H, heads;
  int32_t clear;        // rows behind the last sequence: 0 to leave out as it is, 1 to write zeros
  float scale;
};

template <int DT>
__device__ __forceinline__ float elem(const void* p, int64_t i) {
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return DT == AEKV_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
}

// One wave per (query, head): 64 keys at a time, a lane each for the logits, then a lane for D / 64 dims each.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_attention_kernel(PromptArgs a) {
  __shared__ float qs[4][D], ps[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (w >= static_cast<int64_t>(a.n_q) * a.H) return;
  const int32_t n = static_cast<int32_t>(w / a.H), h = static_cast<int32_t>(w - static_cast<int64_t>(n) * a.H);
  const int32_t kh = h / (a.H / a.heads);
  uint16_t* out = static_cast<uint16_t*>(a.out) + w * D;
  int lo = 0, hi = a.B;
  const bool in = n >= a.cu_q[0] && n < a.cu_q[a.B];
  while (in && hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= n) lo = mid;
    else hi = mid;
  }
  if (!in) {
    if (a.clear)
      for (int i = 0; i < D / 64; ++i) out[lane + 64 * i] = 0;
    if (a.lse && lane == 0) a.lse[w] = kNegInf;
    return;
  }
  const int64_t k0 = max(a.cu_k[lo], 0), k1 = min(a.cu_k[lo + 1], a.n_k);
  const int64_t seen = min<int64_t>(k1 - k0, n - a.cu_q[lo] + 1 + (k1 - k0) - (a.cu_q[lo + 1] - a.cu_q[lo]));
  for (int i = 0; i < D / 64; ++i) qs[wave][lane + 64 * i] = elem<DT>(a.q, n * a.q_token + h * a.q_head + lane + 64 * i);
  __builtin_amdgcn_wave_barrier();
  float m = kNegInf, l = 0.0f, o[D / 64];
  for (int i = 0; i < D / 64; ++i) o[i] = 0.0f;
  for (int64_t base = 0; base < seen; base += 64) {
    const int64_t j = base + lane;
    float s = kNegInf;
    if (j < seen) {
      const int64_t at = (k0 + j) * a.k_token + kh * a.k_head;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot += qs[wave][d] * elem<DT>(a.k, at + d);
      s = dot * a.scale;
    }
    const float m2 = fmaxf(m, wave_max(s));
    const float r = m2 == kNegInf ? 1.0f : expf(m - m2);
    const float p = s == kNegInf ? 0.0f : expf(s - m2);
    l = l * r + wave_sum(p);
    m = m2;
    ps[wave][lane] = p;
    __builtin_amdgcn_wave_barrier();
    for (int i = 0; i < D / 64; ++i) o[i] *= r;
    const int cnt = static_cast<int>(min<int64_t>(64, seen - base));
    for (int k = 0; k < cnt; ++k)
      for (int i = 0; i < D / 64; ++i) o[i] += ps[wave][k] * elem<DT>(a.v, (k0 + base + k) * a.v_token + kh * a.v_head + lane + 64 * i);
    __builtin_amdgcn_wave_barrier();
  }
  const float sk = a.sink ? a.sink[h] : kNegInf;
  const float M = fmaxf(m, sk);
  // (NaN alone leaves a maximum of -inf, and a sum that says so)
  const float f = l == 0.0f ? 0.0f : expf(m - M);
  const float L = (l == 0.0f ? 0.0f : l * f) + (sk == kNegInf ? 0.0f : expf(sk - M));
  for (int i = 0; i < D / 64; ++i) {
    const float y = L == 0.0f ? 0.0f : o[i] * f / L;
    out[lane + 64 * i] = DT == AEKV_BF16 ? static_cast<uint16_t>(pack_bf16x2(y, 0.0f)) : static_cast<uint16_t>(f32_to_f16_bits(y));
  }
  if (a.lse && lane == 0) a.lse[w] = L == 0.0f ? kNegInf : M + logf(L);
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" int aekv_prompt_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t q_token_stride,
                                     int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                     int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int64_t B, int64_t n_q, int64_t n_k, int64_t H,
                                     int64_t heads, int32_t d, const float* sink, float softmax_scale, void* out,
                                     float* lse, int32_t clear_rest, void* stream) {
  const char* who = "aekv_prompt_attention";
  if (dtype != AEKV_F16 && dtype != AEKV_BF16) return fail(AEKV_ERR_DTYPE, "%s: q, k and v must be F16 or BF16", who);
  if (d != 64 && d != 128) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128 supported)", who, d);
  if (B < 0 || n_q < 0 || n_k < 0 || heads < 1 || H < 1 || H % heads)
    return fail(AEKV_ERR_SHAPE, "%s: B=%lld n_q=%lld n_k=%lld, and %lld query heads are no multiple of %lld KV heads", who,
                (long long)B, (long long)n_q, (long long)n_k, (long long)H, (long long)heads);
  if (n_q == 0) return AEKV_OK;
  if (!q || !out || (B > 0 && (!cu_seqlens_q || !cu_seqlens_k)) || (n_k > 0 && (!k || !v)))
    return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (B == 0) return fail(AEKV_ERR_SHAPE, "%s: %lld queries in no sequence", who, (long long)n_q);
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) || (q_token_stride % 8) ||
      (q_head_stride % 8) || (k_token_stride % 8) || (k_head_stride % 8) || (v_token_stride % 8) || (v_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q, k and v rows and out must be 16-byte aligned", who);
  if (n_q > 0x7fffffff || n_k > 0x7fffffff || B > 0x7ffffffe || H > 65535 || n_q * H > kMaxGridThreads / 64 - 4)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld n_q=%lld n_k=%lld H=%lld exceed the grid", who, (long long)B,
                (long long)n_q, (long long)n_k, (long long)H);
  PromptArgs a{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
               cu_seqlens_q, cu_seqlens_k, sink, out, lse, static_cast<int32_t>(n_q), static_cast<int32_t>(n_k),
               static_cast<int32_t>(B), static_cast<int32_t>(H), static_cast<int32_t>(heads), clear_rest, softmax_scale};
  auto fn = dtype == AEKV_F16 ? (d == 64 ? prompt_attention_kernel<AEKV_F16, 64> : prompt_attention_kernel<AEKV_F16, 128>)
                              : (d == 64 ? prompt_attention_kernel<AEKV_BF16, 64> : prompt_attention_kernel<AEKV_BF16, 128>);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(ceil_div(n_q * H, 4))), dim3(256), 0, as_stream(stream), a);
  return check_launch(who);
}
