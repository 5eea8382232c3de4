// Rotary positions on several axes (time, height, width, ..), of q and k in one launch.
//
// Pair i of R has frequency f_i and axis a_i.  Token n, at position p[a, n] on axis a, turns it by t = p[a_i, n] f_i:
//   y1 = x1 cos t - x2 sin t,  y2 = x2 cos t + x1 sin t     (inverse: -t)
// where (x1, x2) are the dims first + 2 i and first + 2 i + 1 (adjacent), or first + i and first + R + i (halves); other dims
// stay as they are.  The angle is a product of an integer and an fp32 number, taken in fp64 (in fp32 it would be off by 2^-24
// of itself, 0.01 at position 200000), as are its cos and sin, which are rounded to fp32; the turned pair is fp32 with one rounding
// to x's type.
//
// A workgroup takes some tokens with all their heads, so that the heads share a token's cos and sin through LDS; its first
// loads are under way while those are made.  A thread holds whole pairs: V neighbouring dims (adjacent), or V dims and their
// partners (halves), so out may be x itself.
//
// Bound by reading and writing the rows: 32768 tokens of 12 + 4 heads of 128 in bf16, 268 MB in 50 us, 5.3 TB/s, where a copy of 256
// MiB reaches 5.5; 5003 tokens of 16 + 16 heads of 64 in fp32, 82 MB in 18 us.  64 tokens take 3.8 us, a launch.  Rows of a
// workgroup and units under way between half and twice these change no case by more than 5 %.
#include "aekv_common.h"

namespace aekv {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 2048;  // pairs with cos and sin in LDS

struct RotateArgs {
  const void* x[2];  // q, k
  void* y[2];
  int64_t x_token[2], x_head[2], y_token[2], y_head[2];  // strides in elements
  const void* pos;
  int64_t pos_axis, pos_token;  // strides
  const float* freq;            // [R]
  const int32_t* axis;          // [R], below the axes of pos
  int64_t n;
  int32_t heads[2], R, first, units, rotated;  // units: of a head; those below `rotated` hold pairs, the rest are copied
  int32_t block;                               // tokens of a workgroup
  int32_t wide;                                // pos is int64
  float sign;
};

template <int BYTES>
struct Word;
template <>
struct Word<4> {
  typedef uint32_t t;
};
template <>
struct Word<8> {
  typedef uint2 t;
};
template <>
struct Word<16> {
  typedef uint4 t;
};

// V elements of type DT, in memory order
template <int DT, int V>
struct Vec {
  static constexpr int kBytes = V * (DT == AEKV_F32 ? 4 : 2), kWord = kBytes > 16 ? 16 : kBytes, kWords = kBytes / kWord;
  typename Word<kWord>::t w[kWords];
  __device__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = static_cast<const typename Word<kWord>::t*>(p)[i];
  }
  __device__ void store(void* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) static_cast<typename Word<kWord>::t*>(p)[i] = w[i];
  }
  struct U32 {
    uint32_t u[kBytes / 4];
  };
  __device__ void get(float (&f)[V]) const {
    const U32 b = __builtin_bit_cast(U32, *this);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (DT == AEKV_F32) f[i] = __builtin_bit_cast(float, b.u[i]);
      else if constexpr (DT == AEKV_F16) f[i] = f16_to_f32((b.u[i / 2] >> (16 * (i % 2))) & 0xFFFFu);
      else f[i] = bf16_to_f32((b.u[i / 2] >> (16 * (i % 2))) & 0xFFFFu);
    }
  }
  __device__ void set(const float (&f)[V]) {
    U32 b;
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      if constexpr (DT == AEKV_F32) b.u[i] = __builtin_bit_cast(uint32_t, f[i]);
      else if constexpr (DT == AEKV_F16) b.u[i] = pack_f16x2(f[2 * i], f[2 * i + 1]);
      else b.u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
    *this = __builtin_bit_cast(Vec, b);
  }
};

// cos and sin of position * f: the angle less whole quarter turns, r, at most pi / 4, and the series of both, in fp64 and rounded
// once, but for the terms from r^5 / 120 and r^6 / 720 on, at most 2^-8.6, which fp32 gives to 2^-30.  (A whole angle up to pi in
// fp32 would be off by 2^-23; all terms in fp64 take a third more registers and a prompt's time from 57 to 63 us.)
__device__ __forceinline__ float2 turn(double p, float f) {
  constexpr double kQuarters = 0.6366197723675814, kHi = 1.5707963267948966, kLo = 6.123233995736766e-17;  // 2 / pi, pi / 2
  const double a = p * static_cast<double>(f), n = rint(a * kQuarters);
  const double r = fma(-n, kLo, fma(-n, kHi, a)), x = r * r;
  const float y = static_cast<float>(x);
  const float s5 = fmaf(fmaf(fmaf(-1.0f / 39916800.0f, y, 1.0f / 362880.0f), y, -1.0f / 5040.0f), y, 1.0f / 120.0f) * y;
  const float c6 = fmaf(fmaf(-1.0f / 3628800.0f, y, 1.0f / 40320.0f), y, -1.0f / 720.0f) * y;
  const float s = static_cast<float>(fma(r * x, s5 - 1.0 / 6.0, r)), c = static_cast<float>(fma(fma(c6 + 1.0 / 24.0, x, -0.5), x, 1.0));
  const double quarter = n - 4.0 * rint(0.25 * n);  // -2 .. 2
  const bool odd = fabs(quarter) == 1.0, half = fabs(quarter) == 2.0;
  const float cosine = odd ? s : c, sine = odd ? c : s;
  return make_float2(half || quarter == 1.0 ? -cosine : cosine, half || quarter == -1.0 ? -sine : sine);
}

template <int DT, int V, bool HALVES>
__global__ __launch_bounds__(kThreads) void rotate_axes_kernel(RotateArgs a) {
  constexpr int kElem = DT == AEKV_F32 ? 4 : 2;
  constexpr int kBatch = V * kElem * (HALVES ? 2 : 1) >= 32 ? 2 : 4;  // units a thread has under way
  __shared__ float2 table[kTable];
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * a.block;
  const int tokens = static_cast<int>(a.n - n0 < a.block ? a.n - n0 : a.block);
  const int per_token = (a.heads[0] + a.heads[1]) * a.units;
  const int total = tokens * per_token;
  bool ready = false;
  for (int base = 0; base < total; base += kThreads * kBatch) {
    Vec<DT, V> one[kBatch], two[kBatch];
    char* to[kBatch];
    int slot[kBatch], unit_of[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = base + i * kThreads + static_cast<int>(threadIdx.x);
      unit_of[i] = -1;
      if (at >= total) continue;
      const int token = at / per_token, in = at - token * per_token;
      int head = in / a.units;
      const int unit = in - head * a.units;
      const int which = head >= a.heads[0];
      head -= which ? a.heads[0] : 0;
      // the unit's first dim: pairs first, then what lies before them and (halves: the second halves are partners) behind
      int dim;
      if (unit < a.rotated) dim = a.first + unit * V;
      else if ((unit - a.rotated) * V < a.first) dim = (unit - a.rotated) * V;
      else dim = (unit - a.rotated) * V + 2 * a.R;
      const char* from = static_cast<const char*>(which ? a.x[1] : a.x[0]) +
                         kElem * ((n0 + token) * (which ? a.x_token[1] : a.x_token[0]) + head * (which ? a.x_head[1] : a.x_head[0]) + dim);
      to[i] = static_cast<char*>(which ? a.y[1] : a.y[0]) +
              kElem * ((n0 + token) * (which ? a.y_token[1] : a.y_token[0]) + head * (which ? a.y_head[1] : a.y_head[0]) + dim);
      one[i].load(from);
      unit_of[i] = unit;
      slot[i] = token * a.R + (HALVES ? unit * V : unit * (V / 2));
      if (HALVES && unit < a.rotated) two[i].load(from + kElem * a.R);
    }
    if (!ready) {
      for (int i = threadIdx.x; i < tokens * a.R; i += kThreads) {
        const int token = i / a.R, pair = i - token * a.R;
        const int64_t at = a.axis[pair] * a.pos_axis + (n0 + token) * a.pos_token;
        const double p = a.wide ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at]) : static_cast<double>(static_cast<const int32_t*>(a.pos)[at]);
        float2 cs = turn(p, a.freq[pair]);
        cs.y *= a.sign;
        table[i] = cs;
      }
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (unit_of[i] < 0) continue;
      if (unit_of[i] < a.rotated) {
        float x[V];
        one[i].get(x);
        if constexpr (HALVES) {
          float z[V], y1[V], y2[V];
          two[i].get(z);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 cs = table[slot[i] + j];
            y1[j] = fmaf(x[j], cs.x, -(z[j] * cs.y));
            y2[j] = fmaf(z[j], cs.x, x[j] * cs.y);
          }
          one[i].set(y1);
          two[i].set(y2);
          two[i].store(to[i] + kElem * a.R);
        } else {
          float y[V];
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 cs = table[slot[i] + j / 2];
            y[j] = fmaf(x[j], cs.x, -(x[j + 1] * cs.y));
            y[j + 1] = fmaf(x[j + 1], cs.x, x[j] * cs.y);
          }
          one[i].set(y);
        }
      }
      one[i].store(to[i]);
    }
  }
}

using rotate_fn = void (*)(RotateArgs);
template <int DT, int V>
rotate_fn pick_pairs(bool halves) {
  return halves ? rotate_axes_kernel<DT, V, true> : rotate_axes_kernel<DT, V, false>;
}
template <int DT>
rotate_fn pick_width(int v, bool halves) {
  return v == 8 ? pick_pairs<DT, 8>(halves) : v == 4 ? pick_pairs<DT, 4>(halves) : pick_pairs<DT, 2>(halves);
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" int aekv_rotate_axes(const void* q, const void* k, int32_t dtype, int64_t n, int32_t H, int32_t heads, int32_t d,
                                int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                const void* positions, int32_t pos_dtype, int32_t axes, int64_t pos_axis_stride,
                                int64_t pos_token_stride, const float* inv_freq, const int32_t* axis, int32_t pairs,
                                int32_t first, int32_t halves, int32_t inverse, void* q_out, void* k_out,
                                int64_t qo_token_stride, int64_t qo_head_stride, int64_t ko_token_stride,
                                int64_t ko_head_stride, void* stream) {
  const char* who = "aekv_rotate_axes";
  if (!is_float_dtype(dtype)) return fail(AEKV_ERR_DTYPE, "%s: q and k must be F32, F16 or BF16", who);
  if (pos_dtype != AEKV_I32 && pos_dtype != AEKV_I64) return fail(AEKV_ERR_DTYPE, "%s: positions must be I32 or I64", who);
  if (n < 0 || H < 0 || heads < 0 || H + static_cast<int64_t>(heads) < 1 || H + static_cast<int64_t>(heads) > 65535 || axes < 1)
    return fail(AEKV_ERR_SHAPE, "%s: n=%lld H=%d heads=%d axes=%d", who, (long long)n, H, heads, axes);
  if (d < 2 || d > 1024 || d % 2) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (even, up to 1024 supported)", who, d);
  if (pairs < 1 || first < 0 || first % 2 || first + 2 * static_cast<int64_t>(pairs) > d || (halves && pairs % 2))
    return fail(AEKV_ERR_VALUE, "%s: %d pairs from dim %d of %d (%s)", who, pairs, first, d, halves ? "halves: an even number" : "an even first dim");
  if (n == 0) return AEKV_OK;
  if ((H && (!q || !q_out)) || (heads && (!k || !k_out)) || !positions || !inv_freq || !axis) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  // the widest unit that the rows and dims allow: 16 bytes of 16-bit elements, 32 of fp32
  const size_t e = dtype_size(dtype);
  auto fits = [&](int v) {
    const size_t bytes = v * e > 16 ? 16 : v * e;
    auto rows = [&](const void* p, int64_t t, int64_t h, int32_t count) {
      return !count || (is_aligned(p, bytes) && t * static_cast<int64_t>(e) % static_cast<int64_t>(bytes) == 0 && h * static_cast<int64_t>(e) % static_cast<int64_t>(bytes) == 0);
    };
    return d % v == 0 && first % v == 0 && (halves ? pairs % v == 0 : 2 * pairs % v == 0) && rows(q, q_token_stride, q_head_stride, H) &&
           rows(k, k_token_stride, k_head_stride, heads) && rows(q_out, qo_token_stride, qo_head_stride, H) && rows(k_out, ko_token_stride, ko_head_stride, heads);
  };
  const int v = fits(8) ? 8 : fits(4) ? 4 : fits(2) ? 2 : 0;
  if (!v) return fail(AEKV_ERR_ALIGN, "%s: rows must be aligned to two elements", who);
  RotateArgs a{};
  a.x[0] = q, a.x[1] = k, a.y[0] = q_out, a.y[1] = k_out;
  a.x_token[0] = q_token_stride, a.x_head[0] = q_head_stride, a.x_token[1] = k_token_stride, a.x_head[1] = k_head_stride;
  a.y_token[0] = qo_token_stride, a.y_head[0] = qo_head_stride, a.y_token[1] = ko_token_stride, a.y_head[1] = ko_head_stride;
  a.pos = positions, a.pos_axis = pos_axis_stride, a.pos_token = pos_token_stride, a.wide = pos_dtype == AEKV_I64;
  a.freq = inv_freq, a.axis = axis, a.n = n, a.heads[0] = H, a.heads[1] = heads, a.R = pairs, a.first = first;
  a.sign = inverse ? -1.0f : 1.0f;
  a.rotated = halves ? pairs / v : 2 * pairs / v;
  // in place what is not turned is there already
  const bool in_place = (!H || (q == q_out && q_token_stride == qo_token_stride && q_head_stride == qo_head_stride)) &&
                        (!heads || (k == k_out && k_token_stride == ko_token_stride && k_head_stride == ko_head_stride));
  a.units = a.rotated + (in_place ? 0 : (d - 2 * pairs) / v);
  const int64_t per_token = (static_cast<int64_t>(H) + heads) * a.units;
  int64_t block = 1024 / per_token;
  if (block * pairs > kTable) block = kTable / pairs;
  if (block < 1) block = 1;
  if (n / block < 1024) block = ceil_div(n, 1024);  // (few tokens: one to a workgroup)
  a.block = static_cast<int32_t>(block);
  const int64_t blocks = ceil_div(n, block);
  if (blocks > kMaxGridThreads / kThreads) return fail(AEKV_ERR_UNSUPPORTED, "%s: %lld tokens exceed the grid", who, (long long)n);
  auto fn = dtype == AEKV_F32 ? pick_width<AEKV_F32>(v, halves) : dtype == AEKV_F16 ? pick_width<AEKV_F16>(v, halves) : pick_width<AEKV_BF16>(v, halves);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, as_stream(stream), a);
  return check_launch(who);
}
