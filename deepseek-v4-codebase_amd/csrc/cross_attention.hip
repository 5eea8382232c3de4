// Attention of packed queries over all states of an encoder, whose length is another: no query waits for a state.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] (one query each where there is no cu_q) and reads the states e = states[b]
// (b without a list): keys and values cu_k[e] .. cu_k[e + 1], heads grouped over KV heads.
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / (sum exp(scale q_i . k) + exp(sink)),  lse_i = log of that sum.
// A query over no states gives 0 and a log sum of the sink's, or -inf.
//
// Rows.  The G heads of a KV head's group share its keys, and so do neighbouring sequences that read the same states (the answers
// to one input): a run's rows are (query, head), query-major, over all its sequences.  Runs end at multiples of 64 sequences.
// One pass: running maximum and sum, the output rescaled only where a maximum moved by more than kMargin.  The weights are rounded
// once to the input's 16 bits for their product with V, the sums of weights and of products are fp32: bf16 has fp32's range; fp16
// ends at 2^-24, so its weights are held 2^kLift higher, and all down to 2^-21 of the largest are normal numbers.
#include "attn_tile.h"

namespace aekv {
namespace {

constexpr int kTile = 64;       // keys of a tile (many rows)
constexpr int kPieceTiles = 8;  // least tiles of a piece of the keys
constexpr int kUnit = 128;      // keys that a workgroup takes at a time (few rows)
constexpr int kTable = 256;     // sequences of a launch (few rows)

struct CrossArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* cu_q;    // [B + 1] or null
  const int32_t* cu_k;    // [E + 1]
  const int32_t* states;  // [B] or null
  const float* sink;      // [H] or null
  uint16_t* out;          // [n_q, H, D]
  float* lse;             // [n_q, H] or null
  float* part;            // partial rows: reference, sum (log2 units), 2 pad, output
  int32_t* desc;          // few rows: [workgroups][8]
  int32_t n_q, n_k, B, E, H, heads, G;
  int32_t clear;          // rows in no sequence: 0 to leave out as it is, 1 to write zeros
  int32_t b0, nb;         // few rows: the launch's sequences
  int32_t n_split, tiles; // many rows
  float scale2;           // |softmax scale| * log2(e), not 0 (times a masked product of -inf it stays -inf); where the
  int32_t flip;           // scale is negative the queries' signs are flipped: a row's largest product is its largest logit.  Where
  uint32_t nan;           // it is NaN, 1 stands for it and the queries become NaN (0x7fff is one in both types; else 0)
};

struct Run {
  int32_t q0, lq, k0, lk;  // the run's queries and keys
};

__device__ __forceinline__ int32_t query_start(const CrossArgs& a, int32_t b) {
  const int32_t c = load_or(a.cu_q, b, a.q, b);
  return min(max(c, 0), a.n_q);  // (n_q H, with a tile's rows, fits 31 bits)
}

// Lane l's view of sequence b0 + l, l < n (b0 a multiple of 64): whether a run starts there, and that run.
__device__ __forceinline__ bool find_run(const CrossArgs& a, int32_t b0, int32_t n, int lane, Run* r) {
  const int32_t b = b0 + min(lane, n - 1);
  const int32_t state = load_or(a.states, b, a.q, b);
  const int32_t c0 = query_start(a, b), c1 = query_start(a, b + 1);
  const int32_t before = __shfl_up(state, 1);
  const bool head = lane < n && (lane == 0 || state != before);
  const uint64_t later = __builtin_amdgcn_ballot_w64(head) & ~((2ull << lane) - 1);
  const int last = (later ? __builtin_ctzll(later) : n) - 1;
  const int32_t end = __shfl(c1, last);
  const bool there = state >= 0 && state < a.E;
  const int32_t e = there ? state : 0;
  const int32_t d0 = a.E > 0 ? a.cu_k[e] : 0, d1 = a.E > 0 ? a.cu_k[e + 1] : 0;
  r->q0 = c0, r->lq = max(end - c0, 0);
  r->k0 = min(max(d0, 0), a.n_k), r->lk = there ? min(max(d1, r->k0), a.n_k) - r->k0 : 0;
  return head;
}

// Rows in no sequence: shared out over the workgroups.
__device__ __forceinline__ void clear_rest(const CrossArgs& a, int words_of_row, int threads) {
  if (!a.cu_q || !(a.clear || a.lse)) return;
  const int32_t s0 = min(max(a.cu_q[0], 0), a.n_q), s1 = min(max(a.cu_q[a.B], s0), a.n_q);
  const int64_t words = static_cast<int64_t>(s0 + a.n_q - s1) * a.H * words_of_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * threads) {
    const int64_t r = i / words_of_row, row = r < static_cast<int64_t>(s0) * a.H ? r : r + static_cast<int64_t>(s1 - s0) * a.H;
    if (a.clear) reinterpret_cast<uint32_t*>(a.out)[row * words_of_row + i % words_of_row] = 0;
    if (a.lse && i % words_of_row == 0) a.lse[row] = kNegInf;
  }
}

// A row's queries as a matrix operand's register: signs and NaN as the scale asks for.
__device__ __forceinline__ uint4 load_query(const CrossArgs& a, const uint16_t* p) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  return make_uint4((w.x ^ a.flip) | a.nan, (w.y ^ a.flip) | a.nan, (w.z ^ a.flip) | a.nan, (w.w ^ a.flip) | a.nan);
}

// Four dims (4 c ..) of one finished row, whose sum is relative to m.
template <int DT, int D>
__device__ __forceinline__ void finish(const CrossArgs& a, int64_t orow, int32_t h, int c, float m, float l, float4 o) {
  using E = Elem<DT>;
  const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
  const float up = fmaxf(m, sk);
  const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
  const float sum = (l == 0.0f ? 0.0f : l * f) + (sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - up));
  const float r = sum == 0.0f ? 0.0f : f / sum;
  *reinterpret_cast<uint2*>(a.out + orow * D + 4 * c) = make_uint2(E::pack(o.x * r, o.y * r), E::pack(o.z * r, o.w * r));
  if (a.lse && c == 0) a.lse[orow] = sum == 0.0f ? kNegInf : (up + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---- few rows ------------------------------------------------------------------------------------------------------
//
// Bound by reading the keys and values.  All tiles' units (kUnit keys of a KV head, for a tile of 16 NT rows) form one line, of
// which every workgroup takes an equal part, so that states of different lengths load the chip evenly; a tile that
// lies in several workgroups' parts is merged by a second kernel.  A wave takes 32 keys of a unit by itself: keys go straight to
// registers, values to its own part of LDS, both one unit ahead, and no wave waits for another before the tile's end.
//
// Matrix layout (v_mfma_f32_16x16x32: A lane l holds A[l % 16][8 (l / 16) + j], B lane l holds B[8 (l / 16) + j][l % 16], D lane
// l register v holds D[4 (l / 16) + v][l % 16]), g = l / 16:
//   S^T = K Q^T: m = key, n = row; two blocks of 16 keys.
//   O^T += V^T P^T: m = dim, n = row; lane group g holds keys 4 g + j and 16 + 4 g + j, its own scores.
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void cross_few_kernel(CrossArgs a) {
  using E = Elem<DT>;
  using v8 = typename E::v8;
  constexpr int kRow = 2 * D, kKS = D / 32, kMB = D / 16, kRT = 16 * NT;
  constexpr int kPer = 1024 / kRow, kLoads = 32 / kPer;  // rows of a staging load, loads of 32 rows
  __shared__ __align__(16) uint8_t V0[4][32 * kRow];
  __shared__ __align__(16) uint8_t V1[4][32 * kRow];
  __shared__ int32_t s_end[kTable], s_q0[kTable], s_lq[kTable], s_k0[kTable], s_lk[kTable];
  __shared__ int64_t s_sum[4];
  __shared__ float2 s_ml[4][kRT];
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  clear_rest(a, D / 2, 256);
  {
    Run r{};
    int64_t x = 0;
    const int32_t n = min(a.nb - 64 * wv, 64);
    if (n > 0 && find_run(a, a.b0 + 64 * wv, n, lane, &r))
      x = static_cast<int64_t>((r.lq * a.G + kRT - 1) / kRT) * a.heads * max((r.lk + kUnit - 1) / kUnit, 1);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(x, d);
      if (lane >= d) x += o;
    }
    if (lane == 63) s_sum[wv] = x;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x += w < wv ? s_sum[w] : 0;
      all += s_sum[w];
    }
    // (the launcher has checked that a line fits 31 bits; one that does not has offsets that are no prefix sums)
    s_end[tid] = all > 0x7fffffff ? 0 : static_cast<int32_t>(x);
    s_q0[tid] = r.q0, s_lq[tid] = r.lq, s_k0[tid] = r.k0, s_lk[tid] = r.lk;
    __syncthreads();
  }
  const int32_t total = __builtin_amdgcn_readfirstlane(s_end[kTable - 1]);
  const int32_t chunk = total / static_cast<int32_t>(gridDim.x) + (total % static_cast<int32_t>(gridDim.x) != 0);
  const int64_t from = static_cast<int64_t>(blockIdx.x) * chunk;
  const int32_t start = static_cast<int32_t>(from < total ? from : total);
  const int32_t stop = static_cast<int32_t>(from + chunk < total ? from + chunk : total);
  if (start >= stop) {
    if (tid == 0) a.desc[8 * blockIdx.x] = -1;
    return;
  }

  // staging: load i of 32 rows writes 1024 bytes, lane l at + 16 l, so lane l loads the chunk that the swizzle puts there
  const int key_in = 16 * lane / kRow, placed = (16 * lane % kRow) / 16;
  int voff[4];
  const int k_stride = static_cast<int>(a.k_token) * 2, v_stride = static_cast<int>(a.v_token) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) voff[i] = key_in * v_stride + 16 * (placed ^ swizzle<D>((kPer * i + key_in) & 15));
  const int koff = n16 * k_stride + 16 * g;
  int tA[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int key = 16 * e + 4 * g + (n16 >> 2), x = (n16 & 3) >> 1;
    tA[e] = key * kRow + ((x ^ swizzle<D>(key & 15)) << 4) + ((n16 & 1) << 3);
  }

  int32_t pos = start;
  while (pos < stop) {
    int32_t lo = 0, hi = a.nb - 1;  // the first run that ends behind pos
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      if (s_end[mid] > pos) hi = mid;
      else lo = mid + 1;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int32_t begin = __builtin_amdgcn_readfirstlane(lo ? s_end[lo - 1] : 0);
    const int32_t q0 = __builtin_amdgcn_readfirstlane(s_q0[lo]), n_rows = __builtin_amdgcn_readfirstlane(s_lq[lo]) * a.G;
    const int32_t k0 = __builtin_amdgcn_readfirstlane(s_k0[lo]), lk = __builtin_amdgcn_readfirstlane(s_lk[lo]);
    const int32_t units = max((lk + kUnit - 1) / kUnit, 1);
    const int32_t th = (pos - begin) / units, u0 = (pos - begin) - th * units;
    const int32_t head = th % a.heads, row0 = th / a.heads * kRT;
    const int32_t n = min(units - u0, stop - pos), u1 = u0 + n;
    if (pos == start && tid == 0) {
      int32_t* d = a.desc + 8 * blockIdx.x;
      d[0] = u0 > 0 ? pos - u0 : -1, d[1] = units, d[2] = q0, d[3] = n_rows, d[4] = row0, d[5] = head, d[6] = chunk;
    }

    v8 qb[NT][kKS];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int32_t row = min(row0 + 16 * t + n16, n_rows - 1), qi = row / a.G, h = head * a.G + (row - qi * a.G);
      const uint16_t* qp = a.q + static_cast<int64_t>(q0 + qi) * a.q_token + h * a.q_head + 8 * g;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) qb[t][ks] = __builtin_bit_cast(v8, load_query(a, qp + 32 * ks));
    }
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k + k0 * a.k_token + head * a.k_head);
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v + k0 * a.v_token + head * a.v_head);
    u32x4_t kr[2][2][kKS];
    // the wave's 32 keys of unit u, read through buffer resources whose range ends at the last key: rows past it are zero, as
    // is all of the unit past the part's last (every step has as many loads under way)
    auto load = [&](int32_t u, auto buf_c) __attribute__((always_inline)) {
      constexpr int buf = decltype(buf_c)::value;
      const int32_t at = u * kUnit + 32 * wv, left = u < u1 ? lk - at : 0;
      const int32_t m = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : left < 32 ? left : 32);  // (the clamp is a vector instruction)
      const int64_t base = m > 0 ? at : 0;
      const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kbase + base * k_stride), 0, m > 0 ? (m - 1) * k_stride + kRow : 0, kBufWord3);
      const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vbase + base * v_stride), 0, m > 0 ? (m - 1) * v_stride + kRow : 0, kBufWord3);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ks = 0; ks < kKS; ++ks) kr[buf][t][ks] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(krs, koff + 64 * ks, 16 * t * k_stride, 0));
      uint8_t* const dst = buf ? V1[wv] : V0[wv];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void_t*)(dst + 1024 * i), 16, voff[i & 3], kPer * i * v_stride, 0, 0);
    };
    float m[NT], l[NT];
    f32x4_t O[NT][kMB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kNegInf, l[t] = 0.0f;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) O[t][mb] = f32x4_t{};
    }
    auto step = [&](int32_t u, auto buf_c) __attribute__((always_inline)) {
      constexpr int buf = decltype(buf_c)::value;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other buffer's values have been read
      load(u + 1, std::integral_constant<int, buf ^ 1>{});
      if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");  // (8 loads of keys, 8 of values under way)
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      const int32_t at = u * kUnit + 32 * wv;
      if (at >= lk || u >= u1) return;
      const uint8_t* vt = buf ? V1[wv] : V0[wv];
      v8 pb[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4_t s[2];
        float top = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = f32x4_t{};
#pragma unroll
          for (int ks = 0; ks < kKS; ++ks) s[kb] = E::mma16(__builtin_bit_cast(v8, kr[buf][kb][ks]), qb[t][ks], s[kb]);
        }
        if (at + 32 > lk) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kb][i] = at + 16 * kb + 4 * g + i < lk ? s[kb][i] : kNegInf;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kb][i]);
        top = fmaxf(top, xor_lane<16>(top));
        top = fmaxf(top, xor_lane<32>(top)) * a.scale2;
        const bool moved = top - m[t] > kMargin + E::kLift;
        if (__builtin_amdgcn_ballot_w64(moved)) {
          const float to = top - E::kLift, r = moved ? __builtin_amdgcn_exp2f(m[t] - to) : 1.0f;
          l[t] *= r;
#pragma unroll
          for (int mb = 0; mb < kMB; ++mb) O[t][mb] *= r;
          m[t] = moved ? to : m[t];
        }
        float nm = m[t] == kNegInf ? 0.0f : -m[t], by = a.scale2;
        // beyond kFar the reference, which is a rounded logit, may lie further from the exact product than the exponentials
        // reach: there a row's logits are all rounded as the reference was
        const bool far = fabsf(m[t]) > kFar && m[t] > kNegInf;
        if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kb][i] = far ? s[kb][i] * a.scale2 + nm : s[kb][i];
          by = far ? 1.0f : by, nm = far ? 0.0f : nm;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], by, nm));
          l[t] += p[i];
        }
        pb[t] = __builtin_bit_cast(v8, make_uint4(E::pack(p[0], p[1]), E::pack(p[2], p[3]), E::pack(p[4], p[5]), E::pack(p[6], p[7])));
      }
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) {
        const i16x4_t x = read_tr16(vt + (tA[0] ^ (mb << 5))), y = read_tr16(vt + (tA[1] ^ (mb << 5)));
        const v8 w = __builtin_bit_cast(v8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int t = 0; t < NT; ++t) O[t][mb] = E::mma16(w, pb[t], O[t][mb]);
      }
    };
    load(u0, std::integral_constant<int, 0>{});
    asm volatile("" ::: "memory");
    int32_t u = u0;
    do {
      step(u, std::integral_constant<int, 0>{});
      step(u + 1, std::integral_constant<int, 1>{});
      u += 2;
    } while (u < u1);

    // the waves' states through their own buffers: row n16's four dims at 16 mb + 4 g, chunks swizzled by the row
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += xor_lane<16>(l[t]);
      l[t] += xor_lane<32>(l[t]);
      if (g == 0) s_ml[wv][16 * t + n16] = make_float2(m[t], l[t]);
      float* const w = reinterpret_cast<float*>(t ? V1[wv] : V0[wv]) + n16 * D;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) *reinterpret_cast<f32x4_t*>(w + 4 * ((4 * mb + g) ^ n16)) = O[t][mb];
    }
    __syncthreads();
    const bool whole = n == units;
    float* const part = a.part + (2 * static_cast<int64_t>(blockIdx.x) + (pos == start ? 0 : 1)) * kRT * (D + 4);
    for (int r = tid / (D / 4); r < kRT; r += 256 / (D / 4)) {
      const int c = tid % (D / 4), row = row0 + r;
      if (row >= n_rows) break;
      float2 ml[4];
      float up = kNegInf;
#pragma unroll
      for (int w = 0; w < 4; ++w) ml[w] = s_ml[w][r], up = fmaxf(up, ml[w].x);
      float sum = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (a state of nothing has a sum of 0; NaN alone leaves a maximum of -inf, and a sum that says so)
        const float f = ml[w].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[w].x - up);
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(r < 16 ? V0[w] : V1[w]) + (r & 15) * D + 4 * (c ^ (r & 15)));
        sum += ml[w].y == 0.0f ? 0.0f : ml[w].y * f;
        if (ml[w].y != 0.0f) o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
      }
      if (whole) {
        const int32_t qi = row / a.G, h = head * a.G + (row - qi * a.G);
        finish<DT, D>(a, static_cast<int64_t>(q0 + qi) * a.H + h, h, c, up, sum, o);
      } else {
        float* p = part + r * (D + 4);
        if (c == 0) *reinterpret_cast<float2*>(p) = make_float2(up, sum);
        *reinterpret_cast<float4*>(p + 4 + 4 * c) = o;
      }
    }
    __syncthreads();
    pos += n;
  }
}

// Merges the tiles that lie in several workgroups' parts: workgroup i has the tile across the i-th border, if that is its first.
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) void cross_few_merge_kernel(CrossArgs a) {
  constexpr int kRT = 16 * NT;
  const int32_t* d = a.desc + 8 * (blockIdx.x + 1);
  const int32_t tpos = d[0], units = d[1], q0 = d[2], n_rows = d[3], row0 = d[4], head = d[5], chunk = d[6];
  const int64_t before = static_cast<int64_t>(blockIdx.x) * chunk;
  if (tpos < 0 || tpos < before) return;
  const int32_t last = (tpos + units - 1) / chunk;  // workgroup of the tile's last unit
  const int c = threadIdx.x % (D / 4);
  for (int r = threadIdx.x / (D / 4); r < kRT; r += 256 / (D / 4)) {
    const int32_t row = row0 + r;
    if (row >= n_rows) break;
    float m = kNegInf, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int CH = 4;  // pieces whose loads go out together
    for (int32_t w0 = blockIdx.x; w0 <= last; w0 += CH) {
      float2 ml[CH];
      float4 x[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int32_t w = min(w0 + i, last);
        const int slot = w == static_cast<int32_t>(blockIdx.x) && tpos != before ? 1 : 0;
        const float* p = a.part + ((2 * static_cast<int64_t>(w) + slot) * kRT + r) * (D + 4);
        ml[i] = *reinterpret_cast<const float2*>(p);
        x[i] = *reinterpret_cast<const float4*>(p + 4 + 4 * c);
      }
      float up = m;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (w0 + i > last || ml[i].y == 0.0f) ml[i] = make_float2(kNegInf, 0.0f), x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (nothing seen)
        up = fmaxf(up, ml[i].x);
      }
      const float f0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
      l = l == 0.0f ? 0.0f : l * f0;
      o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float f = ml[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - up);
        l += ml[i].y == 0.0f ? 0.0f : ml[i].y * f;
        o.x = fmaf(x[i].x, f, o.x), o.y = fmaf(x[i].y, f, o.y), o.z = fmaf(x[i].z, f, o.z), o.w = fmaf(x[i].w, f, o.w);
      }
      m = up;
    }
    const int32_t qi = row / a.G, h = head * a.G + (row - qi * a.G);
    finish<DT, D>(a, static_cast<int64_t>(q0 + qi) * a.H + h, h, c, m, l, o);
  }
}

// ---- many rows -----------------------------------------------------------------------------------------------------
//
// A workgroup takes 32 WR consecutive rows, 32 per wave.  Tiles of 64 keys and values stream through two LDS buffers, loaded one
// tile ahead straight into LDS; with KS = 2 two waves share a row group and take half of every tile each, merged at the end.
// Few row tiles over many keys take the keys in pieces, merged by a second kernel.
//
// Matrix layout (v_mfma_f32_32x32x16: A lane l holds A[l % 32][8 (l / 32) + j], B lane l holds B[8 (l / 32) + j][l % 32],
// D lane l register v holds D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32]), h = l / 32:
//   S^T = K Q^T: m = key, n = row; a lane reads 16-byte chunks of its key's row.
//   O^T += V^T P^T: m = dim, n = row, k = key; lane h holds keys 16 c + 4 h + j and 16 c + 8 + 4 h + j of a 16-key chunk c,
//   its own scores, and V^T comes from the row-major tile through the transposing LDS load.
// LDS rows keep their 16-byte chunks XOR-swizzled by their key, so that both reads touch all banks once.

struct TileAt {
  Run run;
  int32_t row;  // the tile's first row
};

// The workgroup's `t`-th tile (tiles of `rows` rows, in the runs' order).  Sequence b, whose rows start at r, has the places from
// floor(r / rows) + b on: a run that starts there has at least as many as tiles, and there are rows / tiles + B in all.  Blocks of 64
// sequences are searched 64 to a memory round, then the block's runs.  False where the place has no tile.
__device__ __forceinline__ bool find_tile(const CrossArgs& a, int32_t t, int rows, int lane, TileAt* at) {
  int32_t lo = 0, hi = (a.B + 63) / 64;
  while (hi - lo > 1) {
    const int32_t step = (hi - lo + 63) / 64, k = lo + min(step * lane, hi - 1 - lo);
    const uint64_t from = __builtin_amdgcn_ballot_w64(t - query_start(a, 64 * k) * a.G / rows >= 64 * k && step * lane < hi - lo);
    if (!from) return false;  // before the first sequence
    lo += (63 - __builtin_clzll(from)) * step;
    hi = min(lo + step, hi);
  }
  const int32_t b0 = 64 * lo, n = min(a.B - b0, 64);
  Run r;
  const bool head = find_run(a, b0, n, lane, &r);
  const int32_t place = r.q0 * a.G / rows + b0 + lane;
  const uint64_t from = __builtin_amdgcn_ballot_w64(head && t >= place);
  if (!from) return false;
  const int l = 63 - __builtin_clzll(from);
  at->run.q0 = __builtin_amdgcn_readlane(r.q0, l);
  at->run.lq = __builtin_amdgcn_readlane(r.lq, l);
  at->run.k0 = __builtin_amdgcn_readlane(r.k0, l);
  at->run.lk = __builtin_amdgcn_readlane(r.lk, l);
  at->row = (t - __builtin_amdgcn_readlane(place, l)) * rows;
  return at->row < at->run.lq * a.G;
}

template <int DT, int D, int WR, int KS>
__global__ __launch_bounds__(64 * WR * KS) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void cross_many_kernel(CrossArgs a) {
  using E = Elem<DT>;
  using v8 = typename E::v8;
  constexpr int kWaves = WR * KS, kRows = 32 * WR, kRow = 2 * D, kTileBytes = kTile * kRow;
  constexpr int kKB = 2 / KS;              // 32-key blocks of a tile per wave
  constexpr int kPass = 1024 * kWaves;     // bytes that the workgroup stages at a time
  constexpr int kPasses = kTileBytes / kPass;
  constexpr int kMB = D / 32, kKSteps = D / 16;
  static_assert(KS == 1 || KS == 2, "a tile is two 32-key blocks");
  static_assert(kTileBytes % kPass == 0 && kPass % kRow == 0 && kPass / kRow % 8 == 0, "whole rows per pass, the swizzle repeats after two");
  // [K, V][key][swizzled chunks]: separate arrays, so that the compiler sees that loads into one buffer do not write what is
  // read from the other
  __shared__ __align__(16) uint8_t L0[2 * kTileBytes];
  __shared__ __align__(16) uint8_t L1[2 * kTileBytes];

  const int lane = threadIdx.x & 63, rl = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % WR, kh = wv / WR;
  clear_rest(a, D / 2, 64 * kWaves);
  // workgroups: KV heads innermost, then row tiles, then pieces of the keys
  const int32_t head = static_cast<int32_t>(blockIdx.x % a.heads);
  uint32_t index = blockIdx.x / a.heads;
  const int32_t split = static_cast<int32_t>(index / a.tiles);
  index -= split * a.tiles;
  TileAt at;
  if (!find_tile(a, static_cast<int32_t>(index), kRows, lane, &at)) return;  // (the whole workgroup)
  const int32_t q0 = at.run.q0, lk = at.run.lk, k0 = at.run.k0, n_rows = at.run.lq * a.G;
  const int all_tiles = (lk + kTile - 1) / kTile;
  const int per_piece = a.n_split > 1 ? max((all_tiles + a.n_split - 1) / a.n_split, kPieceTiles) : all_tiles;
  const int first_tile = min(split * per_piece, all_tiles), n_tiles = min(first_tile + per_piece, all_tiles);

  // rows past the last are computed as copies of it
  v8 qb[kKSteps];
  const int32_t w0 = at.row + 32 * wr, row = w0 + rl, own = row < n_rows ? row : n_rows - 1;
  const int32_t qi = own / a.G, h = head * a.G + (own - qi * a.G);
  const uint16_t* qp = a.q + static_cast<int64_t>(q0 + qi) * a.q_token + h * a.q_head + 8 * hh;
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) qb[ks] = __builtin_bit_cast(v8, load_query(a, qp + 16 * ks));

  // staging: pass c of wave wv writes bytes [kPass c + 1024 wv, + 1024) of a tile, lane l at + 16 l, so lane l loads the
  // chunk that the swizzle puts there
  const int lin = 1024 * wv + 16 * lane, key_in = lin / kRow, placed = (lin % kRow) / 16;
  int koff[2], voff[2];
  const int k_stride = static_cast<int>(a.k_token) * 2, v_stride = static_cast<int>(a.v_token) * 2;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int c = placed ^ swizzle<D>((kPass / kRow * p + key_in) & 15);
    koff[p] = key_in * k_stride + 16 * c;
    voff[p] = key_in * v_stride + 16 * c;
  }
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k + k0 * a.k_token + head * a.k_head);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v + k0 * a.v_token + head * a.v_head);
  // Tile `it`, read through buffer resources whose range ends at the last key: rows past it are zero and touch no memory
  auto load_tile = [&](int it, auto buf_c) __attribute__((always_inline)) {
    uint8_t* const dst = decltype(buf_c)::value ? L1 : L0;
    const int left = lk - it * kTile, n = left < 0 ? 0 : left < kTile ? left : kTile;
    const int64_t base = n > 0 ? static_cast<int64_t>(it) * kTile : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kbase + base * k_stride), 0, n > 0 ? (n - 1) * k_stride + kRow : 0, kBufWord3);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vbase + base * v_stride), 0, n > 0 ? (n - 1) * v_stride + kRow : 0, kBufWord3);
#pragma unroll
    for (int c = 0; c < kPasses; ++c)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void_t*)(dst + kPass * c + 1024 * wv), 16, koff[c & 1], kPass / kRow * c * k_stride, 0, 0);
#pragma unroll
    for (int c = 0; c < kPasses; ++c)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void_t*)(dst + kTileBytes + kPass * c + 1024 * wv), 16, voff[c & 1], kPass / kRow * c * v_stride, 0, 0);
  };

  // LDS byte offsets.  Row-chunk reads (K): key 32 kb + rl, chunk (2 ks + hh) ^ swizzle(rl): sA ^ 32 ks.  Transposing reads
  // (V, 16-lane group G = lane / 16, s = lane % 16): key 16 c + 8 e + 4 hh + s / 4, dims 32 mb + 16 (G % 2) + 4 (s % 4) ..,
  // i.e. chunk 4 mb + x with x = 2 (G % 2) + (s % 4) / 2, xor the swizzle of the key.
  const int sA = (32 * kKB * kh + rl) * kRow + ((hh ^ swizzle<D>(rl & 15)) << 4);
  int tA[2];
  {
    const int s16 = lane & 15, x = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = 8 * e + 4 * hh + (s16 >> 2);
      tA[e] = (32 * kKB * kh + key) * kRow + ((x ^ swizzle<D>(key)) << 4) + ((s16 & 1) << 3);
    }
  }

  float m = kNegInf, l = 0.0f;  // the reference that weights are relative to (a maximum less kLift), their sum
  f32x16_t O[kMB];
#pragma unroll
  for (int mb = 0; mb < kMB; ++mb) O[mb] = f32x16_t{};

  auto tile = [&](int it, const uint8_t* kt, auto masked_c) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_c)::value;
    const uint8_t* vt = kt + kTileBytes;
    f32x16_t s[kKB];
    float top = kNegInf;
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      s[kb] = f32x16_t{};
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks) {
        const v8 ka = __builtin_bit_cast(v8, *reinterpret_cast<const uint4*>(kt + 32 * kRow * kb + (sA ^ (ks << 5))));
        s[kb] = E::mma(ka, qb[ks], s[kb]);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        if constexpr (masked) s[kb][v] = it * kTile + 32 * kKB * kh + 32 * kb + 8 * (v >> 2) + 4 * hh + (v & 3) < lk ? s[kb][v] : kNegInf;
        top = fmaxf(top, s[kb][v]);
      }
    }
    top = fmaxf(top, xor_lane<32>(top)) * a.scale2;
    // (each row by itself: a row's bits do not depend on the others'; the difference, as m and a constant may round up)
    const bool moved = top - m > kMargin + E::kLift;
    if (__builtin_amdgcn_ballot_w64(moved)) {
      const float to = top - E::kLift, r = moved ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
      l *= r;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) O[mb] *= r;
      m = moved ? to : m;
    }
    float nm = m == kNegInf ? 0.0f : -m, by = a.scale2;
    const bool far = fabsf(m) > kFar && m > kNegInf;  // (as with few rows)
    if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kb][v] = far ? s[kb][v] * a.scale2 + nm : s[kb][v];
      by = far ? 1.0f : by, nm = far ? 0.0f : nm;
    }
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        p[v] = __builtin_amdgcn_exp2f(fmaf(s[kb][v], by, nm));
        l += p[v];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const v8 pb = __builtin_bit_cast(v8, make_uint4(E::pack(p[8 * c], p[8 * c + 1]), E::pack(p[8 * c + 2], p[8 * c + 3]),
                                                        E::pack(p[8 * c + 4], p[8 * c + 5]), E::pack(p[8 * c + 6], p[8 * c + 7])));
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb) {
          const uint8_t* vc = vt + (32 * kb + 16 * c) * kRow;
          const i16x4_t lo = read_tr16(vc + (tA[0] ^ (mb << 6))), hi = read_tr16(vc + (tA[1] ^ (mb << 6)));
          O[mb] = E::mma(__builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pb, O[mb]);
        }
      }
    }
  };
  auto step = [&](int it, auto buf_c) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value;
    __builtin_amdgcn_s_waitcnt(0);  // this wave's part of tile `it` has landed (the compiler does not track these loads)
    __syncthreads();                // every wave's, and the other buffer's readers are done
    if (it + 1 < n_tiles) load_tile(it + 1, std::integral_constant<int, buf ^ 1>{});
    const uint8_t* kt = buf ? L1 : L0;
    if ((it + 1) * kTile <= lk) tile(it, kt, std::false_type{});
    else tile(it, kt, std::true_type{});
  };
  if (first_tile < n_tiles) load_tile(first_tile, std::integral_constant<int, 0>{});
#pragma unroll 1
  for (int it = first_tile; it < n_tiles; it += 2) {
    step(it, std::integral_constant<int, 0>{});
    if (it + 1 < n_tiles) step(it + 1, std::integral_constant<int, 1>{});
  }
  l += xor_lane<32>(l);  // both halves' keys

  if constexpr (KS == 2) {  // the second key half's states into the first's, through the tile buffers
    static_assert(WR * kMB * 16 * 64 * 4 + WR * 2 * 64 * 4 <= 4 * kTileBytes, "the states fit both buffers");
    __syncthreads();
    constexpr int kPerState = kMB * 16 * 64, kFit = 2 * kTileBytes / 4;  // floats
    auto slot = [&](int i) -> float* { return i < kFit ? reinterpret_cast<float*>(L0) + i : reinterpret_cast<float*>(L1) + (i - kFit); };
    static_assert(kFit % 64 == 0, "a run of 64 floats lies in one buffer");
    const int base = wr * (kPerState + 128);
    if (kh == 1) {
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int v = 0; v < 16; ++v) slot(base + (mb * 16 + v) * 64)[lane] = O[mb][v];
      slot(base + kPerState)[lane] = m;
      slot(base + kPerState + 64)[lane] = l;
    }
    __syncthreads();
    if (kh == 1) return;
    const float m1 = slot(base + kPerState)[lane], l1 = slot(base + kPerState + 64)[lane];
    const float up = fmaxf(m, m1);
    // (a state of nothing has a sum of 0; NaN alone leaves a maximum of -inf, and a sum that says so)
    const float f0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up), f1 = l1 == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m1 - up);
    l = (l == 0.0f ? 0.0f : l * f0) + (l1 == 0.0f ? 0.0f : l1 * f1);
    m = up;
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int v = 0; v < 16; ++v) O[mb][v] = O[mb][v] * f0 + slot(base + (mb * 16 + v) * 64)[lane] * f1;
  }
  if (row >= n_rows) return;
  const int64_t orow = static_cast<int64_t>(q0 + qi) * a.H + h;
  if (a.n_split > 1) {
    float* p = a.part + (orow * a.n_split + split) * (D + 4);
    if (hh == 0) *reinterpret_cast<float2*>(p) = make_float2(m, l);
    if (first_tile < n_tiles) {  // (an empty piece's sum of 0 says that it has no output)
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(p + 4 + 32 * mb + 8 * i + 4 * hh) = make_float4(O[mb][4 * i], O[mb][4 * i + 1], O[mb][4 * i + 2], O[mb][4 * i + 3]);
    }
    return;
  }
#pragma unroll
  for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      finish<DT, D>(a, orow, h, 8 * mb + 2 * i + hh, m, l, make_float4(O[mb][4 * i], O[mb][4 * i + 1], O[mb][4 * i + 2], O[mb][4 * i + 3]));
}

// Merges the pieces of the rows: D / 4 lanes hold a row, 4 dims each.
template <int DT, int D>
__global__ __launch_bounds__(256) void cross_many_merge_kernel(CrossArgs a) {
  constexpr int PER = D / 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / PER) + threadIdx.x / PER;
  if (row >= static_cast<int64_t>(a.n_q) * a.H) return;
  const int32_t n = static_cast<int32_t>(row / a.H), h = static_cast<int32_t>(row - static_cast<int64_t>(n) * a.H);
  const int j = threadIdx.x % PER;
  const float* p = a.part + row * a.n_split * (D + 4);
  if (a.cu_q && (n < a.cu_q[0] || n >= a.cu_q[a.B])) return;  // in no sequence
  float m = kNegInf, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int CH = 4;  // pieces whose loads go out together
  for (int s0 = 0; s0 < a.n_split; s0 += CH) {
    float2 ml[CH];
    float4 x[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float* ps = p + min(s0 + c, a.n_split - 1) * (D + 4);
      ml[c] = *reinterpret_cast<const float2*>(ps);
      x[c] = *reinterpret_cast<const float4*>(ps + 4 + 4 * j);
    }
    float up = m;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (s0 + c >= a.n_split || ml[c].y == 0.0f) ml[c] = make_float2(kNegInf, 0.0f), x[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (nothing seen)
      up = fmaxf(up, ml[c].x);
    }
    const float f0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
    l = l == 0.0f ? 0.0f : l * f0;
    o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float f = ml[c].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[c].x - up);
      l += ml[c].y == 0.0f ? 0.0f : ml[c].y * f;
      o.x = fmaf(x[c].x, f, o.x), o.y = fmaf(x[c].y, f, o.y), o.z = fmaf(x[c].z, f, o.z), o.w = fmaf(x[c].w, f, o.w);
    }
    m = up;
  }
  finish<DT, D>(a, row, h, j, m, l, o);
}

using cross_fn = void (*)(CrossArgs);
template <int WR, int KS>
cross_fn pick_many(int32_t dtype, int32_t d) {
  if (dtype == AEKV_F16) return d == 64 ? cross_many_kernel<AEKV_F16, 64, WR, KS> : cross_many_kernel<AEKV_F16, 128, WR, KS>;
  return d == 64 ? cross_many_kernel<AEKV_BF16, 64, WR, KS> : cross_many_kernel<AEKV_BF16, 128, WR, KS>;
}
template <int NT>
cross_fn pick_few(int32_t dtype, int32_t d, bool merge) {
  if (merge) {
    if (dtype == AEKV_F16) return d == 64 ? cross_few_merge_kernel<AEKV_F16, 64, NT> : cross_few_merge_kernel<AEKV_F16, 128, NT>;
    return d == 64 ? cross_few_merge_kernel<AEKV_BF16, 64, NT> : cross_few_merge_kernel<AEKV_BF16, 128, NT>;
  }
  if (dtype == AEKV_F16) return d == 64 ? cross_few_kernel<AEKV_F16, 64, NT> : cross_few_kernel<AEKV_F16, 128, NT>;
  return d == 64 ? cross_few_kernel<AEKV_BF16, 64, NT> : cross_few_kernel<AEKV_BF16, 128, NT>;
}

struct CrossPlan {
  bool few;
  int64_t rows, groups;  // few: rows of a tile, workgroups of a launch
  int64_t tiles, split;  // many
};
CrossPlan plan_cross(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H, int64_t heads, int32_t d) {
  CrossPlan p{};
  const int64_t G = H / heads, rows = n_q * G, runs = E > 0 && E < B ? E : B;
  const int64_t each = ceil_div(rows, runs);
  p.few = each <= 32;
  if (p.few) {
    p.rows = each <= 16 ? 16 : 32;
    // units of a launch's line at most, in 31 bits
    const int64_t tiles = rows / p.rows + B, line = tiles * heads * ceil_div(n_k + kUnit, kUnit);
    if (tiles * heads < (int64_t(1) << 24) && line < 0x7fffffff) {
      p.groups = d == 64 ? 1024 : 512;
      if (p.groups > line) p.groups = line;
      return p;
    }
    p.few = false;
  }
  const int64_t resident = d == 64 ? 768 : 512;
  p.rows = heads * (rows / 128) >= resident ? 128 : 64;
  p.tiles = rows / p.rows + B;
  const int64_t sees = E > 0 ? n_k / E : 0, piece = kTile * kPieceTiles;
  const int64_t room = resident / (ceil_div(rows, p.rows) * heads), most = ceil_div(sees, piece);
  p.split = room < most ? room : most;
  if (p.split < 1) p.split = 1;
  return p;
}

}  // namespace
}  // namespace aekv

using namespace aekv;

static bool cross_fits(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H) {
  return n_q <= 0x7fffffff && n_k <= 0x7fff0000 && B <= 0x7ffffffe && E <= 0x7ffffffe && H <= 65535 && n_q * H <= 0x7fff0000;
}

extern "C" size_t aekv_cross_attention_workspace_size(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H, int64_t heads, int32_t d) {
  if (B <= 0 || E < 0 || n_q <= 0 || n_k < 0 || H <= 0 || heads <= 0 || (d != 64 && d != 128) || H % heads) return 0;
  if (!cross_fits(B, E, n_q, n_k, H)) return 0;  // (the call refuses it)
  const CrossPlan p = plan_cross(B, E, n_q, n_k, H, heads, d);
  if (p.few) return static_cast<size_t>(p.groups) * 32 + static_cast<size_t>(p.groups) * 2 * p.rows * (d + 4) * 4;
  return p.split > 1 ? static_cast<size_t>(n_q * H) * static_cast<size_t>(p.split) * (d + 4) * 4 : 0;
}

extern "C" int aekv_cross_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t q_token_stride,
                                    int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                    int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const int32_t* states, int64_t B, int64_t E, int64_t n_q,
                                    int64_t n_k, int64_t H, int64_t heads, int32_t d, const float* sink,
                                    float softmax_scale, void* out, float* lse, int32_t clear_rest, void* ws,
                                    size_t ws_bytes, void* stream) {
  const char* who = "aekv_cross_attention";
  if (dtype != AEKV_F16 && dtype != AEKV_BF16) return fail(AEKV_ERR_DTYPE, "%s: q, k and v must be F16 or BF16", who);
  if (d != 64 && d != 128) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128 supported)", who, d);
  if (B < 0 || E < 0 || n_q < 0 || n_k < 0 || heads < 1 || H < 1 || H % heads)
    return fail(AEKV_ERR_SHAPE, "%s: B=%lld E=%lld n_q=%lld n_k=%lld, and %lld query heads are no multiple of %lld KV heads", who,
                (long long)B, (long long)E, (long long)n_q, (long long)n_k, (long long)H, (long long)heads);
  if (n_q == 0) return AEKV_OK;
  if (!q || !out || (E > 0 && !cu_seqlens_k) || (n_k > 0 && (!k || !v))) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (B == 0) return fail(AEKV_ERR_SHAPE, "%s: %lld queries in no sequence", who, (long long)n_q);
  if (!cu_seqlens_q && n_q != B) return fail(AEKV_ERR_SHAPE, "%s: without offsets every sequence has one query, got %lld for %lld", who, (long long)n_q, (long long)B);
  if (!states && E != B) return fail(AEKV_ERR_SHAPE, "%s: %lld sequences and %lld states need a list", who, (long long)B, (long long)E);
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) || (q_token_stride % 8) ||
      (q_head_stride % 8) || (k_token_stride % 8) || (k_head_stride % 8) || (v_token_stride % 8) || (v_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q, k and v rows and out must be 16-byte aligned", who);
  if (!cross_fits(B, E, n_q, n_k, H))
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld E=%lld n_q=%lld n_k=%lld H=%lld exceed the grid", who, (long long)B, (long long)E,
                (long long)n_q, (long long)n_k, (long long)H);
  if (k_token_stride * 2 * kTile > 0x3fffffff || v_token_stride * 2 * kTile > 0x3fffffff || k_token_stride < 0 || v_token_stride < 0)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: token strides of %lld and %lld elements", who, (long long)k_token_stride, (long long)v_token_stride);
  const CrossPlan plan = plan_cross(B, E, n_q, n_k, H, heads, d);
  const size_t want = aekv_cross_attention_workspace_size(B, E, n_q, n_k, H, heads, d);
  if (want && (!ws || ws_bytes < want)) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  const bool none = softmax_scale != softmax_scale;
  CrossArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.q_token = q_token_stride, a.q_head = q_head_stride, a.k_token = k_token_stride, a.k_head = k_head_stride, a.v_token = v_token_stride, a.v_head = v_head_stride;
  a.cu_q = cu_seqlens_q, a.cu_k = cu_seqlens_k, a.states = states, a.sink = sink, a.out = static_cast<uint16_t*>(out), a.lse = lse;
  a.n_q = static_cast<int32_t>(n_q), a.n_k = static_cast<int32_t>(n_k), a.B = static_cast<int32_t>(B), a.E = static_cast<int32_t>(E);
  a.H = static_cast<int32_t>(H), a.heads = static_cast<int32_t>(heads), a.G = static_cast<int32_t>(H / heads), a.clear = clear_rest;
  a.scale2 = none ? 1.0f : fmaxf(fabsf(softmax_scale) * kLog2e, 0x1p-126f), a.flip = softmax_scale < 0.0f ? 0x80008000u : 0u, a.nan = none ? 0x7fff7fffu : 0u;
  const hipStream_t st = as_stream(stream);
  if (plan.few) {
    a.desc = static_cast<int32_t*>(ws);
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + plan.groups * 32);
    const uint32_t groups = static_cast<uint32_t>(plan.groups);
    for (int64_t b0 = 0; b0 < B; b0 += kTable) {
      a.b0 = static_cast<int32_t>(b0), a.nb = static_cast<int32_t>(B - b0 < kTable ? B - b0 : kTable);
      hipLaunchKernelGGL((plan.rows == 16 ? pick_few<1>(dtype, d, false) : pick_few<2>(dtype, d, false)), dim3(groups), dim3(256), 0, st, a);
      if (const int rc = check_launch(who)) return rc;
      if (groups == 1) continue;
      hipLaunchKernelGGL((plan.rows == 16 ? pick_few<1>(dtype, d, true) : pick_few<2>(dtype, d, true)), dim3(groups - 1), dim3(256), 0, st, a);
      if (const int rc = check_launch(who)) return rc;
    }
    return AEKV_OK;
  }
  if (plan.tiles * heads * plan.split > kMaxGridThreads / 256 || ceil_div(n_q * H, 256 / (d / 4)) > kMaxGridThreads / 256)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld n_q=%lld H=%lld exceed the grid", who, (long long)B, (long long)n_q, (long long)H);
  a.part = static_cast<float*>(ws), a.n_split = static_cast<int32_t>(plan.split), a.tiles = static_cast<int32_t>(plan.tiles);
  auto fn = plan.rows == 128 ? pick_many<4, 1>(dtype, d) : pick_many<2, 2>(dtype, d);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(plan.tiles * heads * plan.split)), dim3(256), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  if (plan.split == 1) return AEKV_OK;
  auto mg = dtype == AEKV_F16 ? (d == 64 ? cross_many_merge_kernel<AEKV_F16, 64> : cross_many_merge_kernel<AEKV_F16, 128>)
                              : (d == 64 ? cross_many_merge_kernel<AEKV_BF16, 64> : cross_many_merge_kernel<AEKV_BF16, 128>);
  hipLaunchKernelGGL(mg, dim3(static_cast<uint32_t>(ceil_div(n_q * H, 256 / (d / 4)))), dim3(256), 0, st, a);
  return check_launch(who);
}
