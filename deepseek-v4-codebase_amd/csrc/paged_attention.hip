// Attention of a sequence's newest tokens over its paged per-head cache in TurboQuant codes.
//
// Token t (of T, the last T slots of each sequence) of query head h sees slots j < lengths[b] - T + 1 + t of KV head
// h / (H / heads), as far as the table, or the tracker, reaches:  l_j = scale q . K_j,  p_j = exp(l_j) / (sum exp(l) + exp(sink_h)),  out = sum_j p_j V_j.
// With the codec's orthogonal rotation R = c Had diag (K_j = s_j R^T codes_j) both products stay in the rotated domain:
//   q . K_j = s_j (R q) . codes_j        sum_j p_j V_j = R^T sum_j p_j s_j codes_j
// so a query is rotated once, an output is rotated back once, and a cached row costs its codes and one scale: the kernel
// is bound by reading them, 2 (D bits / 8 + 4) bytes per slot and KV head.
//
// Work split.  The T tokens x G heads of a KV head's group are rows; a workgroup takes 16 MT of them and one piece of the
// sequence, its four waves alternate over steps of 32 slots, and their states are merged through LDS.  Where a launch has
// too few workgroups the sequence is split over n_split pieces, merged by a second kernel.  One pass: running maximum and
// sum, the output rescaled only where a row's maximum moved by more than kMargin.
//
// Loads.  A wave's steps go straight into LDS, each wave in a ring of its own of three stages (two where a row has 128
// bytes, so that two workgroups stay on a CU), the next ones requested before a step is waited for: with the loads in
// registers a CU held one step of each wave (one sequence of 262144 slots, 12 heads: 120 us, staged 109).  The queries and
// the first steps are requested before the rotation runs.
//
// Measured (dim 128, 4 bits).  One sequence of 262144 slots, 12 heads of 12: 428 MB in 87 to 91 us, 4.7 to 4.9 TB/s, what a
// large copy reaches (5.0), with the merge 96 us.  64 ragged sequences of up to 16384 slots, 12 heads of 4, tracked: 75 us,
// the merge and the weights' sum 13 (a form with 40 of a step's 222 vector instructions less took as long).  16 tokens x 8
// heads of 8 sequences of up to 5001 slots, dim 64, 8 bits: 20 us, the rotations, four steps behind one another in each
// wave, and the merge of the waves.
//
// Matrix layout (v_mfma_f32_16x16x32: A lane l holds A[l % 16][8 (l / 16) + j], B lane l holds B[8 (l / 16) + j][l % 16],
// D lane l register i holds D[4 (l / 16) + i][l % 16]), g = l / 16:
//   S^T = K Q^T: m = slot, n = row.  The order of the dims within a product is free, so a lane reads the D / 4 contiguous
//     codes [g D / 4, (g + 1) D / 4) of its slot and product c takes 8 of them; the query has them in the same places.
//     The codes are exact in fp16; the rotated query, scaled to the top of fp16's range, goes in as two fp16 parts (22
//     bits), so that a logit has fp32's accuracy, which the accumulated weights need.
//   O^T += V^T P^T: m = dim, n = row, k = slot: lane g holds slots 4 g + i and 16 + 4 g + i, exactly the slots of its own
//     scores, so the weights need no data movement.  A lane reads the D / 16 codes of dims [n D / 16, ..) of those eight
//     slots, and product e takes one dim of each: the transpose is within the lane.  The weights, times their slots'
//     scales, go in as two bf16 parts (17 bits; the scales' range is fp32's, which fp16 has not), the codes as bf16 with
//     an offset that makes them one bit operation each; a product with ones gives the sum that takes the offset out.
//   A lane ends with D / 4 contiguous dims of one row, so both rotations are D / 4-point butterflies in the lane and two
//   exchanges between lanes.
#include <type_traits>

#include "paged_cache.h"
#include "tq_device.h"

namespace aekv {
namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMargin = 8.0f;  // log2 units: a row's maximum moves when it is exceeded by this (weights up to 2^8)
constexpr int kWaves = 4, kThreads = 64 * kWaves, kStep = 32, kRound = kStep * kWaves;

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

struct PagedArgs {
  PagePool pool;
  const void* q;
  int64_t q_batch, q_token, q_head;  // strides in elements
  const int32_t* lengths;            // [B]
  const float* diag;
  const float* sink;                 // [H] or null
  float* weights;                    // [B, heads, capacity] or null
  float* lse;                        // [B, T, H], log2 units, inf for a sum of 0 (with weights)
  float* logits;                     // [B, heads, rows, logit_slots], log2 units, -inf where hidden; or null
  float* part;                       // [B, T, H, n_split, D + 4]: max, sum (log2 units), 2 pad, rotated output
  void* out;                         // [B, T, H, D]
  int32_t reach;                     // slots of a sequence that can be seen: the table's, or the tracker's capacity
  int64_t capacity, logit_slots;
  int32_t T, H, G, rows, row_blocks, n_split;
  int32_t B, ranked;                 // workgroups by their sequences' lengths: 1 up to 64 of them, 2 up to kRanked; 0: by index
  float scale2, wscale;              // softmax scale * log2(e), fp32(D^-1/2)
};

// Slots of sequence b that its last token sees.
__device__ __forceinline__ int32_t newest_sees(const PagedArgs& a, int64_t b) { return max(min(a.lengths[b], a.reach), 0); }
// Of its n such slots those that token `tok` of the T newest sees.  The causal bound counts back from the given length, which
// may lie past what can be reached; that is cut off afterwards.
__device__ __forceinline__ int32_t token_sees(const PagedArgs& a, int32_t length, int32_t n, int32_t tok) {
  return min(max(length - (a.T - 1 - tok), 0), n);  // (length >= 0: nothing overflows)
}
// The sequence that comes r-th when the longest come first, by eighths of a power of two, equal ones by their index; *n: its
// slots.  The r-th largest key bit by bit, then its holder; a lane holds a sequence of each CH.
template <int CH>
__device__ __forceinline__ int32_t ranked_sequence(const PagedArgs& a, int32_t r, int lane, int32_t* n) {
  int32_t len[CH], key[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int32_t b = 64 * c + lane;
    len[c] = newest_sees(a, min(b, a.B - 1));
    // 1 + 8 times the exponent and 3 bits of the length + 1, below 256 (31 exponents); 0 past the last sequence
    key[c] = b < a.B ? 1 + static_cast<int32_t>((__builtin_bit_cast(uint32_t, static_cast<float>(len[c] + 1)) >> 20) - (127u << 3)) : 0;
  }
  auto count = [&](int32_t least) __attribute__((always_inline)) {
    int m = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) m += __popcll(__builtin_amdgcn_ballot_w64(key[c] >= least));
    return m;
  };
  int32_t v = 0;
#pragma unroll
  for (int bit = 128; bit > 0; bit >>= 1)
    if (count(v | bit) > r) v |= bit;
  int k = r - count(v + 1);
  int32_t b = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(key[c] == v);
    const uint64_t it = __builtin_amdgcn_ballot_w64(key[c] == v && __popcll(eq & ((1ull << lane) - 1)) == k);
    if (it) {
      const int at = __builtin_ctzll(it);
      b = 64 * c + at, *n = __builtin_amdgcn_readlane(len[c], at);
    }
    k -= __popcll(eq);
  }
  return b;
}

// The piece length of a sequence of n slots: whole rounds of the workgroup's waves.
__device__ __forceinline__ int32_t piece_slots(int32_t n, int32_t n_split) {
  const int32_t per = (n + n_split - 1) / n_split;
  return max((per + kRound - 1) / kRound * kRound, kRound);
}

// Butterflies of a vector whose dims [g D / 4, (g + 1) D / 4) this lane holds (g = lane / 16).
template <int N>
__device__ __forceinline__ void rotate_lane(float (&a)[N], int lane) {
#pragma unroll
  for (int h = 1; h < N; h <<= 1)
#pragma unroll
    for (int blk = 0; blk < N; blk += 2 * h)
#pragma unroll
      for (int i = 0; i < h; ++i) {
        const float x = a[blk + i], y = a[blk + h + i];
        a[blk + i] = x + y;
        a[blk + h + i] = x - y;
      }
  const float s16 = (lane & 16) ? -1.0f : 1.0f, s32 = (lane & 32) ? -1.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = fmaf(a[i], s16, xor_lane<16>(a[i]));
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = fmaf(a[i], s32, xor_lane<32>(a[i]));
}

// Place of element j of a product's operand among its 8 codes: the order in which unpacking a word of nibbles leaves them
// (halves of a register hold nibbles i and i + 4), or that of the bytes.
template <int BITS>
constexpr int code_place(int j) {
  return BITS == 4 ? (j & 1) * 4 + (j >> 1) : j;
}

// 8 codes as exact fp16.  Nibbles in two's complement: xor 8 makes them 0 .. 15, 0x6400 | u is 1024 + u and 0x6400 | 16 u
// is 1024 + 16 u in fp16; bytes likewise, offset by 128.
template <int BITS>
__device__ __forceinline__ f16x8_t codes_f16(const uint32_t* w) {
  uint4 r;
  if constexpr (BITS == 4) {
    const f16x2_t off = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
    const f16x2_t off16 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
    const f16x2_t s16 = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const uint32_t v = w[0], u = w[0] >> 8;
    r.x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, (v & 0x000F000Fu) ^ 0x64086408u) + off);
    r.y = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (v & 0x00F000F0u) ^ 0x64806480u), s16, off16));
    r.z = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, (u & 0x000F000Fu) ^ 0x64086408u) + off);
    r.w = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (u & 0x00F000F0u) ^ 0x64806480u), s16, off16));
  } else {
    const f16x2_t off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const uint32_t v = w[0] ^ 0x80808080u, u = w[1] ^ 0x80808080u;
    auto two = [&](uint32_t x, uint32_t sel) {  // bytes (b, 0x64, b', 0x64)
      return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, sel)) + off);
    };
    r.x = two(v, 0x07010700u);
    r.y = two(v, 0x07030702u);
    r.z = two(u, 0x07010700u);
    r.w = two(u, 0x07030702u);
  }
  return __builtin_bit_cast(f16x8_t, r);
}

template <int D, int BITS>
struct PagedGeom {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kKB = kRowBytes / 4;   // bytes of a slot's K row per lane
  static constexpr int kKW = kKB / 4;         // words
  static constexpr int kVB = kRowBytes / 16;  // bytes of a slot's V row per lane (2, 4 or 8)
  static constexpr int kNC = D / 32;          // K products per 16 slots
  static constexpr int kNE = D / 16;          // V products per 32 slots: codes per lane and slot
  static constexpr int kWords = kVB > 4 ? 2 : 1;
  // what the bf16 form of a code is more than the code: 16 + 8 for nibbles (0x4180 | 8 u is 16 + u), 128 for bytes
  static constexpr float kBias = BITS == 4 ? 24.0f : 128.0f;
};

// What a step of 32 slots loads.
template <int D, int BITS>
struct StepData {
  using G = PagedGeom<D, BITS>;
  uint32_t k[2][G::kKW];
  f32x4_t ks[2], vs[2];
  uint32_t v[8][G::kWords];
};

// The wave's page ids: lane 2 i + k holds that of tile k (16 slots) of its i-th step from `first`; -1 where a tile has none.
// (What the table says past the sequence's end does not matter: those slots are hidden.)
__device__ __forceinline__ int32_t load_pages(const PagedArgs& a, int64_t b, int32_t first, int lane) {
  const int64_t slot = static_cast<int64_t>(first) + kRound * (lane >> 1) + 16 * (lane & 1);
  int32_t page = -1;
  if (slot < a.reach) page = a.pool.table[b * a.pool.max_pages + (slot >> a.pool.page_shift)];
  return page >= 0 && page < a.pool.pages ? page : -1;
}

// A step's K codes and scales.
template <int D, int BITS>
__device__ __forceinline__ void load_keys(const PagedArgs& a, int32_t kh, int32_t slot, int32_t p0, int32_t p1, int lane,
                                          StepData<D, BITS>& s) {
  using G = PagedGeom<D, BITS>;
  const int n = lane & 15, g = lane >> 4;
  const int32_t in_page = (1 << a.pool.page_shift) - 1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int32_t page = k ? p1 : p0;  // wave-uniform
    // (a tile without a page reads the pool's first row, and is masked)
    const int64_t row = page < 0 ? 0 : ((static_cast<int64_t>(page) * a.pool.heads + kh) << a.pool.page_shift) + ((slot + 16 * k) & in_page);
    const uint8_t* kr = a.pool.k_codes + row * G::kRowBytes + (n * G::kRowBytes + g * G::kKB);
    if constexpr (G::kKW == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(kr);
      s.k[k][0] = w.x, s.k[k][1] = w.y;
    } else {
#pragma unroll
      for (int i = 0; i < G::kKW / 4; ++i) {
        const uint4 w = reinterpret_cast<const uint4*>(kr)[i];
        s.k[k][4 * i] = w.x, s.k[k][4 * i + 1] = w.y, s.k[k][4 * i + 2] = w.z, s.k[k][4 * i + 3] = w.w;
      }
    }
    s.ks[k] = *reinterpret_cast<const f32x4_t*>(a.pool.k_scale + row + 4 * g);
  }
}

// A step of 32 slots on its way into LDS, straight from memory.  K: unit l (16 bytes) of a load is what lane l will read.
// V: the rows (slots 16 k + 4 g + i) in the order (k, i, g), so that a lane's word of its slots 16 k + 4 g + i lies at
// 4 k + i rows of 64 lanes' words: every read is one run of the lanes.  Scales: K's 32, then V's.
template <int D, int BITS>
struct Stage {
  using G = PagedGeom<D, BITS>;
  static constexpr int kHalf = 32 * G::kRowBytes;    // K's bytes, and V's
  static constexpr int kBytes = 2 * kHalf + 256;
  static constexpr int kLoads = 2 * (kHalf / 1024) + 1;  // load instructions of a step
  static constexpr int kStages = G::kRowBytes == 128 ? 2 : 3;
};

typedef __attribute__((address_space(3))) void lds_void_t;
typedef const __attribute__((address_space(1))) void global_void_t;
// 16 (4) bytes per lane from each lane's own address to `to` and on, lane after lane.
__device__ __forceinline__ void load_lds16(const void* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_void_t*)from, (lds_void_t*)to, 16, 0, 0);
}
__device__ __forceinline__ void load_lds4(const void* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_void_t*)from, (lds_void_t*)to, 4, 0, 0);
}

// Issues a step's loads; p0 and p1 are its tiles' pages (a tile without one reads the pool's first rows, and is masked).
template <int D, int BITS>
__device__ __forceinline__ void issue_step(const PagedArgs& a, int32_t kh, int32_t slot, int32_t p0, int32_t p1, int lane, uint8_t* st) {
  using S = Stage<D, BITS>;
  constexpr int RB = PagedGeom<D, BITS>::kRowBytes;
  const int32_t in_page = (1 << a.pool.page_shift) - 1;
  const int64_t r0 = p0 < 0 ? 0 : ((static_cast<int64_t>(p0) * a.pool.heads + kh) << a.pool.page_shift) + (slot & in_page);
  const int64_t r1 = p1 < 0 ? 0 : ((static_cast<int64_t>(p1) * a.pool.heads + kh) << a.pool.page_shift) + ((slot + 16) & in_page);
  const int n = lane & 15, g = lane >> 4;
  if constexpr (RB == 32) {  // both tiles in one load: 2 units a row
    const int64_t row = lane < 32 ? r0 : r1;
    const int u = lane & 31;
    load_lds16(a.pool.k_codes + row * RB + 16 * u, st);
    // LDS row R = u / 2 of the tile is slot 4 (R % 4) + R / 4
    load_lds16(a.pool.v_codes + row * RB + (4 * ((u >> 1) & 3) + (u >> 3)) * RB + 16 * (u & 1), st + S::kHalf);
  } else {
    constexpr int PER = RB / 64;  // loads of a tile
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int q = 0; q < PER; ++q)
        load_lds16(a.pool.k_codes + (k ? r1 : r0) * RB + (n * RB + g * (RB / 4) + 16 * q), st + 1024 * (PER * k + q));
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int u = 64 * q + lane, R = u / (RB / 16);
        load_lds16(a.pool.v_codes + (k ? r1 : r0) * RB + ((4 * (R & 3) + (R >> 2)) * RB + 16 * (u % (RB / 16))), st + S::kHalf + 1024 * (PER * k + q));
      }
  }
  const int64_t row = ((lane & 16) ? r1 : r0) + n;
  load_lds4((lane < 32 ? a.pool.k_scale : a.pool.v_scale) + row, st + 2 * S::kHalf);
}

// Reads a landed step back.
template <int D, int BITS>
__device__ __forceinline__ void read_step(const uint8_t* st, int lane, StepData<D, BITS>& s) {
  using G = PagedGeom<D, BITS>;
  using S = Stage<D, BITS>;
  const int n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (G::kKW == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(st + 512 * k + 32 * n + 8 * g);
      s.k[k][0] = w.x, s.k[k][1] = w.y;
    } else {
#pragma unroll
      for (int i = 0; i < G::kKW / 4; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(st + 1024 * (G::kKW / 4 * k + i) + 16 * lane);
        s.k[k][4 * i] = w.x, s.k[k][4 * i + 1] = w.y, s.k[k][4 * i + 2] = w.z, s.k[k][4 * i + 3] = w.w;
      }
    }
    s.ks[k] = *reinterpret_cast<const f32x4_t*>(st + 2 * S::kHalf + 64 * k + 16 * g);
    s.vs[k] = *reinterpret_cast<const f32x4_t*>(st + 2 * S::kHalf + 128 + 64 * k + 16 * g);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint8_t* vr = st + S::kHalf + 64 * G::kVB * j + G::kVB * lane;
    if constexpr (G::kVB == 2) s.v[j][0] = *reinterpret_cast<const uint16_t*>(vr);
    else if constexpr (G::kVB == 4) s.v[j][0] = *reinterpret_cast<const uint32_t*>(vr);
    else {
      const uint2 w = *reinterpret_cast<const uint2*>(vr);
      s.v[j][0] = w.x, s.v[j][1] = w.y;
    }
  }
}

// Waits until at most N of the wave's memory operations are on their way (its loads land in order).  The empty asm keeps
// the LDS reads that follow from moving up.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));  // vmcnt alone
  asm volatile("" ::: "memory");
}

// Dim e of the eight slots as bf16 with the offset kBias.
template <int D, int BITS>
__device__ __forceinline__ bf16x8_t values_bf16(const uint32_t (&v)[8][PagedGeom<D, BITS>::kWords], int e) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BITS == 4) {
      // half-words of two slots side by side, then the nibble moved to the mantissa's top bits
      const uint32_t t = __builtin_amdgcn_perm(v[2 * i + 1][0], v[2 * i][0], (e & 4) ? 0x07060302u : 0x05040100u);
      const int place = 4 * (e & 3);
      const uint32_t m = place == 0 ? t << 3 : t >> (place - 3);
      r[i] = (m & 0x00780078u) ^ 0x41C041C0u;  // 0x4180 | (n ^ 8) << 3
    } else {
      const uint32_t x = v[2 * i][e >> 2], y = v[2 * i + 1][e >> 2];
      const int sh = 8 * (e & 3);
      r[i] = pack_bf16x2(static_cast<float>((x >> sh) & 255u), static_cast<float>((y >> sh) & 255u));
    }
  }
  return __builtin_bit_cast(bf16x8_t, make_uint4(r[0], r[1], r[2], r[3]));
}

// A row's query as it lies in memory: this lane's D / 4 elements (a row past the last reads the first).
template <int D>
__device__ __forceinline__ void load_query(const PagedArgs& a, int64_t b, int32_t kh, int32_t row, bool in, int lane, uint4 (&w)[D / 32]) {
  const int32_t t = in ? row / a.G : 0, h = kh * a.G + (in ? row - t * a.G : 0);
  const uint4* qp = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (b * a.q_batch + t * a.q_token + h * a.q_head + (lane >> 4) * (D / 4)));
#pragma unroll
  for (int i = 0; i < D / 32; ++i) w[i] = qp[i];
}

// A row's query, rotated, in two fp16 parts in the products' order; *factor takes a score to a logit in log2 units.
template <int DT, int D, int BITS>
__device__ __forceinline__ void query_parts(const PagedArgs& a, const uint4 (&qw)[D / 32], bool in, int lane,
                                            f16x8_t (&hi)[D / 32], f16x8_t (&lo)[D / 32], float* factor) {
  constexpr int N = D / 4;
  const int g = lane >> 4;
  float x[N];
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const uint32_t u[4] = {qw[i].x, qw[i].y, qw[i].z, qw[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * i + 2 * j] = DT == AEKV_BF16 ? bf16_to_f32(u[j] & 0xffffu) : f16_to_f32(u[j] & 0xffffu);
      x[8 * i + 2 * j + 1] = DT == AEKV_BF16 ? bf16_to_f32(u[j] >> 16) : f16_to_f32(u[j] >> 16);
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const f32x4_t d = *reinterpret_cast<const f32x4_t*>(a.diag + g * N + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * i + j] = in ? x[4 * i + j] * d[j] : 0.0f;
  }
  rotate_lane<N>(x, lane);
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
  m = fmaxf(m, xor_lane<16>(m));
  m = fmaxf(m, xor_lane<32>(m));
  // the largest to [2^13, 2^14): the second part of an element above 2^-27 of it is then a normal fp16 number
  const int e = m > 0.0f && m < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(m) : 0;
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = __builtin_amdgcn_ldexpf(x[8 * c + code_place<BITS>(j)], e);
      hi[c][j] = static_cast<_Float16>(y);
      lo[c][j] = static_cast<_Float16>(y - static_cast<float>(hi[c][j]));
    }
  *factor = __builtin_amdgcn_ldexpf(a.wscale * a.scale2, -e);
}

// Scores of the step's 2 x 16 slots against 16 rows, in log2 units: slot 16 k + 4 g + i, row lane % 16.
template <int D, int BITS>
__device__ __forceinline__ void score_step(const f16x8_t (&kc)[2][D / 32], const f32x4_t (&ks)[2], const f16x8_t (&hi)[D / 32],
                                           const f16x8_t (&lo)[D / 32], float factor, f32x4_t (&x)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < D / 32; ++c) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[k][c], lo[c], s, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[k][c], hi[c], s, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[k][i] = s[i] * (ks[k][i] * factor);
  }
}

template <int DT, int N>
__device__ __forceinline__ void store_row(void* out, int64_t at, const float (&y)[N]) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = DT == AEKV_BF16 ? pack_bf16x2(y[2 * i], y[2 * i + 1]) : (f32_to_f16_bits(y[2 * i]) | (f32_to_f16_bits(y[2 * i + 1]) << 16));
  uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
  for (int i = 0; i < N / 8; ++i) p[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

template <int DT, int D, int BITS, int MT>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_kernel(PagedArgs a) {
  using G = PagedGeom<D, BITS>;
  using S = Stage<D, BITS>;
  constexpr int N = D / 4, NS = S::kStages;
  // a ring of stages for each wave; afterwards stage w holds wave w + 1's state for the merge.  Arrays of their own, so
  // that the compiler sees that loads into one do not write what is read from another.
  __shared__ __align__(16) uint8_t st0[kWaves * S::kBytes];
  __shared__ __align__(16) uint8_t st1[kWaves * S::kBytes];
  __shared__ __align__(16) uint8_t st2[NS == 3 ? kWaves * S::kBytes : 16];
  static_assert(MT * (N + 2) * 256 <= kWaves * S::kBytes, "a wave's state fits a stage");
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups: pieces innermost, then row blocks, then KV heads, then sequences
  uint32_t wg = blockIdx.x;
  const int32_t split = static_cast<int32_t>(wg % a.n_split);
  wg /= a.n_split;
  const int32_t rb = static_cast<int32_t>(wg % a.row_blocks);
  wg /= a.row_blocks;
  const int32_t kh = static_cast<int32_t>(wg % a.pool.heads);
  int64_t b = wg / a.pool.heads;
  int32_t n, pages = -1;
  if (a.ranked == 1) b = ranked_sequence<1>(a, static_cast<int32_t>(b), lane, &n);
  else if (a.ranked == 2) b = ranked_sequence<8>(a, static_cast<int32_t>(b), lane, &n);
  if (a.n_split == 1) pages = load_pages(a, b, kStep * wave, lane);  // (of a whole sequence: not after its length)
  if (!a.ranked) n = newest_sees(a, b);
  const int32_t length = max(a.lengths[b], 0);
  const int32_t piece = piece_slots(n, a.n_split);
  const int32_t p0 = split * static_cast<int64_t>(piece) < n ? split * piece : n, p1 = min(static_cast<int64_t>(p0) + piece, static_cast<int64_t>(n));
  if (split > 0 && p0 >= p1) return;  // (the merge knows how many pieces a sequence has)

  // the queries are requested first, then the first steps; the rotation runs while those are on their way
  int32_t row[MT];
  uint4 qw[MT][D / 32];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    row[t] = (rb * MT + t) * 16 + (lane & 15);
    load_query<D>(a, b, kh, row[t], row[t] < a.rows, lane, qw[t]);
  }
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u));
  const int32_t first = p0 + kStep * wave;
  const int n_steps = first < p1 ? (p1 - first + kRound - 1) / kRound : 0;
  uint32_t bad[NS] = {};  // bit k: tile k of the stage's step has no page
  auto stage = [&](auto which) -> uint8_t* {
    return (decltype(which)::value == 0 ? st0 : decltype(which)::value == 1 ? st1 : st2) + wave * S::kBytes;
  };
  auto load = [&](int i, auto which) __attribute__((always_inline)) {
    if ((i & 31) == 0 && (i > 0 || a.n_split > 1)) pages = load_pages(a, b, first + kRound * i, lane);
    const int32_t g0 = __builtin_amdgcn_readlane(pages, 2 * (i & 31)), g1 = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1);
    bad[decltype(which)::value] = (g0 < 0 ? 1u : 0u) | (g1 < 0 ? 2u : 0u);
    issue_step<D, BITS>(a, kh, first + kRound * i, g0, g1, lane, stage(which));
  };
  if (n_steps > 0) load(0, std::integral_constant<int, 0>{});
  if (NS == 3 && n_steps > 1) load(1, std::integral_constant<int, 1>{});

  f16x8_t qhi[MT][D / 32], qlo[MT][D / 32];
  float factor[MT], m[MT], l[MT];
  int32_t sees[MT];
  f32x4_t o[MT][G::kNE], ones_sum[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const bool in = row[t] < a.rows;
    query_parts<DT, D, BITS>(a, qw[t], in, lane, qhi[t], qlo[t], &factor[t]);
    sees[t] = in ? token_sees(a, length, n, row[t] / a.G) : n;
    m[t] = kNegInf, l[t] = 0.0f;
#pragma unroll
    for (int e = 0; e < G::kNE; ++e) o[t][e] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    ones_sum[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int32_t sees_all = token_sees(a, length, n, rb * MT * 16 / a.G);  // the fewest that a row of the block sees

  // a landed step; `whole`: every row sees all of it
  auto body = [&](const StepData<D, BITS>& s, int32_t base, uint32_t none, auto whole_c) __attribute__((always_inline)) {
    constexpr bool whole = decltype(whole_c)::value;
    f16x8_t kc[2][D / 32];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kc[k][c] = codes_f16<BITS>(&s.k[k][c * BITS / 4]);
    bf16x8_t phi[MT], plo[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      f32x4_t x[2];
      score_step<D, BITS>(kc, s.ks, qhi[t], qlo[t], factor[t], x);
      bool hide[2][4] = {};
      if constexpr (!whole) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            hide[k][j] = ((none >> k) & 1u) || base + 16 * k + 4 * g + j >= sees[t];
            x[k][j] = hide[k][j] ? kNegInf : x[k][j];
          }
      }
      if (a.logits && row[t] < a.rows) {
        float* lg = a.logits + ((b * a.pool.heads + kh) * a.rows + row[t]) * a.logit_slots + base + 4 * g;
        *reinterpret_cast<f32x4_t*>(lg) = x[0];
        *reinterpret_cast<f32x4_t*>(lg + 16) = x[1];
      }
      float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
      top = fmaxf(top, xor_lane<16>(top));
      top = fmaxf(top, xor_lane<32>(top));
      // (each row by itself: a row's bits do not depend on the others')
      const bool moved = top > m[t] + kMargin;
      if (__builtin_amdgcn_ballot_w64(moved)) {
        const float r = moved ? __builtin_amdgcn_exp2f(m[t] - top) : 1.0f;
        l[t] *= r;
#pragma unroll
        for (int e = 0; e < G::kNE; ++e) o[t][e] *= r;
        ones_sum[t] *= r;
        m[t] = moved ? top : m[t];
      }
      const float nm = m[t] == kNegInf ? 0.0f : -m[t];
      float c[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = __builtin_amdgcn_exp2f(x[k][j] + nm);
          l[t] += p;
          c[k][j] = p * s.vs[k][j];
          if constexpr (!whole) c[k][j] = hide[k][j] ? 0.0f : c[k][j];  // (whatever a hidden slot's scale is)
        }
      uint32_t h[4], r[4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float c0 = c[k][2 * j], c1 = c[k][2 * j + 1];
          const uint32_t u = pack_bf16x2(c0, c1);
          h[2 * k + j] = u;
          r[2 * k + j] = pack_bf16x2(c0 - bf16_to_f32(u), c1 - __builtin_bit_cast(float, u & 0xffff0000u));
        }
      phi[t] = __builtin_bit_cast(bf16x8_t, make_uint4(h[0], h[1], h[2], h[3]));
      plo[t] = __builtin_bit_cast(bf16x8_t, make_uint4(r[0], r[1], r[2], r[3]));
      ones_sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, phi[t], ones_sum[t], 0, 0, 0);
      ones_sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, plo[t], ones_sum[t], 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < G::kNE; ++e) {
      // (a step's codes are flipped once: xor 0x80 makes bytes 0 .. 255)
      uint32_t v[8][G::kWords];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int q = 0; q < G::kWords; ++q) v[j][q] = BITS == 8 ? s.v[j][q] ^ 0x80808080u : s.v[j][q];
      const bf16x8_t va = values_bf16<D, BITS>(v, e);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, phi[t], o[t][e], 0, 0, 0);
        o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, plo[t], o[t][e], 0, 0, 0);
      }
    }
  };
  // one step: the loads of the one NS - 1 ahead go out, then this one's are waited for
  auto compute = [&](int i, auto which) __attribute__((always_inline)) {
    constexpr int w = decltype(which)::value;
    if (i + NS - 1 < n_steps) {
      load(i + NS - 1, std::integral_constant<int, (w + NS - 1) % NS>{});
      wait_loads<(NS - 1) * S::kLoads>();
    } else {
      wait_loads<0>();
    }
    StepData<D, BITS> s;
    read_step<D, BITS>(stage(which), lane, s);
    const int32_t base = first + kRound * i;
    if (bad[w] == 0 && base + kStep <= sees_all) body(s, base, 0u, std::true_type{});
    else body(s, base, bad[w], std::false_type{});
  };
#pragma unroll 1
  for (int i = 0; i < n_steps; i += NS) {
    compute(i, std::integral_constant<int, 0>{});
    if (i + 1 >= n_steps) break;
    compute(i + 1, std::integral_constant<int, 1>{});
    if constexpr (NS == 3) {
      if (i + 2 >= n_steps) break;
      compute(i + 2, std::integral_constant<int, 2>{});
    }
  }

  // the wave's rows in order of their dims, the offset out; then the waves' states into the first one's
  float y[MT][N];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    l[t] += xor_lane<16>(l[t]);
    l[t] += xor_lane<32>(l[t]);
#pragma unroll
    for (int e = 0; e < G::kNE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[t][G::kNE * i + e] = o[t][e][i] - G::kBias * ones_sum[t][i];
  }
  // state of wave w + 1: word i of row tile t at (t (N + 2) + i) 64 + lane, then its maximum and sum
  auto state = [&](int w) { return reinterpret_cast<float*>(NS == 3 ? (w == 0 ? st0 : w == 1 ? st1 : st2) : (w == 0 ? st0 : w == 1 ? st1 : st0 + kWaves * S::kBytes / 2)); };
  static_assert(NS == 3 || 2 * MT * (N + 2) * 256 <= kWaves * S::kBytes, "two states fit a stage");
  __syncthreads();  // every wave has read its last stage
  if (wave > 0) {
    float* p = state(wave - 1);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < N; ++i) p[(t * (N + 2) + i) * 64 + lane] = y[t][i];
      p[(t * (N + 2) + N) * 64 + lane] = m[t];
      p[(t * (N + 2) + N + 1) * 64 + lane] = l[t];
    }
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    float top = m[t], pm[kWaves - 1], pl[kWaves - 1];
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) {
      pm[w] = state(w)[(t * (N + 2) + N) * 64 + lane];
      pl[w] = state(w)[(t * (N + 2) + N + 1) * 64 + lane];
      top = fmaxf(top, pm[w]);
    }
    // (a state of nothing has a sum of 0; NaN alone leaves a maximum of -inf, and a sum that says so)
    const float f = l[t] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
    l[t] = l[t] == 0.0f ? 0.0f : l[t] * f;
#pragma unroll
    for (int i = 0; i < N; ++i) y[t][i] *= f;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) {
      const float fw = pl[w] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(pm[w] - top);
      l[t] += pl[w] == 0.0f ? 0.0f : pl[w] * fw;
#pragma unroll
      for (int i = 0; i < N; ++i) y[t][i] = fmaf(state(w)[(t * (N + 2) + i) * 64 + lane], fw, y[t][i]);
    }
    m[t] = top;
    if (row[t] >= a.rows) continue;
    const int32_t tok = row[t] / a.G, h = kh * a.G + (row[t] - tok * a.G);
    const int64_t orow = (b * a.T + tok) * a.H + h;
    if (a.n_split > 1) {
      float* p = a.part + (orow * a.n_split + split) * (D + 4);
      if (g == 0) p[0] = m[t], p[1] = l[t];
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        *reinterpret_cast<f32x4_t*>(p + 4 + g * N + 4 * i) = f32x4_t{y[t][4 * i], y[t][4 * i + 1], y[t][4 * i + 2], y[t][4 * i + 3]};
    }
  }
  if (a.n_split > 1) return;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const bool in = row[t] < a.rows;
    const int32_t tok = in ? row[t] / a.G : 0, h = in ? kh * a.G + (row[t] - tok * a.G) : 0;
    const int64_t orow = (b * a.T + tok) * a.H + h;
    const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
    const float top = fmaxf(m[t], sk);
    const float f = l[t] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
    const float sum = l[t] * f + (sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - top));
    const float r = sum == 0.0f ? 0.0f : f / sum * a.wscale;
#pragma unroll
    for (int i = 0; i < N; ++i) y[t][i] *= r;
    rotate_lane<N>(y[t], lane);
#pragma unroll
    for (int i = 0; i < N; ++i) y[t][i] *= a.diag[g * N + i];
    if (in) {
      store_row<DT, N>(a.out, orow * D + g * N, y[t]);
      if (a.lse && g == 0) a.lse[orow] = sum == 0.0f ? -kNegInf : top + __builtin_amdgcn_logf(sum);
    }
  }
}

// Merges the pieces of one row and rotates it back: the workgroup's waves take every fourth piece each.  Bound by the chain
// of its loads: 12 rows of 128 pieces 8 us with four pieces requested at a time, 6.5 with eight (sixteen, whose registers
// halve the waves on a CU, made 2048 rows of 5 pieces 0.8 us slower).
template <int DT, int D>
__device__ __forceinline__ void merge_row(const PagedArgs& a, int64_t orow) {
  constexpr int PER = D / 64;
  __shared__ float s_o[kWaves][D], s_ml[kWaves][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = orow / (static_cast<int64_t>(a.T) * a.H);
  const int32_t h = static_cast<int32_t>(orow % a.H);
  const int32_t n = newest_sees(a, b);
  const int32_t piece = piece_slots(n, a.n_split);
  const int pieces = max((n + piece - 1) / piece, 1);
  const float* p = a.part + orow * a.n_split * (D + 4);
  float m = kNegInf, l = 0.0f, x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = 0.0f;
  // CH pieces at a time, all their loads issued together (a piece past the last counts as empty)
  auto merge = [&](auto ch) __attribute__((always_inline)) {
    constexpr int CH = decltype(ch)::value;
    for (int s0 = wave; s0 < (CH < 8 ? wave + 1 : pieces); s0 += kWaves * CH) {  // (2, 4: one pass, whose loads do not wait for the length)
      float pm[CH], pl[CH], v[CH][PER];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int s = s0 + kWaves * c;
        const float* ps = p + static_cast<int64_t>(min(s, a.n_split - 1)) * (D + 4);
        pm[c] = ps[0], pl[c] = ps[1];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[c][i] = ps[4 + PER * lane + i];
      }
      float top = m;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (s0 + kWaves * c >= pieces) {  // (what lies there is anything)
          pm[c] = kNegInf, pl[c] = 0.0f;
#pragma unroll
          for (int i = 0; i < PER; ++i) v[c][i] = 0.0f;
        }
        top = fmaxf(top, pm[c]);
      }
      const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
      l = l == 0.0f ? 0.0f : l * f;
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] *= f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float fp = pl[c] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(pm[c] - top);
        l += pl[c] == 0.0f ? 0.0f : pl[c] * fp;
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] += v[c][i] * fp;
      }
      m = top;
    }
  };
  if (a.n_split <= 2 * kWaves) merge(std::integral_constant<int, 2>{});
  else if (a.n_split <= 4 * kWaves) merge(std::integral_constant<int, 4>{});
  else merge(std::integral_constant<int, 8>{});
#pragma unroll
  for (int i = 0; i < PER; ++i) s_o[wave][PER * lane + i] = x[i];
  if (lane == 0) s_ml[wave][0] = m, s_ml[wave][1] = l;
  __syncthreads();
  if (wave > 0) return;
  const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
  float top = sk;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_ml[w][0]);
  float sum = sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - top);
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float lw = s_ml[w][1], f = lw == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][0] - top);
    sum += lw == 0.0f ? 0.0f : lw * f;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = fmaf(s_o[w][PER * lane + i], f, x[i]);
  }
  const float r = sum == 0.0f ? 0.0f : a.wscale / sum;
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] *= r;
  wht_butterflies<D, PER>(x, lane);
  uint32_t w[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float y = x[i] * a.diag[PER * lane + i];
    w[i] = DT == AEKV_BF16 ? (pack_bf16x2(y, 0.0f) & 0xffffu) : f32_to_f16_bits(y);
  }
  uint16_t* out = static_cast<uint16_t*>(a.out) + orow * D + PER * lane;
  if constexpr (PER == 2) *reinterpret_cast<uint32_t*>(out) = w[0] | (w[1] << 16);
  else out[0] = static_cast<uint16_t>(w[0]);
  if (a.lse && lane == 0) a.lse[orow] = sum == 0.0f ? -kNegInf : top + __builtin_amdgcn_logf(sum);
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedArgs a) {
  merge_row<DT, D>(a, blockIdx.x);
}

// The weights of a sequence's slots from the logits that the attention left and the rows' log sums: four slots to a thread.
// Reads 4 bytes per row and slot, reads and writes the weights: 64 sequences x 4 heads x 3 rows of up to 16384 slots, 10 us.
// MERGED: the log sums come from the pieces' maxima and sums (16 lanes to a row), so that the pieces' merge need not come first.
constexpr int kAddSlots = 1024;   // of a workgroup
constexpr int kLogitRows = 16;    // most rows of a KV head whose logits are kept

template <bool MERGED, int D>
__device__ __forceinline__ void add_weights(const PagedArgs& a, uint32_t block, int32_t blocks) {
  __shared__ float s_lse[kLogitRows];
  const int32_t j0 = static_cast<int32_t>(block % blocks) * kAddSlots, j = j0 + 4 * static_cast<int32_t>(threadIdx.x);
  const int64_t bk = block / blocks, b = bk / a.pool.heads;
  const int32_t kh = static_cast<int32_t>(bk - b * a.pool.heads);
  const int32_t n = newest_sees(a, b);
  if (j0 >= n) return;  // (the whole workgroup)
  const int32_t r = static_cast<int32_t>(threadIdx.x) >> 4, own = min(r, a.rows - 1), t = own / a.G, h = kh * a.G + (own - t * a.G);
  const int64_t orow = (b * a.T + t) * a.H + h;
  float lse;
  if constexpr (MERGED) {
    const int32_t piece = piece_slots(n, a.n_split), pieces = (n + piece - 1) / piece;
    const float* p = a.part + orow * a.n_split * (D + 4);
    float m = kNegInf, l = 0.0f;
    for (int s = threadIdx.x & 15; s < pieces; s += 16) {
      const float2 ml = *reinterpret_cast<const float2*>(p + static_cast<int64_t>(s) * (D + 4));
      const float top = fmaxf(m, ml.x);
      l = (l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f(m - top)) + (ml.y == 0.0f ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - top));
      m = top;
    }
    const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
    float top = fmaxf(m, sk);
    top = fmaxf(top, xor_lane<1>(top)), top = fmaxf(top, xor_lane<2>(top)), top = fmaxf(top, xor_lane<4>(top)), top = fmaxf(top, xor_lane<8>(top));
    l = l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f(m - top);
    l += xor_lane<1>(l), l += xor_lane<2>(l), l += xor_lane<4>(l), l += xor_lane<8>(l);
    l += sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - top);
    lse = l == 0.0f ? -kNegInf : top + __builtin_amdgcn_logf(l);
  } else {
    lse = a.lse[orow];
  }
  if ((threadIdx.x & 15) == 0) s_lse[r] = lse;
  __syncthreads();
  if (j >= n) return;
  const float* lg = a.logits + bk * a.rows * a.logit_slots + j;
  float* w = a.weights + bk * a.capacity + j;
  const bool vec = (a.capacity & 3) == 0 && j + 4 <= n;  // (weights is 16-byte aligned: the launcher checks)
  f32x4_t before = {0.0f, 0.0f, 0.0f, 0.0f}, sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (vec) before = *reinterpret_cast<const f32x4_t*>(w);
#pragma unroll 4
  for (int32_t i = 0; i < a.rows; ++i) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(lg + i * a.logit_slots);  // (the step's 32 slots are all there)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += x[e] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(x[e] - s_lse[i]);  // (hidden: nothing, whatever the row's sum is)
  }
  if (vec) {
    *reinterpret_cast<f32x4_t*>(w) = before + sum;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < n) w[e] += sum[e];
  }
}

__global__ __launch_bounds__(kThreads) void paged_add_kernel(PagedArgs a, int32_t blocks) { add_weights<false, 64>(a, blockIdx.x, blocks); }

// Both ends of a tracked call in pieces, in one launch: `rows` workgroups merge a row each, the others add (the 64 sequences
// above 96.4 -> 94.9 us).
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void paged_merge_add_kernel(PagedArgs a, uint32_t rows, int32_t blocks) {
  if (blockIdx.x < rows) merge_row<DT, D>(a, blockIdx.x);
  else add_weights<true, D>(a, blockIdx.x - rows, blocks);
}

// The weights of a piece of a sequence's slots, from the rows' log sums: each wave scores steps of 32 slots against every
// row of the KV head's group, 16 at a time (their query parts in LDS), and adds the sums over the rows.  Bound by the
// rotations that come before the first step and then the vector work of the scores: 128 rows, 8 sequences x 2 heads of up
// to 5001 slots, dim 64, 8 bits: 14 us.
constexpr int kWeightTiles = 8;  // row tiles whose parts LDS holds at a time

template <int DT, int D, int BITS>
__global__ __launch_bounds__(kThreads) void paged_weights_kernel(PagedArgs a) {
  constexpr int NC = D / 32;
  __shared__ __align__(16) f16x8_t s_hi[kWeightTiles][NC][64], s_lo[kWeightTiles][NC][64];
  __shared__ float s_f[kWeightTiles][16], s_lse[kWeightTiles][16];
  __shared__ int32_t s_sees[kWeightTiles][16];
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t wg = blockIdx.x;
  const int32_t split = static_cast<int32_t>(wg % a.n_split);
  wg /= a.n_split;
  const int32_t kh = static_cast<int32_t>(wg % a.pool.heads);
  const int64_t b = wg / a.pool.heads;
  const int32_t n = newest_sees(a, b), length = max(a.lengths[b], 0);
  const int32_t piece = piece_slots(n, a.n_split);
  const int32_t p0 = split * static_cast<int64_t>(piece) < n ? split * piece : n, p1 = min(static_cast<int64_t>(p0) + piece, static_cast<int64_t>(n));
  if (p0 >= p1) return;  // (the whole workgroup)
  float* weights = a.weights + (b * a.pool.heads + kh) * a.capacity;
  const int32_t first = p0 + kStep * wave;
  const int n_steps = first < p1 ? (p1 - first + kRound - 1) / kRound : 0;
  const int tiles = (a.rows + 15) / 16;
  for (int t0 = 0; t0 < tiles; t0 += kWeightTiles) {
    const int nt = min(tiles - t0, kWeightTiles);
    if (t0 > 0) __syncthreads();
    for (int t = wave; t < nt; t += kWaves) {
      const int32_t row = (t0 + t) * 16 + (lane & 15);
      const bool in = row < a.rows;
      f16x8_t hi[NC], lo[NC];
      float factor;
      uint4 qw[NC];
      load_query<D>(a, b, kh, row, in, lane, qw);
      query_parts<DT, D, BITS>(a, qw, in, lane, hi, lo, &factor);
#pragma unroll
      for (int c = 0; c < NC; ++c) s_hi[t][c][lane] = hi[c], s_lo[t][c][lane] = lo[c];
      if (g == 0) {
        const int32_t tok = in ? row / a.G : 0, h = in ? kh * a.G + (row - tok * a.G) : 0;
        s_f[t][lane] = factor;
        s_lse[t][lane] = a.lse[(b * a.T + tok) * a.H + h];
        s_sees[t][lane] = in ? token_sees(a, length, n, tok) : 0;
      }
    }
    __syncthreads();
    int32_t pages = -1, g0 = -1, g1 = -1;
    StepData<D, BITS> s, next;
    auto load = [&](int i) __attribute__((always_inline)) {
      if ((i & 31) == 0) pages = load_pages(a, b, first + kRound * i, lane);
      g0 = __builtin_amdgcn_readlane(pages, 2 * (i & 31)), g1 = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1);
      load_keys<D, BITS>(a, kh, first + kRound * i, g0, g1, lane, next);
    };
    if (n_steps > 0) load(0);
#pragma unroll 1
    for (int i = 0; i < n_steps; ++i) {
      const int32_t base = first + kRound * i;
      s = next;
      const uint32_t bad = (g0 < 0 ? 1u : 0u) | (g1 < 0 ? 2u : 0u);
      f16x8_t kc[2][NC];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c) kc[k][c] = codes_f16<BITS>(&s.k[k][c * BITS / 4]);
      if (i + 1 < n_steps) load(i + 1);
      f32x4_t sum[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
      for (int t = 0; t < nt; ++t) {
        f16x8_t hi[NC], lo[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) hi[c] = s_hi[t][c][lane], lo[c] = s_lo[t][c][lane];
        f32x4_t x[2];
        score_step<D, BITS>(kc, s.ks, hi, lo, s_f[t][lane & 15], x);
        const float lse = s_lse[t][lane & 15];
        const int32_t sees = s_sees[t][lane & 15];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool hide = ((bad >> k) & 1u) || base + 16 * k + 4 * g + j >= sees;
            sum[k][j] += hide ? 0.0f : __builtin_amdgcn_exp2f(x[k][j] - lse);
          }
      }
      // over the 16 rows
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = sum[k][j];
          v += xor_lane<1>(v);
          v += xor_lane<2>(v);
          v += xor_lane<4>(v);
          v += xor_lane<8>(v);
          sum[k][j] = v;
        }
        const int j = lane & 15;
        const int32_t slot = base + 16 * k + 4 * g + j;
        if (j < 4 && slot < p1 && !((bad >> k) & 1u)) {
          const float v = j == 0 ? sum[k][0] : j == 1 ? sum[k][1] : j == 2 ? sum[k][2] : sum[k][3];
          if (v != 0.0f) weights[slot] += v;
        }
      }
    }
  }
}

using paged_fn = void (*)(PagedArgs);

template <int DT>
paged_fn pick_paged(int d, int bits, int mt) {
  if (mt == 2) return bits == 8 ? paged_attention_kernel<DT, 64, 8, 2> : paged_attention_kernel<DT, 64, 4, 2>;
  if (d == 64) return bits == 8 ? paged_attention_kernel<DT, 64, 8, 1> : paged_attention_kernel<DT, 64, 4, 1>;
  return bits == 8 ? paged_attention_kernel<DT, 128, 8, 1> : paged_attention_kernel<DT, 128, 4, 1>;
}

template <int DT>
paged_fn pick_weights(int d, int bits) {
  if (d == 64) return bits == 8 ? paged_weights_kernel<DT, 64, 8> : paged_weights_kernel<DT, 64, 4>;
  return bits == 8 ? paged_weights_kernel<DT, 128, 8> : paged_weights_kernel<DT, 128, 4>;
}

// Pieces of a sequence: enough workgroups for the chip (1536: three per CU, twice over, which evens out sequences of
// different lengths; one sequence of 262144 slots x 12 heads, 1024 / 1536 / 2048 / 3000 workgroups: 111 / 101 / 109 / 113
// us, 64 ragged ones of up to 16384 slots x 4 heads 122 / 119 / 117 / 119), but none of fewer than 512 slots beyond 512
// workgroups (a workgroup's rotations and merge cost as much as some 500 slots), and none without a whole round of slots.
// Tables of up to kOnePiece slots are not split: for many sequences the merge's launch costs more than their few rounds
// (64 of 256 / 512 / 768 slots x 4 heads, split 12.3 / 13.8 / 15.5 us, whole 9.7 / 11.6 / 13.9), for one it costs as much of
// the host's time as it saves of the card's (512 slots, replayed from a graph 9.5 and 11.3 us, called 13.8 and 10.1).
constexpr int64_t kOnePiece = 512;
int64_t paged_pieces(int64_t groups, int64_t slots) {
  if (slots <= kOnePiece) return 1;
  const int64_t few = ceil_div(512, groups), some = ceil_div(slots, 512);
  const int64_t want = ceil_div(1536, groups), most = ceil_div(slots, kRound);
  int64_t n = few > some ? few : some;
  n = n < want ? n : want;
  n = n < most ? n : most;
  return n < 1 ? 1 : n;
}

// A batch whose workgroups do not all run together starts its longest sequences first, so that no long one is left for the
// end, where pieces can be long enough for that to count: finding the order costs a workgroup some 1 us.  By index / longest
// first, 12 heads of 4, dim 128, 4 bits: 64 ragged sequences of up to 16384 slots 98.3 / 85.9 us, one of 16384 among 63 of
// 1024 47.3 / 35.8, in pieces of 682 slots (16 of up to 16384) 34.3 / 36.7.
constexpr int64_t kRanked = 512, kRankedSlots = 2048;

// Whether a call of these sizes (a multiple of the KV heads' query heads) fits a launch.
bool paged_fits(int64_t B, int64_t T, int64_t H, int64_t heads, int64_t blocks) {
  return B <= 0x7fffffff && H <= 65535 && T <= 0x7fffff && T * (H / heads) <= 0x3fffffff &&
         static_cast<double>(B) * static_cast<double>(heads * blocks) <= kMaxGridThreads / kThreads / 4 &&
         static_cast<double>(B) * static_cast<double>(T * H) <= kMaxGridThreads / kThreads;
}

// Row tiles of a wave: two share a step's unpacked codes where there are as many rows and registers.  At dim 128 two take all
// 256 registers and spill (4 bits; at 8 the waves' states do not fit a stage of LDS either), so each 16 rows read the codes
// again: 32 sequences of 16384 slots, 12 heads of 4, 4 bits, one token (3 rows) 64 us, 5 (15) 72, 16 (48) 160.
int paged_row_tiles(int64_t rows, int32_t d) { return rows > 16 && d == 64 ? 2 : 1; }

// Tracked calls of few rows keep their logits and sum them afterwards; of many rows the scores are computed again, which
// reads a slot's K codes instead of 8 bytes a row.
size_t paged_logit_bytes(int64_t B, int64_t heads, int64_t rows, int64_t slots) {
  if (rows > kLogitRows) return 0;
  const double bytes = 4.0 * static_cast<double>(B) * heads * rows * static_cast<double>(slots + 32);
  return bytes > 2147483648.0 ? 0 : static_cast<size_t>(B * heads * rows) * align_up(static_cast<size_t>(slots), 32) * 4;
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" size_t aekv_paged_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t heads, int32_t d,
                                                      int64_t slots, int32_t tracked) {
  if (B <= 0 || T <= 0 || H <= 0 || heads <= 0 || d <= 0 || slots <= 0 || H % heads || T > 0x7fffff || H > 65535) return 0;
  const int64_t rows = T * (H / heads), blocks = ceil_div(rows, 16 * paged_row_tiles(rows, d));
  if (!paged_fits(B, T, H, heads, blocks)) return 0;  // (the call refuses it)
  const int64_t n = paged_pieces(B * heads * blocks, slots);
  return (tracked ? align_up(static_cast<size_t>(B * T * H) * 4, 16) + paged_logit_bytes(B, heads, rows, slots) : 0) +
         (n > 1 ? static_cast<size_t>(B * T * H) * static_cast<size_t>(n) * (d + 4) * 4 : 0);
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
  if (!is_aligned(q, 16) || !is_aligned(out, 16) || !is_aligned(ws, 16) || !is_aligned(diag, 16) || !is_aligned(weights, 16) || (q_batch_stride % 8) ||
      (q_token_stride % 8) || (q_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q rows, out, diag, weights and workspace must be 16-byte aligned", who);
  const int64_t slots = max_pages * page_size, rows = H <= 65535 && T <= 0x7fffff ? T * (H / heads) : 1;
  const int mt = paged_row_tiles(rows, d);
  const int64_t blocks = ceil_div(rows, 16 * mt);
  if (!paged_fits(B, T, H, heads, blocks))
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld T=%lld H=%lld exceed the grid", who, (long long)B, (long long)T, (long long)H);
  const size_t want = aekv_paged_attention_workspace_size(B, T, H, heads, d, slots, weights != nullptr);
  if (want && (!ws || ws_bytes < want)) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  int64_t reach = pages > 0 ? slots : 0;
  if (weights && capacity < reach) reach = capacity;
  a.q = q;
  a.q_batch = q_batch_stride;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.lengths = lengths;
  a.diag = diag;
  a.sink = sink;
  a.weights = reach > 0 ? weights : nullptr;
  a.lse = a.weights ? static_cast<float*>(ws) : nullptr;
  // the workspace: the rows' log sums, the logits, the pieces
  const size_t lse_bytes = weights ? align_up(static_cast<size_t>(B * T * H) * 4, 16) : 0;
  const size_t logit_bytes = weights ? paged_logit_bytes(B, heads, rows, slots) : 0;
  a.logits = a.weights && logit_bytes ? reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + lse_bytes) : nullptr;
  a.logit_slots = static_cast<int64_t>(align_up(static_cast<size_t>(slots), 32));
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + lse_bytes + logit_bytes);
  a.out = out;
  a.reach = static_cast<int32_t>(reach);
  a.capacity = capacity;
  a.T = static_cast<int32_t>(T);
  a.H = static_cast<int32_t>(H);
  a.G = static_cast<int32_t>(H / heads);
  a.rows = static_cast<int32_t>(rows);
  a.row_blocks = static_cast<int32_t>(blocks);
  a.n_split = static_cast<int32_t>(paged_pieces(B * heads * blocks, slots));
  a.B = static_cast<int32_t>(B);
  a.ranked = B > 1 && B <= kRanked && reach / a.n_split >= kRankedSlots && B * heads * blocks * a.n_split > 768 ? (B <= 64 ? 1 : 2) : 0;
  a.scale2 = softmax_scale * kLog2e;
  a.wscale = wht_scale(d);
  const hipStream_t st = as_stream(stream);
  auto fn = dtype == AEKV_F16 ? pick_paged<AEKV_F16>(d, bits, mt) : pick_paged<AEKV_BF16>(d, bits, mt);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(B * heads * blocks * a.n_split)), dim3(kThreads), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  const int32_t per = a.logits ? static_cast<int32_t>(ceil_div(reach, kAddSlots)) : 0;
  if (a.n_split > 1 && a.logits) {
    auto mg = dtype == AEKV_F16 ? (d == 64 ? paged_merge_add_kernel<AEKV_F16, 64> : paged_merge_add_kernel<AEKV_F16, 128>)
                                : (d == 64 ? paged_merge_add_kernel<AEKV_BF16, 64> : paged_merge_add_kernel<AEKV_BF16, 128>);
    hipLaunchKernelGGL(mg, dim3(static_cast<uint32_t>(B * T * H + B * heads * per)), dim3(kThreads), 0, st, a, static_cast<uint32_t>(B * T * H), per);
    return check_launch(who);
  }
  if (a.n_split > 1) {
    auto mg = dtype == AEKV_F16 ? (d == 64 ? paged_merge_kernel<AEKV_F16, 64> : paged_merge_kernel<AEKV_F16, 128>)
                                : (d == 64 ? paged_merge_kernel<AEKV_BF16, 64> : paged_merge_kernel<AEKV_BF16, 128>);
    hipLaunchKernelGGL(mg, dim3(static_cast<uint32_t>(B * T * H)), dim3(kThreads), 0, st, a);
    if (const int rc = check_launch(who)) return rc;
  }
  if (!a.weights) return AEKV_OK;
  if (a.logits) {
    hipLaunchKernelGGL(paged_add_kernel, dim3(static_cast<uint32_t>(B * heads * per)), dim3(kThreads), 0, st, a, per);
    return check_launch(who);
  }
  a.n_split = static_cast<int32_t>(paged_pieces(B * heads, slots));
  auto wf = dtype == AEKV_F16 ? pick_weights<AEKV_F16>(d, bits) : pick_weights<AEKV_BF16>(d, bits);
  hipLaunchKernelGGL(wf, dim3(static_cast<uint32_t>(B * heads * a.n_split)), dim3(kThreads), 0, st, a);
  return check_launch(who);
}
