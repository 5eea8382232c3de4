// The fast encode of vectors held 32 elements to a lane (D = 64 and 128), shared by the codec's kernels and by the append
// into a paged cache.  Bit for bit encode_lane's codes and scales (tq_device.h).
#pragma once

#include "tq_device.h"

namespace aekv {
namespace {

constexpr float kMagic8 = 12582920.0f;  // 1.5 * 2^23 + 8: RN(t + kMagic8) = kMagic8 + rne(t), ulp 1

// Stages h = 32 and h = 64 on eight registers: a += s * a(partner), the partner's value read by
// v_fmac_f32 through DPP quad_perm [1,0,3,2] (lane ^ 1), then [2,3,0,1] (lane ^ 2).  Written as
// inline asm because the compiler only forms v_fmac from its VOP3 FMA after the pass that folds
// DPP moves, and VOP3 has no DPP form on gfx950.  A DPP read of a VGPR needs two wait states after
// the VALU write of it: s_nop 1 covers the code before the block, and inside it every register is
// read through DPP eight instructions after its write.
__device__ __forceinline__ void quad_stages8(float& a0, float& a1, float& a2, float& a3, float& a4, float& a5,
                                             float& a6, float& a7, float s32, float s64) {
  asm("s_nop 1\n"
      "v_fmac_f32_dpp %0, %0, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %1, %1, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %2, %2, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %3, %3, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %4, %4, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %5, %5, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %6, %6, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %7, %7, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %0, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %1, %1, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %2, %2, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %3, %3, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %4, %4, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %5, %5, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %6, %6, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %7, %7, %9 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf"
      : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3), "+v"(a4), "+v"(a5), "+v"(a6), "+v"(a7)
      : "v"(s32), "v"(s64));
}

// ue, uo: bit patterns of M8 + n (n in [-7, 7]), whose low byte is n + 8 in [1, 15].
// Returns a word whose low byte is (n_odd + 8) << 4 | (n_even + 8); bits 8.. are garbage.
__device__ __forceinline__ uint32_t nib_pair(uint32_t ue, uint32_t uo) { return (uo << 4) | ue; }

// Low bytes of four nib_pair words -> one dword of two's-complement nibbles (xor 8 per nibble
// turns the offset-binary n + 8 into n & 15).
__device__ __forceinline__ uint32_t pack4(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
  const uint32_t lo = __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u);  // [b0.0, b1.0, 0, 0]
  const uint32_t hi = __builtin_amdgcn_perm(b3, b2, 0x04000c0cu);  // [0, 0, b2.0, b3.0]
  return (lo | hi) ^ 0x88888888u;
}

// max(acc, |x|, |y|) as one v_max3_f32 with abs source modifiers.
__device__ __forceinline__ float max3_abs(float acc, float x, float y) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(acc), "v"(x), "v"(y));
  return r;
}

constexpr float kMagic128 = 12583040.0f;  // 1.5 * 2^23 + 128

template <int BITS, int D>
struct FastEnc {
  static constexpr int LPV = D / 32;               // lanes per vector
  static constexpr int VPW = 64 / LPV;             // vectors per wave (one group)
  static constexpr int RB = BITS == 8 ? D : D / 2; // code bytes per vector
  static constexpr int LB = RB / LPV;              // code bytes per lane (16 or 32)
  static constexpr float Q = BITS == 8 ? 127.0f : 7.0f;
};

// Stage h = 32 alone (lane ^ 1 through DPP quad_perm [1,0,3,2]) on eight registers, as in
// quad_stages8.
__device__ __forceinline__ void pair_stage8(float& a0, float& a1, float& a2, float& a3, float& a4, float& a5,
                                            float& a6, float& a7, float s32) {
  asm("s_nop 1\n"
      "v_fmac_f32_dpp %0, %0, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %1, %1, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %2, %2, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %3, %3, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %4, %4, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %5, %5, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %6, %6, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %7, %7, %8 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf"
      : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3), "+v"(a4), "+v"(a5), "+v"(a6), "+v"(a7)
      : "v"(s32));
}

// Encodes the 32 elements that this lane holds of one vector (lane part g of its LPV; 16 packed words of 16-bit elements,
// dm their diag sign masks: bit 15 the low element's, bit 31 the high one's) and ends with store(o, m), the lane's code
// bytes and the vector's m (the scale is m / Q).  Both ends of an interval around the quantiser's factor are tried; where
// they round apart the wave divides.  Where some lane's vector holds an infinity or a NaN, or lies beyond the range where
// the interval's ends are normal numbers, the wave ends with exact() instead, which takes encode_lane's sequence.
template <int DT, int BITS, int D, typename Exact, typename Store>
__device__ __forceinline__ void fast_encode_lane(const uint32_t (&w)[16], const uint32_t (&dm)[16], int g, float c, float cq,
                                                 Exact exact, Store store) {
  using F = FastEnc<BITS, D>;
  constexpr int LPV = F::LPV, NW = F::LB / 4;  // code dwords per lane
  float a[32];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    // stage h = 1 on x * diag: lo + hi, lo - hi
    float lo, hi;
    if constexpr (DT == AEKV_BF16) {
      lo = __builtin_bit_cast(float, (w[k] + dm[k]) << 16);
      hi = __builtin_bit_cast(float, __builtin_amdgcn_bitop3_b32(w[k], 0xFFFF0000u, dm[k], 0x48));
    } else {
      const uint32_t s = w[k] ^ dm[k];
      lo = f16_to_f32(s & 0xFFFFu);
      hi = f16_to_f32(s >> 16);
    }
    a[2 * k] = lo + hi;
    a[2 * k + 1] = lo - hi;
  }
#pragma unroll
  for (int h = 2; h < 32; h <<= 1) {
#pragma unroll
    for (int blk = 0; blk < 32; blk += 2 * h) {
#pragma unroll
      for (int i = 0; i < h; ++i) {
        const float p = a[blk + i], q = a[blk + h + i];
        a[blk + i] = p + q;
        a[blk + h + i] = p - q;
      }
    }
  }
  const float s32 = (g & 1) ? -1.0f : 1.0f;
  float sigma = s32;
  if constexpr (LPV == 4) {
    const float s64 = (g & 2) ? -1.0f : 1.0f;
    sigma = s32 * s64;
#pragma unroll
    for (int r = 0; r < 32; r += 8)
      quad_stages8(a[r], a[r + 1], a[r + 2], a[r + 3], a[r + 4], a[r + 5], a[r + 6], a[r + 7], s32, s64);
  } else {
#pragma unroll
    for (int r = 0; r < 32; r += 8)
      pair_stage8(a[r], a[r + 1], a[r + 2], a[r + 3], a[r + 4], a[r + 5], a[r + 6], a[r + 7], s32);
  }
  // m = max(RN(c max|raw|), 1e-8) over the LPV lanes of the vector
  float mr = 0.0f;
#pragma unroll
  for (int r = 0; r < 32; r += 2) mr = max3_abs(mr, a[r], a[r + 1]);
  mr = fmaxf(mr, xor_lane<1>(mr));
  if constexpr (LPV == 4) mr = fmaxf(mr, xor_lane<2>(mr));
  const float m = fmaxf(mr * c, 1e-8f);
  const float K = cq * __builtin_amdgcn_rcpf(m);
  const float klo = (K - K * 0x1.4p-21f) * sigma, khi = (K + K * 0x1.4p-21f) * sigma;
  constexpr float kMag = BITS == 8 ? kMagic128 : kMagic8;
  constexpr int EPW = BITS == 8 ? 4 : 8;  // elements per code dword
  uint32_t o[NW];
  uint32_t diff = 0u;
#pragma unroll
  for (int dw = 0; dw < NW; ++dw) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (BITS == 8) {
        const float x0 = a[EPW * dw + j];
        const uint32_t u0 = __builtin_bit_cast(uint32_t, fmaf(x0, klo, kMag));
        diff = __builtin_amdgcn_bitop3_b32(diff, u0, __builtin_bit_cast(uint32_t, fmaf(x0, khi, kMag)), 0xF6);
        b[j] = u0;
      } else {
        const float x0 = a[EPW * dw + 2 * j], x1 = a[EPW * dw + 2 * j + 1];
        const uint32_t u0 = __builtin_bit_cast(uint32_t, fmaf(x0, klo, kMag));
        const uint32_t u1 = __builtin_bit_cast(uint32_t, fmaf(x1, klo, kMag));
        diff = __builtin_amdgcn_bitop3_b32(diff, u0, __builtin_bit_cast(uint32_t, fmaf(x0, khi, kMag)), 0xF6);
        diff = __builtin_amdgcn_bitop3_b32(diff, u1, __builtin_bit_cast(uint32_t, fmaf(x1, khi, kMag)), 0xF6);
        b[j] = nib_pair(u0, u1);
      }
    }
    if constexpr (BITS == 8) {
      const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);  // [b0.0, b1.0, 0, 0]
      const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);  // [0, 0, b2.0, b3.0]
      o[dw] = (lo | hi) ^ 0x80808080u;
    } else {
      o[dw] = pack4(b[0], b[1], b[2], b[3]);
    }
  }
  // (every output sums every input, so a lane's first output shows an infinite or NaN input)
  // (2^100: K and its margin stay normal numbers)
  const bool odd = !(mr < 0x1p100f) || !(fabsf(a[0]) < __builtin_inff());
  if (__builtin_amdgcn_ballot_w64(odd) != 0) {
    exact();
    return;
  }
  if (__builtin_amdgcn_ballot_w64(diff != 0u) != 0) {  // some rounding the interval cannot decide
    float rlo = klo, rhi = khi;
    asm volatile("" : "+v"(rlo), "+v"(rhi));  // (the 64 products are formed again here, not kept in registers)
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const bool open = fmaf(a[e], rlo, kMag) != fmaf(a[e], rhi, kMag);
      if (__builtin_amdgcn_ballot_w64(open) == 0) continue;  // wave-uniform
      float t = ((a[e] * sigma) * c) / m;  // correctly rounded division, then * Q, rne
      t = fminf(fmaxf(rintf(t * F::Q), -F::Q), F::Q);
      constexpr int kBits = 32 / EPW;
      constexpr uint32_t kMask = BITS == 8 ? 0xFFu : 0xFu;
      const int sh = kBits * (e % EPW);
      const uint32_t code = (static_cast<uint32_t>(static_cast<int>(t)) & kMask) << sh;
      o[e / EPW] = open ? (o[e / EPW] & ~(kMask << sh)) | code : o[e / EPW];
    }
  }
  store(o, m);
}

}  // namespace
}  // namespace aekv
