// What the attention kernels over 16-bit keys and values share: the element types with their matrix instructions, and the
// layout of a tile of rows in LDS.
#pragma once

#include <type_traits>

#include "aekv_common.h"

namespace aekv {
namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMargin = 8.0f;        // log2 units a maximum moves before what it weighted is rescaled
constexpr float kFar = 0x1p22f;        // log2 units: below, a logit is rounded by a quarter at most
constexpr int kBufWord3 = 0x00020000;  // buffer resource word 3: raw 32-bit data, range-checked

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short i16x4_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
typedef __attribute__((address_space(3))) void lds_void_t;

template <int DT>
struct Elem;
template <>
struct Elem<AEKV_BF16> {
  typedef bf16x8_t v8;
  static constexpr uint32_t kExp = 0x7F80u;  // infinity; NaN above it
  static constexpr float kLift = 0.0f;       // log2 of what a weight at the reference is held as
  __device__ static f32x16_t mma(v8 a, v8 b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  __device__ static f32x4_t mma16(v8 a, v8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  __device__ static float value(uint32_t u) { return bf16_to_f32(u); }
};
template <>
struct Elem<AEKV_F16> {
  typedef f16x8_t v8;
  static constexpr uint32_t kExp = 0x7C00u;
  static constexpr float kLift = 7.0f;  // (kMargin more and 2^15 is below the largest)
  __device__ static f32x16_t mma(v8 a, v8 b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  __device__ static f32x4_t mma16(v8 a, v8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  __device__ static float value(uint32_t u) { return f16_to_f32(u); }
};

// Chunk c of key r lies at c ^ swizzle(r) of its row.  256-byte rows: 16 keys' equal chunks fall on 16 places, and 4 keys
// (4 i ..) x 4 chunks as well; 128-byte rows, two of which share the 256 bytes of all banks, likewise.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

__device__ __forceinline__ i16x4_t read_tr16(const uint8_t* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p)); }

}  // namespace
}  // namespace aekv
