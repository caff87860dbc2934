// Rows held in 4 bits, shared by fp4.hip and fp4_attention.hip: groups of 32
// values, each 16 bytes of codes (the lower half of a byte first) and one scale
// byte s.  A code is a sign, two bits of exponent and one of fraction: 0, 0.5, 1,
// 1.5, 2, 3, 4 or 6, times 2^(s - 127); s = 255 makes the whole group NaN.  This
// is the OCP microscaling format MXFP4.  CDNA4 converts two codes under a scale
// in one instruction, and their values are exact in BF16.
#pragma once

#include <cstdint>

#include "dl_device.h"
#include "dl_internal.h"

namespace dl::fp4 {

constexpr int kGroup = 32, kGroupBytes = 16;
constexpr uint32_t kNanScale = 255;
// Largest scale byte that quantising gives: 6 * 2^(252 - 127) is still finite.
constexpr uint32_t kMostScale = 252;

inline uint64_t groups_of(uint64_t width) { return ceil_div(width, kGroup); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The conversions read a scale's exponent field alone: the scale byte's bits as
// they are, 2^-127 among them, and NaN for 255.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes to eight BF16 values in order.
__device__ __forceinline__ u32x4 to_bf16(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// FP32 values as the exact sum of three BF16 values each (8 significant bits at a
// time), for products on the BF16 matrix cores that round nothing.  A value that
// is not finite is its first part alone.
__device__ __forceinline__ void split(float v, uint32_t (&part)[3]) {  // in the upper halves
  const bool finite = fabsf(v) < INFINITY;
  part[0] = v == v ? __float_as_uint(v) & 0xffff0000u : 0x7fc00000u;
  const float rest = finite ? v - __uint_as_float(part[0]) : 0.0f;
  part[1] = __float_as_uint(rest) & 0xffff0000u;
  part[2] = __float_as_uint(rest - __uint_as_float(part[1]));
}
struct Parts {
  u32x4 part[3];
};
__device__ __forceinline__ Parts split(const float (&x)[8]) {
  Parts p;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t lo[3], hi[3];
    split(x[2 * w], lo);
    split(x[2 * w + 1], hi);
#pragma unroll
    for (int i = 0; i < 3; ++i) p.part[i][w] = __builtin_amdgcn_perm(hi[i], lo[i], 0x07060302u);
  }
  return p;
}

// The scale byte of a group whose largest magnitude has these FP32 bits: the power
// of two under which it lies in [3.5, 7), so that no value passes 6, the largest
// code, by more than half of the step there; kNanScale if a value is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  if (largest >= 0x7f800000u) return kNanScale;
  const int32_t s = static_cast<int32_t>((largest + 0x200000u) >> 23) - 2;
  return static_cast<uint32_t>(min(max(s, 0), static_cast<int32_t>(kMostScale)));
}

// Eight values to eight codes: to nearest, ties to the even code, 6 at most.
__device__ __forceinline__ uint32_t to_codes(const float (&x)[8], uint32_t byte) {
  if (byte == kNanScale) return 0;
  const float by = scale_of(byte);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], by, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], by, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], by, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], by, 3);
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Eight consecutive elements of a row that has `width`, from `at` on; zeros past
// the width.  Pieces: the row is whole 16-byte pieces.
template <class T, bool kPieces>
__device__ __forceinline__ void load_eight(const T* row, uint32_t at, uint32_t width, float (&x)[8]) {
  if constexpr (kPieces) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
      const u32x4 v = at + i * kPer < width ? *reinterpret_cast<const u32x4*>(row + at + i * kPer) : u32x4{};
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if constexpr (sizeof(T) == 4)
          x[i * kPer + e] = __uint_as_float(v[e]);
        else
          x[i * kPer + e] = e % 2 ? dl_bf16_hi(v[e / 2]) : dl_bf16_lo(v[e / 2]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = at + e < width ? load_elem(row, at + e) : 0.0f;
  }
}

// s_waitcnt immediate: at most n vector-memory operations and no LDS operation
// outstanding.
constexpr unsigned lds_wait(unsigned n) { return vm_wait(n) & ~0x0f00u; }

// Four consecutive outputs of a row.
template <class T>
__device__ __forceinline__ void store_four(T* to, const f32x4& v, uint64_t left, bool whole) {
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  } four;
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(four.v, e, v[e]);
  if (whole && left >= 4) {
    *reinterpret_cast<Four*>(to) = four;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (static_cast<uint64_t>(e) < left) to[e] = four.v[e];
  }
}

}  // namespace dl::fp4
