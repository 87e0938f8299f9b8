// MXFP4: blocks of 32 consecutive numbers share a power of two.  A number is code * 2^(byte - 127):
// the code is e2m1 (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6 and their
// negatives), two codes to a byte, the lower index in the lower four bits; the scale byte is e8m0,
// 255 marks a block that held an infinity or a NaN (every number of it is then a NaN).
#pragma once

#include "common.h"

namespace afir {

enum ElemKind { kElemF32 = 0, kElemF16 = 1, kElemBF16 = 2 };   // the elem_type field of the operators' tiling data

constexpr int kMxBlock = 32;        // numbers that share a scale
constexpr int kMxBlockBytes = 16;   // their codes

// Scale byte of a block whose largest magnitude has the float32 bits `top`: the exponent of the
// largest power of two not above it, less two, so that the block's largest number lands in [4, 8)
// before it is rounded and what lies above 6 saturates.  Biased exponents 0 to 2 (and blocks of
// zeros) take the smallest scale, 2^-127.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t biased = top >> 23;
  return biased == 255u ? 255u : (biased > 2u ? biased - 2u : 0u);
}
// 2^(byte - 127) as float32 (byte 0: a denormal).  A block marked 255 is coded with zeros; its
// scale reads as infinity here and is not used.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// Eight floats -> eight codes.  The conversion divides by the scale, rounds to nearest even and
// saturates at 6 in one step.
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}
// ... and back: the numbers the codes stand for, exact in float32, f16 and bf16 whenever the
// block's own numbers were of that type (a rounded number is a multiple of the same step)
__device__ __forceinline__ void mx_decode8(uint32_t w, float scale, float (&v)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// Storage types.  The vector accesses are declared with the alignment of one element: global
// accesses of 16 bytes need none beyond that on this target, so rows of odd length take the same
// path as aligned ones.
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));
typedef uint32_t u32_u __attribute__((aligned(2)));

template <int KIND>
struct Elem;
template <>
struct Elem<kElemF32> {
  typedef float type;
  static constexpr int kPer16 = 4;
  __device__ static float load(const void *p, int64_t i) { return static_cast<const float *>(p)[i]; }
  __device__ static void store(void *p, int64_t i, float v) { static_cast<float *>(p)[i] = v; }
  // the `N` numbers of N / 4 16-byte words
  template <int N>
  __device__ static void unpack(const uint32_t (&w)[N], float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
  }
  template <int N>
  __device__ static void pack(const float (&v)[N], uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
  }
};
template <>
struct Elem<kElemF16> {
  typedef uint16_t type;
  static constexpr int kPer16 = 8;
  __device__ static float load(const void *p, int64_t i) { return f16_lo(static_cast<const uint16_t *>(p)[i]); }
  __device__ static void store(void *p, int64_t i, float v) {
    static_cast<uint16_t *>(p)[i] = (uint16_t)pack_f16(v, 0.f);
  }
  template <int W, int N>
  __device__ static void unpack(const uint32_t (&w)[W], float (&v)[N]) {
    static_assert(N == 2 * W, "two to a word");
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[2 * i] = f16_lo(w[i]);
      v[2 * i + 1] = f16_hi(w[i]);
    }
  }
  template <int W, int N>
  __device__ static void pack(const float (&v)[N], uint32_t (&w)[W]) {
    static_assert(N == 2 * W, "two to a word");
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = pack_f16(v[2 * i], v[2 * i + 1]);
  }
};
template <>
struct Elem<kElemBF16> {
  typedef uint16_t type;
  static constexpr int kPer16 = 8;
  __device__ static float load(const void *p, int64_t i) { return bf16_lo(static_cast<const uint16_t *>(p)[i]); }
  __device__ static void store(void *p, int64_t i, float v) {
    static_cast<uint16_t *>(p)[i] = (uint16_t)pack_bf16_hw(v, 0.f);
  }
  template <int W, int N>
  __device__ static void unpack(const uint32_t (&w)[W], float (&v)[N]) {
    static_assert(N == 2 * W, "two to a word");
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  template <int W, int N>
  __device__ static void pack(const float (&v)[N], uint32_t (&w)[W]) {
    static_assert(N == 2 * W, "two to a word");
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = pack_bf16_hw(v[2 * i], v[2 * i + 1]);
  }
};

}  // namespace afir
