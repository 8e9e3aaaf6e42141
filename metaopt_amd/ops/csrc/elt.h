// 16-bit element types of the kernels that take bf16 and fp16 alike: conversions, packing (round
// to nearest even) and the matrix instructions of either type.
#pragma once
#include "common.h"

namespace mopt {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  static constexpr int kShift = 0;
  static __device__ __forceinline__ float up(uint32_t h) { return bf2f((bf16_t)h); }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return pack2bf(a, b); }
  // (a, b) minus the halves of p: a's difference is p . (-1, 0) + a, one instruction with no unpacking
  static __device__ __forceinline__ f32x2_t less2(float a, float b, uint32_t p) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    uint32_t lo = 0xBF80u, hi = 0xBF800000u;             // (-1, 0), (0, -1)
    asm("" : "+s"(lo), "+s"(hi));                        // (in registers, not as an f32 constant)
    return f32x2_t{__builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, p), __builtin_bit_cast(pair, lo), a, false),
                   __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, p), __builtin_bit_cast(pair, hi), b, false)};
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

struct Fp16 {
  // Probabilities of a long context lie among the subnormal fp16 values (below 2^-14, where a
  // rounding is no longer relative): the backward products take them 2^12 times as large.  (Score
  // gradients go with the incoming gradient's size: lm_window.hip scales them as they come.)
  static constexpr int kShift = 12;
  static __device__ __forceinline__ float up(uint32_t h) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_t));
  }
  static __device__ __forceinline__ f32x2_t less2(float a, float b, uint32_t p) {
    const f16x2_t h = __builtin_bit_cast(f16x2_t, p);
    return f32x2_t{fmaf((float)h[0], -1.f, a), fmaf((float)h[1], -1.f, b)};
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

template <class E>
__device__ __forceinline__ void up8(const u32x4& w, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = E::up(w[e] & 0xFFFF);
    f[2 * e + 1] = E::up(w[e] >> 16);
  }
}

template <class E>
__device__ __forceinline__ u32x4 down8(const float (&f)[8]) {
  return u32x4{E::pack2(f[0], f[1]), E::pack2(f[2], f[3]), E::pack2(f[4], f[5]),
               E::pack2(f[6], f[7])};
}

}  // namespace mopt
