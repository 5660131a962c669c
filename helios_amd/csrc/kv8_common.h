// Codes of the 8-bit KV cache, shared by the kernels that write, read and attend to it.
#pragma once

#include "hx_common.h"

namespace hx8 {

// e4m3 codes (largest 448) and whole numbers -127 .. 127. Both are exact in fp16 and in bf16.
struct E4m3 {
  static constexpr float kMost = 448.f;
};
struct Int8 {
  static constexpr float kMost = 127.f;
};

// Least scale of a row: its reciprocal and its logarithm stay ordinary fp32 numbers.
constexpr float kLeastScale = 0x1p-100f;

// Four values, each |x| <= kMost (1 + 2^-23), rounded to nearest even.
template <typename C>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d);
template <>
__device__ __forceinline__ uint32_t encode4<E4m3>(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
template <>
__device__ __forceinline__ uint32_t encode4<Int8>(float a, float b, float c, float d) {
  auto byte = [](float x) { return (uint32_t)(int)__builtin_rintf(x) & 0xffu; };
  return byte(a) | byte(b) << 8 | byte(c) << 16 | byte(d) << 24;
}

// Four codes widened to fp32, exactly.
template <typename C>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]);
template <>
__device__ __forceinline__ void decode4<E4m3>(uint32_t w, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0];
  x[1] = lo[1];
  x[2] = hi[0];
  x[3] = hi[1];
}
template <>
__device__ __forceinline__ void decode4<Int8>(uint32_t w, float (&x)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (float)(int)(int8_t)(w >> (8 * e));
}

// Four codes as two packed pairs of fp16, exactly. Whole numbers: with its sign turned a byte is
// c + 128; under the exponent of 1024 it is the number 1152 + c.
template <typename C>
__device__ __forceinline__ uint2 to_f16(uint32_t w);
template <>
__device__ __forceinline__ uint2 to_f16<E4m3>(uint32_t w) {
  return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)));
}
template <>
__device__ __forceinline__ uint2 to_f16<Int8>(uint32_t w) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const uint32_t u = w ^ 0x80808080u;
  const h2 off = {(_Float16)1152.f, (_Float16)1152.f};
  const h2 lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
  return make_uint2(__builtin_bit_cast(uint32_t, lo - off), __builtin_bit_cast(uint32_t, hi - off));
}

}  // namespace hx8
