// 16-bit element types of the operators that take bf16 or fp16.
#pragma once

#include "common.hpp"

namespace oudjat {

// 16-bit element types: E::to8 / E::from8 between a 16-byte chunk and eight floats.
struct ElemBf16 {
  static __device__ __forceinline__ void to8(const uint4& v, float* f) { unpack8(v, f); }
  static __device__ __forceinline__ uint4 from8(const float* f) { return pack8(f); }
};
struct ElemFp16 {
  typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void to8(const uint4& v, float* f) {
    const h8_t h = __builtin_bit_cast(h8_t, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
  }
  static __device__ __forceinline__ uint4 from8(const float* f) {
    h8_t h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)f[e];
    return __builtin_bit_cast(uint4, h);
  }
};

__device__ __forceinline__ uint4 load16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void store16(uint16_t* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

}  // namespace oudjat
