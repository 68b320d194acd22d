// Helpers shared by the attention kernels: the online softmax's reference maximum, lane exchanges, and the LDS
// layout of key and value tiles.
#pragma once

#include "common.hpp"

namespace oudjat {

static constexpr int kKeyTile = 64;

typedef float f32x8_t __attribute__((ext_vector_type(8)));

// Eight fp32 -> bf16 (RNE) as four packed converts.
__device__ __forceinline__ bf16x8_t pack_bf16x8(const float* f) {
  const f32x8_t v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
  return __builtin_convertvector(v, bf16x8_t);
}

// Reference maximum of the online softmax: it moves to the running maximum only when that exceeds it
// by more than 8 in the exp2 domain (and always from -inf), so most tiles keep the same reference and
// skip rescaling the output; probabilities stay below 2^8 and the final O / l is unchanged.
__device__ __forceinline__ float softmax_ref_max(float m_ref, float tile_max, float scale_log2) {
  const float m_run = fmaxf(m_ref, tile_max);
  return (m_run - m_ref) * scale_log2 > 8.0f ? m_run : m_ref;
}

// Lane exchange with lane l ^ 32 through v_permlane32_swap (a VALU op, no LDS round trip): swapping
// the halves of two copies of x leaves x_l and x_{l^32} in the two results of every lane.
__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The same with lane l ^ 16 through v_permlane16_swap (rows of 16 lanes swapped pairwise).
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Slot of 16-byte chunk c in key row r of a tile: c ^ row_swz(r), so that 16 keys at one chunk (a K fragment
// read) cover all banks. Dh = 128: also the 4 keys x 4 chunks that half a wave's V transpose read takes
// (four consecutive keys differ in the chunk index above the 4 chunks).
template <int DH>
__device__ __forceinline__ int row_swz(int row) {
  return DH == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : row & 7;
}

// Slot of 16-byte chunk `chunk` in 128-byte key row `row`: chunk ^ sw(row), sw a permutation of the
// row pair m = (row >> 1) & 7 (so 16 consecutive keys at one chunk cover all 64 banks) that also
// flips bit 2 on odd pairs (so keys k and k + 2 -- one 4x16 transpose read -- use opposite halves
// of the row). sw(row + 16 j) = sw(row).
__device__ __forceinline__ int kv_swz(int row) {
  const int m = (row >> 1) & 7;
  return m ^ ((m & 1) << 2);
}
__device__ __forceinline__ int kv_slot(int row, int chunk) { return row * 128 + ((chunk ^ kv_swz(row)) << 4); }
// The same for 256-byte rows (Dh = 128).
template <int DH>
__device__ __forceinline__ int tile_swz(int row) {
  return DH == 128 ? row_swz<128>(row) : kv_swz(row);
}
template <int DH>
__device__ __forceinline__ int tile_slot(int row, int chunk) {
  return row * DH * 2 + ((chunk ^ tile_swz<DH>(row)) << 4);
}

}  // namespace oudjat
