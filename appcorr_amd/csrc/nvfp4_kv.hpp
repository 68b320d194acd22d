// K/V caches in NVFP4, as the kernels see them (format: nvfp4_kv.hip).
#pragma once

#include "nvfp4.hpp"
#include "packed_attn.hpp"

namespace oudjat {

// codes [B, N, 2, Hk, Dh / 2] and scales [B, N, 2, Hk, Dh / 16], strides in bytes, the last dims contiguous; ts [2, Hk].
struct KvNvfp4 {
  uint8_t* codes;
  int64_t bs, ns, cs, hs;
  uint8_t* scales;
  int64_t sbs, sns, scs, shs;
  const float* ts;
  int64_t B, N;
  int Hk;
};

// Strides and alignment of a cache; an OUDJAT status.
int check_kv_nvfp4(const KvNvfp4& c, int64_t Dh, const char* what);

}  // namespace oudjat
