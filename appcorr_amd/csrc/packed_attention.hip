// Grouped-head attention of packed query rows over the keys of their own sequences, causal or not.
//
// Row r of sequence s (m rows, n keys) sees the keys j < n (causal: j <= n - m + i for its i-th row):
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * (q . k_j) - max_j ...)
// with the running maximum and sum of an online softmax in fp32. Hidden keys are not read, so whatever they hold
// has no influence; a row that sees none is 0.
//
// One wave per (row, query head): 64 keys at a time, a key per lane for the scores, then Dh / 64 dims per lane for
// the values.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace oudjat {

struct PackedAttn {
  const uint16_t* q;
  int64_t q_rs, q_hs;
  const uint16_t *k, *v;
  int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
  const void *cu_q, *keys;
  uint16_t* out;
  int64_t o_rs;
  int rows, S, Hq, G;
  int key_cap;
  bool cu_wide, keys_wide, batched, causal, fp16;
  float scale_log2;
};

__device__ __forceinline__ int64_t load_idx(const void* p, int i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ int clamp_idx(int64_t v, int lo, int hi) {
  return v < lo ? lo : (v > hi ? hi : (int)v);
}
__device__ __forceinline__ float elem(uint16_t x, bool fp16) {
  return fp16 ? (float)__builtin_bit_cast(_Float16, x) : bf16_to_f32(x);
}

template <int DH>
__global__ __launch_bounds__(256) void packed_attn_kernel(PackedAttn a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (int64_t)a.rows * a.Hq) return;
  const int row = (int)(unit / a.Hq), h = (int)(unit - (int64_t)row * a.Hq), hk = h / a.G;
  int lo = 0, hi = a.S;
  while (lo < hi) {  // first sequence that ends past the row
    const int mid = (lo + hi) >> 1;
    if (clamp_idx(load_idx(a.cu_q, mid + 1, a.cu_wide), 0, a.rows) > row) hi = mid;
    else lo = mid + 1;
  }
  const int s = lo;
  if (s >= a.S) return;
  const int q0 = clamp_idx(load_idx(a.cu_q, s, a.cu_wide), 0, a.rows);
  if (row < q0) return;
  const int m = clamp_idx(load_idx(a.cu_q, s + 1, a.cu_wide), q0, a.rows) - q0;
  int n, k0 = 0;
  if (a.batched) {
    n = clamp_idx(load_idx(a.keys, s, a.keys_wide), 0, a.key_cap);
  } else {
    k0 = clamp_idx(load_idx(a.keys, s, a.keys_wide), 0, a.key_cap);
    n = clamp_idx(load_idx(a.keys, s + 1, a.keys_wide), k0, a.key_cap) - k0;
  }
  const int lim = a.causal ? min(n, max(0, n - m + (row - q0) + 1)) : n;
  const uint16_t* qp = a.q + (int64_t)row * a.q_rs + (int64_t)h * a.q_hs;
  const uint16_t* kp = a.k + (a.batched ? (int64_t)s * a.k_bs : (int64_t)k0 * a.k_rs) + (int64_t)hk * a.k_hs;
  const uint16_t* vp = a.v + (a.batched ? (int64_t)s * a.v_bs : (int64_t)k0 * a.v_rs) + (int64_t)hk * a.v_hs;
  float o[DH / 64] = {}, mx = -INFINITY, l = 0.0f;
  for (int j0 = 0; j0 < lim; j0 += 64) {
    const int j = j0 + lane;
    float sc = -INFINITY;
    if (j < lim) {
      sc = 0.0f;
      const uint16_t* kr = kp + (int64_t)j * a.k_rs;
      for (int d = 0; d < DH; ++d) sc = fmaf(elem(qp[d], a.fp16), elem(kr[d], a.fp16), sc);
      sc *= a.scale_log2;
    }
    const float m_new = fmaxf(mx, wave_max(sc)), ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = exp2f(mx - ref), p = exp2f(sc - ref);
    l = l * alpha + wave_sum(p);
    mx = m_new;
    for (int e = 0; e < DH / 64; ++e) o[e] *= alpha;
    const int here = min(64, lim - j0);
    for (int i = 0; i < here; ++i) {
      const float pi = __shfl(p, i, 64);
      for (int e = 0; e < DH / 64; ++e)
        o[e] = fmaf(pi, elem(vp[(int64_t)(j0 + i) * a.v_rs + e * 64 + lane], a.fp16), o[e]);
    }
  }
  uint16_t* op = a.out + (int64_t)row * a.o_rs + (int64_t)h * DH;
  for (int e = 0; e < DH / 64; ++e) {
    const float y = lim ? o[e] / l : 0.0f;
    op[e * 64 + lane] = a.fp16 ? __builtin_bit_cast(uint16_t, (_Float16)y) : (uint16_t)f32_to_bf16(y);
  }
}

}  // namespace oudjat

using namespace oudjat;

extern "C" int64_t oudjat_packed_attention_workspace_elems(int64_t rows, int64_t S, int64_t Hq, int64_t Hk, int64_t Dh) {
  return 0;
}

extern "C" int oudjat_packed_attention(const uint16_t* q, int64_t q_rs, int64_t q_hs, int64_t rows, int64_t Hq, int64_t Dh,
                                       const uint16_t* k, int64_t k_bs, int64_t k_rs, int64_t k_hs, const uint16_t* v,
                                       int64_t v_bs, int64_t v_rs, int64_t v_hs, int64_t Hk, int64_t key_cap,
                                       int batched, const void* cu_q, int cu_wide, const void* keys, int keys_wide,
                                       int64_t S, float scale, int causal, int dtype, uint16_t* out, int64_t out_rs,
                                       float* workspace, int64_t workspace_elems, oudjat_stream_t stream) {
  const char* what = "packed_attention";
  OUDJAT_REQUIRE(rows >= 0 && S >= 0 && Hq > 0 && Hk > 0 && Dh > 0 && key_cap >= 0 && workspace_elems >= 0,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad size", what);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(std::isfinite(scale) && scale > 0.0f, OUDJAT_ERR_INVALID_ARGUMENT, "%s: scale must be positive", what);
  OUDJAT_REQUIRE(Dh == 64 || Dh == 128, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (64 or 128)", what, (long long)Dh);
  OUDJAT_REQUIRE(Hq % Hk == 0, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: %lld query heads over %lld key heads", what,
                 (long long)Hq, (long long)Hk);
  if (rows == 0 || S == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE(q && cu_q && keys && out && (key_cap == 0 || (k && v)), OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer",
                 what);
  OUDJAT_REQUIRE(q_rs >= 0 && q_hs >= 0 && k_bs >= 0 && k_rs >= 0 && k_hs >= 0 && v_bs >= 0 && v_rs >= 0 && v_hs >= 0 &&
                     out_rs >= 0,
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: negative stride", what);
  OUDJAT_REQUIRE(((q_rs | q_hs | k_bs | k_rs | k_hs | v_bs | v_rs | v_hs) % 8) == 0 && out_rs % 4 == 0 && aligned(q, 16) &&
                     aligned(k, 16) && aligned(v, 16) && aligned(out, 8) && aligned(cu_q, cu_wide ? 8 : 4) &&
                     aligned(keys, keys_wide ? 8 : 4),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned q, k and v rows and heads required", what);
  OUDJAT_REQUIRE(rows * (Hq / Hk) < (1 << 30) && Hq <= 65535 && S < (1 << 24) && key_cap < (1 << 30) &&
                     k_rs < (1 << 24) && v_rs < (1 << 24),
                 OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  PackedAttn a{q, q_rs, q_hs, k, v, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, cu_q, keys, out, out_rs, (int)rows, (int)S,
               (int)Hq, (int)(Hq / Hk), (int)key_cap, cu_wide != 0, keys_wide != 0, batched != 0, causal != 0,
               dtype == OUDJAT_FP16, scale * 1.4426950408889634f};
  const unsigned grid = (unsigned)cdiv(rows * Hq, 4);
  if (Dh == 64) packed_attn_kernel<64><<<grid, 256, 0, as_stream(stream)>>>(a);
  else packed_attn_kernel<128><<<grid, 256, 0, as_stream(stream)>>>(a);
  return check_launch(what);
}
