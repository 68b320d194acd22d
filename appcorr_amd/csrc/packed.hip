// Rows of sequences of different lengths, packed one after another: their offsets and cache slots from the
// sequences' lengths, the rotation of q and k by positions with several axes, and the per-head norm of q and k
// with that rotation and the K/V write in one pass. The attention over such rows is in packed_attention.hip.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace oudjat {

// ------------------------------------------------------------------------------------------------
// packed_plan. With nq_s = max(q_lens[s], 0), nk_s = max(k_lens[s], 0) and the offsets c_s = min(sum of nq before s,
// rows), sequence s has rows c_s .. c_{s+1} - 1, the first of its new rows where the buffer ends inside them. A
// sequence's new rows are its last tokens, so row r is token first_s + r - c_s, first_s = nk_s - nq_s, and the keys that
// go with the rows that are there are n_s = max(0, first_s + c_{s+1} - c_s). A token has a slot where it is not negative
// and below cache_len. Packed keys: sequence s has key rows from the sum of n before it on, if all n_s fit into
// key_rows, else none, and its rows no slots.
// Every workgroup scans all lengths for itself (at most kPlanMaxSeqs of them, read from L2, offsets in LDS) and
// then looks its own rows up by bisection, so that the plan is one launch and no workgroup waits for another.
// Bound by that scan's latency: a thread reads its lengths eight at a time, scans within its wave by lane
// shuffles and across waves through LDS.
// ------------------------------------------------------------------------------------------------
static constexpr int kPlanThreads = 256;
static constexpr int kPlanMaxSeqs = 4096;     // 2 x 16 KB of LDS
static constexpr int kPlanRowsPerThread = 2;  // one 16-byte store to each of the two maps

__device__ __forceinline__ int64_t load_len(const void* p, int i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ int64_t clamp_len(int64_t v, int64_t hi) { return v < 0 ? 0 : (v < hi ? v : hi); }

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) {
  const uint32_t lo = __shfl_up((uint32_t)v, d, 64), hi = __shfl_up((uint32_t)((uint64_t)v >> 32), d, 64);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sums before this thread over the workgroup (exclusive), and the total, of one value per thread.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* wave_sums, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = shfl_up64(incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 63) wave_sums[wave] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(
    const void* __restrict__ q_lens, int q_wide, const void* __restrict__ k_lens, int k_wide, int S, int64_t rows,
    int64_t key_cap, int packed_keys, int32_t* __restrict__ cu_q, int32_t* __restrict__ k_out,
    int64_t* __restrict__ cu_k, int64_t* __restrict__ batch_idx, int64_t* __restrict__ token_idx) {
  extern __shared__ int32_t plan_lds[];
  int32_t* ends = plan_lds;         // c_{s+1}
  int32_t* toks = plan_lds + S;     // first_s - c_s: token of row r is toks[s] + r; INT32_MIN: no row has a slot
  __shared__ int64_t wave_sums[kPlanThreads / 64];
  __shared__ int32_t last_fit;      // packed keys: the key rows before the first sequence that does not fit
  const int tid = threadIdx.x;
  const int per = (S + kPlanThreads - 1) / kPlanThreads;
  const int s0 = min(tid * per, S), s1 = min(s0 + per, S);
  int64_t nq = 0, nk = 0, total, a[8], b[8];
  auto load = [&](int s) {  // lengths of sequences s .. s + 7
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = min(s + e, S - 1);
      a[e] = load_len(q_lens, i, q_wide);
      b[e] = load_len(k_lens, i, k_wide);
    }
  };
  for (int s = s0; s < s1; s += 8) {
    load(s);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (s + e < s1) nq += clamp_len(a[e], rows);
  }
  int64_t cq = block_scan(nq, wave_sums, &total);
  const int begin0 = (int)min(cq, rows);
  auto keys = [&](int64_t q, int64_t k, int64_t kept) {  // n_s
    return max(max(k, (int64_t)0) - max(q, (int64_t)0) + kept, (int64_t)0);
  };
  // n_s in the running sum: what a cache holds of them, or (packed) all, as far as it matters that they do not fit.
  const int64_t most = packed_keys ? key_cap + 1 : key_cap;
  auto take = [&](int s, int64_t q, int64_t k) {
    const int64_t begin = min(cq, rows);
    cq += clamp_len(q, rows);
    const int64_t end = min(cq, rows), n = keys(q, k, end - begin), first = n - (end - begin);
    nk += min(n, most);
    ends[s] = (int32_t)end;
    toks[s] = n > 0 && first < key_cap ? (int32_t)(first - begin) : INT32_MIN;  // (n > 0: first > -end)
  };
  if (per == 1) {  // up to 256 sequences
    if (s0 < s1) take(s0, a[0], b[0]);
  } else {
    for (int s = s0; s < s1; s += 8) {
      load(s);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (s + e < s1) take(s + e, a[e], b[e]);
    }
  }
  int64_t ck = block_scan(nk, wave_sums, &total);
  const bool writer = blockIdx.x == 0;  // the per-sequence results are written once
  int past = s1;                        // packed keys: this thread's first sequence that does not fit
  if (packed_keys || writer) {
    int begin = begin0;
    for (int s = s0; s < s1; ++s) {
      const int end = ends[s], t = toks[s];
      const int64_t n = t != INT32_MIN ? (int64_t)t + end
                                       : keys(load_len(q_lens, s, q_wide), load_len(k_lens, s, k_wide), end - begin);
      const int64_t before = ck;
      begin = end;
      ck += min(n, most);
      const bool fits = !packed_keys || ck <= key_cap;
      if (!fits) {
        toks[s] = INT32_MIN;
        past = min(past, s);
        if (before <= key_cap) last_fit = (int32_t)before;  // (one sequence of all)
      }
      if (writer) {
        cu_q[s + 1] = end;
        k_out[s] = fits ? (int32_t)min(n, (int64_t)INT32_MAX) : 0;
        if (fits) cu_k[s + 1] = ck;
      }
    }
    if (writer && tid == 0) {
      cu_q[0] = 0;
      cu_k[0] = 0;
    }
  }
  __syncthreads();
  if (writer)
    for (int s = past; s < s1; ++s) cu_k[s + 1] = last_fit;
  const int64_t r0 = ((int64_t)blockIdx.x * kPlanThreads + tid) * kPlanRowsPerThread;
  if (r0 >= rows) return;
  int64_t bi[kPlanRowsPerThread], ti[kPlanRowsPerThread];
#pragma unroll
  for (int e = 0; e < kPlanRowsPerThread; ++e) {
    const int r = (int)r0 + e;  // rows < 2^31 - 1: no overflow
    int lo = 0, hi = S;         // first s with ends[s] > r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    const int64_t t = lo < S ? (int64_t)toks[lo] + r : -1;
    const bool slot = t >= 0 && t < key_cap;
    bi[e] = slot ? lo : -1;
    ti[e] = slot ? t : -1;
  }
  if (r0 + 1 < rows) {
    typedef int64_t i64x2_t __attribute__((ext_vector_type(2)));
    *reinterpret_cast<i64x2_t*>(batch_idx + r0) = i64x2_t{bi[0], bi[1]};
    *reinterpret_cast<i64x2_t*>(token_idx + r0) = i64x2_t{ti[0], ti[1]};
  } else {
    batch_idx[r0] = bi[0];
    token_idx[r0] = ti[0];
  }
}

// ------------------------------------------------------------------------------------------------
// Rotation by positions. Of a head's dims, the first R are rotated in pairs (i, i + R/2), pair i by the angle
// pos[row, axis(i)] * inv_freq[i]; axis(i) is the section that i falls into (sections: how many consecutive
// frequencies each axis has). The angle is formed in 64 bits and reduced to a fraction of a turn before it is
// rounded: at position 2^20 and frequency 1 a 32-bit product is off by 2^-4 of a radian. A row's sines and
// cosines are computed once, one pair per thread, and shared by its heads through LDS.
// ------------------------------------------------------------------------------------------------
static constexpr int kRopeThreads = 256;
static constexpr int kMaxAxes = 4;

struct AxisRope {
  const void* pos;      // [rows, axes], any strides
  int64_t pos_rs, pos_as;
  int pos_kind;         // 0 int32, 1 int64, 2 fp32
  const float* inv_freq;
  int half;             // R / 2
  int end[kMaxAxes];    // first pair past axis a's section
};

__device__ __forceinline__ void axis_sincos(const AxisRope& a, int64_t row, int pair, float* sn, float* cs) {
  int axis = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes - 1; ++i) axis += pair >= a.end[i];
  const int64_t at = row * a.pos_rs + axis * a.pos_as;
  const double p = a.pos_kind == 0   ? (double)static_cast<const int32_t*>(a.pos)[at]
                   : a.pos_kind == 1 ? (double)static_cast<const int64_t*>(a.pos)[at]
                                     : (double)static_cast<const float*>(a.pos)[at];
  const double turns = p * (double)a.inv_freq[pair] * 0.15915494309189533577;  // 1 / (2 pi)
  const float half_turns = (float)(2.0 * (turns - rint(turns)));               // -1 .. 1
  sincospif(half_turns, sn, cs);
}

// Cosines and sines of rows row0 .. row0 + n - 1 to lds [n][2][half], one (row, pair) per thread.
__device__ __forceinline__ void fill_rope_table(const AxisRope& a, float* lds, int64_t row0, int n) {
  for (int i = threadIdx.x; i < n * a.half; i += kRopeThreads) {
    const int r = i / a.half, p = i - r * a.half;
    float sn, cs;
    axis_sincos(a, row0 + r, p, &sn, &cs);
    lds[(2 * r) * a.half + p] = cs;
    lds[(2 * r + 1) * a.half + p] = sn;
  }
}

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

// A workgroup takes `per_wg` rows: (row, head, 16 dims) items, one per thread: chunk pair c < R/16 holds dims 8c .. and
// R/2 + 8c .., the others 16 dims that are copied. Every q and k element is read and written once; an item's loads
// and stores do not depend on another's, so in place is fine. Bound by HBM: a thread has U items' loads in flight,
// the first of them while the rows' sines and cosines are computed (16404 rows, 32 + 8 heads of 128, 336 MB: U = 1
// 76 us, 4 70 us, 4.8 TB/s, 6 71 us; a copy of 2 GB runs at 4.9). U = 1 where a workgroup has one item per thread.
template <class E, int U>
__global__ __launch_bounds__(kRopeThreads) void rope_axes_kernel(
    AxisRope a, const uint16_t* q, int64_t q_rs, int64_t q_hs, const uint16_t* k, int64_t k_rs, int64_t k_hs,
    uint16_t* qo, int64_t qo_rs, int64_t qo_hs, uint16_t* ko, int64_t ko_rs, int64_t ko_hs, int64_t rows, int Hq,
    int Hk, int Dh, int per_wg) {
  extern __shared__ __align__(16) float rope_lds[];
  const int half = a.half, tid = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * per_wg;
  const int n = (int)min((int64_t)per_wg, rows - row0);
  const int cph = Dh / 16, H = Hq + Hk, items = n * H * cph, rot = half / 8;
  uint4 x0[U], x1[U];
  uint16_t* dst[U];
  int r[U], c[U];
  auto first = [&](int u) { return c[u] < rot ? 8 * c[u] : 16 * c[u]; };
  auto second = [&](int u) { return c[u] < rot ? half + 8 * c[u] : 16 * c[u] + 8; };
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * kRopeThreads, items - 1);
      const int rh = i / cph;
      c[u] = i - rh * cph;
      r[u] = rh / H;
      const int h = rh - r[u] * H;
      const int64_t row = row0 + r[u];
      const bool is_q = h < Hq;
      const uint16_t* src = is_q ? q + row * q_rs + h * q_hs : k + row * k_rs + (h - Hq) * k_hs;
      dst[u] = is_q ? qo + row * qo_rs + h * qo_hs : ko + row * ko_rs + (h - Hq) * ko_hs;
      x0[u] = load16(src + first(u));
      x1[u] = load16(src + second(u));
    }
  };
  load(tid);
  fill_rope_table(a, rope_lds, row0, n);
  __syncthreads();
  for (int i0 = tid; i0 < items; i0 += kRopeThreads * U) {
    if (i0 != tid) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * kRopeThreads >= items) break;
      if (c[u] < rot) {
        const float* cs = rope_lds + (2 * r[u]) * half + 8 * c[u];
        float l[8], g[8], cv[8], sv[8];
        E::to8(x0[u], l);
        E::to8(x1[u], g);
        load8f(cs, cv);
        load8f(cs + half, sv);
        rope8(l, g, cv, cv, sv, sv);
        x0[u] = E::from8(l);
        x1[u] = E::from8(g);
      }
      store16(dst[u] + first(u), x0[u]);
      store16(dst[u] + second(u), x1[u]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Norm of every q and k head, rotation, K/V write. qkv row: Hq query heads, Hk key heads, Hk value heads of Dh.
// RMS: y = x / sqrt(mean(x^2) + eps) * w;  LayerNorm: the same of x - mean(x), plus b. Then the rotation, then one
// rounding to the type; values are copied. Dh / 16 lanes hold a head, 16 dims each (as above), so that its sums
// are two to three lane exchanges, and a thread keeps the weights of its dims for all heads it takes. A row whose
// slot lies outside the cache is skipped. Bound by HBM: 16404 rows, 32 + 2 x 8 heads of 128, 398 MB, 81.8 us
// (4.87 TB/s); one token of 32 streams 4.7 us, a launch and two dependent rounds of loads; the branch for heads out of
// fp32's range costs 0.1 us of it.
// ------------------------------------------------------------------------------------------------
template <class E, int DH, bool LAYER>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kv_kernel(
    AxisRope a, const uint16_t* __restrict__ qkv, int64_t x_rs, int64_t rows, int Hq, int Hk,
    const uint16_t* __restrict__ qw, const uint16_t* __restrict__ qb, const uint16_t* __restrict__ kw,
    const uint16_t* __restrict__ kb, float eps, const int64_t* __restrict__ batch_idx,
    const int64_t* __restrict__ token_idx, uint16_t* __restrict__ kv, int64_t kv_bs, int64_t kv_ns, int64_t kv_cs,
    int64_t B, int64_t N, uint16_t* __restrict__ qo, int64_t qo_rs, int per_wg) {
  constexpr int L = DH / 16;  // lanes of a head
  extern __shared__ __align__(16) float rope_lds[];  // [per_wg][2][half]
  const int half = a.half, tid = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * per_wg;
  const int n = (int)min((int64_t)per_wg, rows - row0);
  const int c = tid % L, rot = half / 8;
  const bool turned = c < rot;
  const int d0 = turned ? 8 * c : 16 * c, d1 = turned ? half + 8 * c : 16 * c + 8;
  const uint4 one = E::from8((const float[8]){1, 1, 1, 1, 1, 1, 1, 1}), zero = make_uint4(0, 0, 0, 0);
  uint4 w[2][2], b[2][2];  // [q, k][chunk]
  w[0][0] = qw ? load16(qw + d0) : one;
  w[0][1] = qw ? load16(qw + d1) : one;
  w[1][0] = kw ? load16(kw + d0) : one;
  w[1][1] = kw ? load16(kw + d1) : one;
  if constexpr (LAYER) {
    b[0][0] = qb ? load16(qb + d0) : zero;
    b[0][1] = qb ? load16(qb + d1) : zero;
    b[1][0] = kb ? load16(kb + d0) : zero;
    b[1][1] = kb ? load16(kb + d1) : zero;
  }
  const int H = Hq + 2 * Hk, heads = n * H;
  int r, h;
  int64_t row, bi, ti;
  uint4 x0, x1;
  auto load = [&](int i) {  // (head i of the workgroup's rows, the last one where there is none)
    i = min(i, heads - 1);
    r = i / H;
    h = i - r * H;
    row = row0 + r;
    const uint16_t* src = qkv + row * x_rs + (int64_t)h * DH;
    x0 = load16(src + d0);
    x1 = load16(src + d1);
    bi = batch_idx[row];
    ti = token_idx[row];
  };
  load(tid / L);
  fill_rope_table(a, rope_lds, row0, n);
  __syncthreads();
  for (int i = tid / L; i < heads; i += kRopeThreads / L) {  // the L lanes of a head stay together
    if (i != tid / L) load(i);
    if (bi < 0 || bi >= B || ti < 0 || ti >= N) continue;
    uint16_t* dst;
    if (h < Hq) dst = qo + row * qo_rs + (int64_t)h * DH;
    else {
      const int hk = h < Hq + Hk ? h - Hq : h - Hq - Hk;
      dst = kv + bi * kv_bs + ti * kv_ns + (h < Hq + Hk ? 0 : kv_cs) + (int64_t)hk * DH;
    }
    if (h < Hq + Hk) {
      float x[16], y[16];
      E::to8(x0, x);
      E::to8(x1, x + 8);
      // mean(x^2) + eps of the head's values (LayerNorm: less their mean, which is taken off x).
      auto variance = [&](float eps_) {
        if constexpr (LAYER) {
          float s = 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e) s += x[e];
#pragma unroll
          for (int d = L / 2; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
          s *= 1.0f / DH;
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] -= s;
        }
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) ss += __shfl_xor(ss, d, 64);
        return fmaf(ss, 1.0f / DH, eps_);
      };
      float var = variance(eps);
      if (!(var > 0x1p-100f && var < 0x1p126f)) {
        // Sums or squares that leave fp32's range (bf16 values from 1e19 on; below 1e-15 where eps is as small): the head
        // again, scaled by a power of two that takes its largest value to 1 .. 4, or from far below towards it.
        E::to8(x0, x);
        E::to8(x1, x + 8);
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        const int exponent = (int)(__float_as_uint(top) >> 23) - 127;
        const float scale = ldexpf(1.0f, -max(var < 1.0f ? -100 : 0, min(126, exponent)));  // (eps scale^2 is finite)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= scale;
        var = variance(eps * scale * scale);
      }
      const float inv = 1.0f / sqrtf(var);
      const int which = h < Hq ? 0 : 1;
      E::to8(which ? w[1][0] : w[0][0], y);
      E::to8(which ? w[1][1] : w[0][1], y + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = x[e] * inv * y[e];
      if constexpr (LAYER) {
        E::to8(which ? b[1][0] : b[0][0], y);
        E::to8(which ? b[1][1] : b[0][1], y + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] += y[e];
      }
      if (turned) {
        float cv[8], sv[8];
        load8f(rope_lds + (2 * r) * half + 8 * c, cv);
        load8f(rope_lds + (2 * r + 1) * half + 8 * c, sv);
        rope8(x, x + 8, cv, cv, sv, sv);
      }
      x0 = E::from8(x);
      x1 = E::from8(x + 8);
    }
    store16(dst + d0, x0);
    store16(dst + d1, x1);
  }
}

// Rows a workgroup takes: one while few (latency), else as many as its threads have pairs for. Measured (us, one row a
// workgroup -> 256 / half rows; 32 + 8 heads of 128, rope and norm): 512 rows 5.7 -> 7.1 and 6.1 -> 10.1, 2048 rows
// 12.9 -> 11.0 and 13.7 -> 15.2, 16404 rows 77 -> 72 and 82 -> 83; 6 + 6 heads of 64, 16404 rows 24 -> 15 and 30 -> 19.
static int rope_rows_per_wg(int64_t rows, int half) {
  return rows < 2048 ? 1 : std::max(1, kRopeThreads / half);
}

static int make_axis_rope(AxisRope* a, const void* pos, int pos_kind, int64_t pos_rs, int64_t pos_as, int64_t axes,
                          const float* inv_freq, const int64_t* sections, int64_t Dh, const char* what) {
  OUDJAT_REQUIRE(pos && inv_freq && sections, OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(pos_kind >= 0 && pos_kind <= 2, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad position type %d", what, pos_kind);
  OUDJAT_REQUIRE(axes >= 1 && axes <= kMaxAxes, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: %lld axes (1 to %d)", what,
                 (long long)axes, kMaxAxes);
  int64_t half = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    const int64_t n = i < axes ? sections[i] : 0;
    OUDJAT_REQUIRE(n >= 0 && n <= Dh, OUDJAT_ERR_INVALID_ARGUMENT, "%s: section of %lld frequencies", what, (long long)n);
    half += n;
    a->end[i] = i < axes - 1 ? (int)half : INT32_MAX;  // the last axis takes the rest
  }
  OUDJAT_REQUIRE(half > 0 && half % 8 == 0 && 2 * half <= Dh, OUDJAT_ERR_UNSUPPORTED_SHAPE,
                 "%s: %lld frequencies (a multiple of 8 up to Dh / 2)", what, (long long)half);
  OUDJAT_REQUIRE(aligned(pos, pos_kind == 1 ? 8 : 4) && aligned(inv_freq, 4), OUDJAT_ERR_UNSUPPORTED_LAYOUT,
                 "%s: unaligned positions or frequencies", what);
  a->pos = pos;
  a->pos_rs = pos_rs;
  a->pos_as = pos_as;
  a->pos_kind = pos_kind;
  a->inv_freq = inv_freq;
  a->half = (int)half;
  return OUDJAT_OK;
}

}  // namespace oudjat

using namespace oudjat;

extern "C" int oudjat_packed_plan(const void* q_lens, int q_wide, const void* k_lens, int k_wide, int64_t S, int64_t rows,
                                  int64_t key_cap, int packed_keys, int32_t* cu_q, int32_t* k_out, int64_t* cu_k,
                                  int64_t* batch_idx, int64_t* token_idx, oudjat_stream_t stream) {
  const char* what = "packed_plan";
  OUDJAT_REQUIRE(S >= 0 && rows >= 0 && key_cap >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  OUDJAT_REQUIRE(S <= kPlanMaxSeqs && rows < INT32_MAX && key_cap < INT32_MAX, OUDJAT_ERR_TOO_LARGE,
                 "%s: at most %d sequences, fewer than 2^31 - 1 rows and keys", what, kPlanMaxSeqs);
  OUDJAT_REQUIRE(cu_q && cu_k && (S == 0 || (q_lens && k_lens && k_out)) && (rows == 0 || (batch_idx && token_idx)),
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(aligned(q_lens, q_wide ? 8 : 4) && aligned(k_lens, k_wide ? 8 : 4) && aligned(cu_q, 4) &&
                     aligned(k_out, 4) && aligned(cu_k, 8) && aligned(batch_idx, 16) && aligned(token_idx, 16),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: unaligned tensor (16 bytes for the row maps)", what);
  const int64_t grid = std::max<int64_t>(1, cdiv(rows, kPlanThreads * kPlanRowsPerThread));
  packed_plan_kernel<<<(unsigned)grid, kPlanThreads, (size_t)S * 8, as_stream(stream)>>>(
      q_lens, q_wide, k_lens, k_wide, (int)S, rows, key_cap, packed_keys, cu_q, k_out, cu_k, batch_idx, token_idx);
  return check_launch(what);
}

extern "C" int oudjat_rope_axes(const uint16_t* q, int64_t q_rs, int64_t q_hs, const uint16_t* k, int64_t k_rs,
                                int64_t k_hs, int64_t rows, int64_t Hq, int64_t Hk, int64_t Dh, int dtype,
                                const void* pos, int pos_kind, int64_t pos_rs, int64_t pos_as, int64_t axes,
                                const float* inv_freq, const int64_t* sections, uint16_t* q_out, int64_t qo_rs,
                                int64_t qo_hs, uint16_t* k_out, int64_t ko_rs, int64_t ko_hs, oudjat_stream_t stream) {
  const char* what = "rope_axes";
  OUDJAT_REQUIRE(rows >= 0 && Hq >= 0 && Hk >= 0 && Dh >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  OUDJAT_REQUIRE(dtype == 0 || dtype == 1, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d", what, dtype);
  if (rows == 0 || Hq + Hk == 0 || Dh == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)), OUDJAT_ERR_INVALID_ARGUMENT,
                 "%s: null pointer", what);
  OUDJAT_REQUIRE(Dh % 16 == 0 && Dh <= 512, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (a multiple of 16 up to 512)",
                 what, (long long)Dh);
  OUDJAT_REQUIRE(((q_rs | q_hs | k_rs | k_hs | qo_rs | qo_hs | ko_rs | ko_hs) % 8) == 0 && aligned(q, 16) &&
                     aligned(k, 16) && aligned(q_out, 16) && aligned(k_out, 16),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned rows and heads required", what);
  OUDJAT_REQUIRE(entries_apart({{rows, qo_rs}, {Hq, qo_hs}}, Dh) && entries_apart({{rows, ko_rs}, {Hk, ko_hs}}, Dh),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: the rows and heads of an output must not overlap", what);
  AxisRope a;
  const int rc = make_axis_rope(&a, pos, pos_kind, pos_rs, pos_as, axes, inv_freq, sections, Dh, what);
  if (rc != OUDJAT_OK) return rc;
  OUDJAT_REQUIRE(Hq == 0 || Hk == 0 || q_out != k_out, OUDJAT_ERR_INVALID_ARGUMENT,
                 "%s: q_out and k_out are the same buffer", what);
  const int per = rope_rows_per_wg(rows, a.half);
  OUDJAT_REQUIRE(cdiv(rows, per) < (1 << 24) && (Hq + Hk) * Dh * per < INT32_MAX, OUDJAT_ERR_TOO_LARGE, "%s: too large",
                 what);
  auto go = [&](auto e, auto u) {
    rope_axes_kernel<decltype(e), decltype(u)::value>
        <<<(unsigned)cdiv(rows, per), kRopeThreads, (size_t)per * 2 * a.half * 4, as_stream(stream)>>>(
            a, q, q_rs, q_hs, k, k_rs, k_hs, q_out, qo_rs, qo_hs, k_out, ko_rs, ko_hs, rows, (int)Hq, (int)Hk, (int)Dh,
            per);
  };
  auto by_items = [&](auto e) {
    if (per * (Hq + Hk) * Dh / 16 > kRopeThreads) go(e, std::integral_constant<int, 4>{});
    else go(e, std::integral_constant<int, 1>{});
  };
  if (dtype == 0) by_items(ElemBf16{});
  else by_items(ElemFp16{});
  return check_launch(what);
}

extern "C" int oudjat_qk_norm_rope_kv(const uint16_t* qkv, int64_t x_rs, int64_t rows, int64_t Hq, int64_t Hk, int64_t Dh,
                                      int dtype, int layer_norm, const uint16_t* qw, const uint16_t* qb,
                                      const uint16_t* kw, const uint16_t* kb, float eps, const void* pos, int pos_kind,
                                      int64_t pos_rs, int64_t pos_as, int64_t axes, const float* inv_freq,
                                      const int64_t* sections, const int64_t* batch_idx, const int64_t* token_idx,
                                      uint16_t* kv, int64_t kv_bs, int64_t kv_ns, int64_t kv_cs, int64_t B, int64_t N,
                                      uint16_t* q_out, int64_t qo_rs, oudjat_stream_t stream) {
  const char* what = "qk_norm_rope_kv";
  OUDJAT_REQUIRE(rows >= 0 && Hq > 0 && Hk > 0 && Dh > 0 && B >= 0 && N >= 0, OUDJAT_ERR_INVALID_ARGUMENT,
                 "%s: bad size", what);
  OUDJAT_REQUIRE(dtype == 0 || dtype == 1, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d", what, dtype);
  OUDJAT_REQUIRE(eps >= 0.0f, OUDJAT_ERR_INVALID_ARGUMENT, "%s: eps must not be negative or NaN", what);
  OUDJAT_REQUIRE(layer_norm || (!qb && !kb), OUDJAT_ERR_INVALID_ARGUMENT, "%s: a bias without layer_norm", what);
  if (rows == 0) return OUDJAT_OK;
  const bool empty = B == 0 || N == 0;  // a cache without slots: every row is skipped
  OUDJAT_REQUIRE(qkv && batch_idx && token_idx && (kv || empty) && q_out, OUDJAT_ERR_INVALID_ARGUMENT,
                 "%s: null pointer", what);
  OUDJAT_REQUIRE(Dh == 64 || Dh == 128, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (64 or 128)", what, (long long)Dh);
  OUDJAT_REQUIRE(((x_rs | kv_bs | kv_ns | kv_cs | qo_rs) % 8) == 0 && aligned(qkv, 16) && aligned(kv, 16) &&
                     aligned(q_out, 16) && aligned(qw, 16) && aligned(qb, 16) && aligned(kw, 16) && aligned(kb, 16) &&
                     aligned(batch_idx, 8) && aligned(token_idx, 8),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned rows and weights required", what);
  OUDJAT_REQUIRE(entries_apart({{rows, qo_rs}}, Hq * Dh) && entries_apart({{B, kv_bs}, {N, kv_ns}, {2, kv_cs}}, Hk * Dh),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: the rows of q_out and of the cache must not overlap", what);
  AxisRope a;
  const int rc = make_axis_rope(&a, pos, pos_kind, pos_rs, pos_as, axes, inv_freq, sections, Dh, what);
  if (rc != OUDJAT_OK) return rc;
  const int per = rope_rows_per_wg(rows, a.half);
  OUDJAT_REQUIRE(cdiv(rows, per) < (1 << 24) && (Hq + 2 * Hk) * Dh * per < INT32_MAX, OUDJAT_ERR_TOO_LARGE,
                 "%s: too large", what);
  if (empty) return OUDJAT_OK;
  auto go = [&](auto e, auto dh, auto layer) {
    qk_norm_rope_kv_kernel<decltype(e), decltype(dh)::value, decltype(layer)::value>
        <<<(unsigned)cdiv(rows, per), kRopeThreads, (size_t)per * 2 * a.half * 4, as_stream(stream)>>>(
            a, qkv, x_rs, rows, (int)Hq, (int)Hk, qw, qb, kw, kb, eps, batch_idx, token_idx, kv, kv_bs, kv_ns, kv_cs, B,
            N, q_out, qo_rs, per);
  };
  auto by_norm = [&](auto e, auto dh) {
    if (layer_norm) go(e, dh, std::true_type{});
    else go(e, dh, std::false_type{});
  };
  auto by_dim = [&](auto e) {
    if (Dh == 64) by_norm(e, std::integral_constant<int, 64>{});
    else by_norm(e, std::integral_constant<int, 128>{});
  };
  if (dtype == 0) by_dim(ElemBf16{});
  else by_dim(ElemFp16{});
  return check_launch(what);
}
