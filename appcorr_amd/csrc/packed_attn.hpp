// What the attentions of packed query rows share: how a workgroup finds its item (a tile of rows, a part of its keys)
// from the sequences' lengths, the matrix cores' element types, and the merge of the parts of split keys.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "attn.hpp"
#include "common.hpp"

namespace oudjat {

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));

// Division of 0 .. 2^31 - 1 by a number that the launch fixes: x / d = x * ceil(2^(31 + b) / d) >> (31 + b), 2^b >= d.
struct Divisor {
  uint32_t d, mul, shift;
  explicit Divisor(uint32_t n) : d(n), shift(0) {
    while ((1u << shift) < n) ++shift;
    mul = (uint32_t)(((1ull << (31 + shift)) + n - 1) / n);
  }
  __device__ __forceinline__ int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * mul) >> (31 + shift)); }
};

struct PackedAttn {
  const uint16_t* q;
  int64_t q_rs, q_hs;
  const uint16_t *k, *v;
  int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
  const void *cu_q, *keys;
  uint16_t* out;
  int64_t o_rs;
  int rows, S, Hk, G;
  Divisor by_hk, by_g;
  int key_cap;
  bool cu_wide, keys_wide, batched, causal, search;
  bool values_overlap;  // value rows closer than one row: past a tile's last key its descriptor shows values again
  float scale_log2;
  // Key parts: 0 = never split; else the number of parts that a key head's items are cut into at the most, beside
  // their own number, and the fewest key tiles of a part.
  int target, min_tiles;
  int items;      // items a key head has at the most (the grid)
  float* ws;      // the items' partial results
  int4* heads;    // per (item, key head): parts to merge from this item on (0: none), first row, packed row, rows
};

// Element types on the matrix cores.
struct AttnBf16 {
  typedef bf16x8_t v8;
  static constexpr int kOne = 0x3f80, kExp = 0x7f80;
  static __device__ __forceinline__ f32x16_t mfma32(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mfma16(v8 a, v8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum8(v8 p, float acc) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 ones = {(__bf16)1.0f, (__bf16)1.0f};
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 0, 1), ones, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 2, 3), ones, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 4, 5), ones, acc, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 6, 7), ones, acc, false);
  }
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
};
struct AttnFp16 {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr int kOne = 0x3c00, kExp = 0x7c00;
  static __device__ __forceinline__ f32x16_t mfma32(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mfma16(v8 a, v8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum8(v8 p, float acc) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 ones = {(_Float16)1.0f, (_Float16)1.0f};
    acc = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 0, 1), ones, acc, false);
    acc = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 2, 3), ones, acc, false);
    acc = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 4, 5), ones, acc, false);
    return __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 6, 7), ones, acc, false);
  }
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
};

template <class E>
__device__ __forceinline__ typename E::v8 as8(const uint4& v) {
  return __builtin_bit_cast(typename E::v8, v);
}
template <class E>
__device__ __forceinline__ typename E::v8 round8(const float* f) {
  const f32x8_t v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
  return __builtin_convertvector(v, typename E::v8);
}

// Entry i of an int32 or int64 tensor, cut to 32 bits. Without branches, so that the loads of several entries overlap
// (a branch on the width put a wait behind every one).
__device__ __forceinline__ int load_idx(const void* p, int i, bool wide) {
  const int32_t* w = static_cast<const int32_t*>(p) + ((int64_t)i << (wide ? 1 : 0));
  const int lo = w[0], hi = w[wide ? 1 : 0];
  return wide && hi != lo >> 31 ? (hi < 0 ? INT32_MIN : INT32_MAX) : lo;
}
__device__ __forceinline__ int clamp_idx(int v, int lo, int hi) { return max(lo, min(hi, v)); }

// A sequence's rows and keys, and the item that a workgroup takes of it. Uniform over the wave.
struct Item {
  int seq, q0, m, n, k0;  // first row, rows, keys, first key row (packed keys)
  int before;             // causal: row i sees the first before + i + 1 of the keys
  int tile, part, parts;
};

// Sequence s: rows and keys, cut to the buffers. Rows and keys that are cut off still count for what the others see: the
// last row of the uncut sequence sees the last of its uncut keys.
__device__ __forceinline__ void load_seq(const PackedAttn& a, int s, Item& t) {
  const int c0 = load_idx(a.cu_q, s, a.cu_wide), c1 = load_idx(a.cu_q, s + 1, a.cu_wide);
  const int k0 = load_idx(a.keys, s, a.keys_wide), k1 = load_idx(a.keys, s + (a.batched ? 0 : 1), a.keys_wide);
  t.q0 = clamp_idx(c0, 0, a.rows);
  t.m = clamp_idx(c1, t.q0, a.rows) - t.q0;
  t.k0 = a.batched ? 0 : clamp_idx(k0, 0, a.key_cap);
  t.n = clamp_idx(k1, t.k0, a.key_cap) - t.k0;
  // (m, n < 2^30: what passes them either way sees all or nothing)
  const int64_t before = (int64_t)k1 - t.k0 - ((int64_t)c1 - t.q0);
  t.before = (int)max(-(int64_t)(1 << 30), min((int64_t)(1 << 30), before));
}

// Wave-wide sums and maxima by data-parallel moves (no LDS round trips): value of every lane combined with those of
// all lanes before it; lane 63 has the whole.
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T x, F&& f) {
  auto from = [&](auto ctrl, auto rows) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                             decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  x = f(x, from(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}));  // row_shr:1
  x = f(x, from(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}));  // row_shr:2
  x = f(x, from(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}));  // row_shr:4
  x = f(x, from(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}));  // row_shr:8
  x = f(x, from(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}));  // row_bcast:15 to rows 1 and 3
  x = f(x, from(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}));  // row_bcast:31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }
__device__ __forceinline__ float last_lane(float x) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

// Item number `item` of a key head, tiles of R packed rows and KT keys; false if there is none. Two numberings:
//
// Scan (up to 64 sequences, up to kSortedSeqs with long keys, any number if keys are split): the sequences' items one
// after another, 64 sequences at a time. Parts of a sequence's tiles: its key tiles / C, rounded, with C =
// max(min_tiles, units / target) and units the key tiles of all tiles, so that a key head has at most its own tiles +
// target items. Up to kSortedSeqs sequences the items of the longer ones (more than half of the longest's keys, then
// more than a quarter) come first, so that the last workgroups are short.
//
// Search (more sequences, no split): sequence s starts at number floor(cu_q[s] G / R) + s, which leaves room for all
// its tiles, so that the sequence of a number is found by a 64-way search in cu_q, two loads up to 4096 sequences (one
// token each of 4096 sequences, 16 over 4 heads of 64, 200 keys: 956 us by the scan, 222 by the search; of 256 26, 17).
static constexpr int kSortedSeqs = 256;

template <int R, int KT>
__device__ __forceinline__ bool search_item(const PackedAttn& a, int item, Item& w) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.S;
  while (true) {  // the last s of lo .. lo + n - 1 that starts at or before the item
    const int step = (n + 63) / 64, s = lo + lane * step;
    const bool before = s < lo + n && clamp_idx(load_idx(a.cu_q, s, a.cu_wide), 0, a.rows) * a.G / R + s <= item;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
    if (c == 0) return false;
    lo += (c - 1) * step;
    if (step == 1) break;
    n = min(step, a.S - lo);
  }
  load_seq(a, lo, w);
  const int tiles = (w.m * a.G + R - 1) / R, from_first = item - (w.q0 * a.G / R + lo);
  w.seq = lo;
  w.part = 0;
  w.parts = 1;
  w.tile = tiles - 1 - from_first;
  return from_first >= 0 && w.tile >= 0;
}

template <int R, int KT>
__device__ __forceinline__ bool scan_item(const PackedAttn& a, int item, Item& w) {
  const int lane = threadIdx.x & 63;
  Item t;
  int chunk = 1, top = 0;
  auto tiles = [&]() { return (t.m * a.G + R - 1) / R; };
  auto key_tiles = [&]() { return (t.n + KT - 1) / KT; };
  auto load = [&](int s0) {
    t.q0 = t.m = t.n = t.k0 = t.before = 0;
    if (s0 + lane < a.S) load_seq(a, s0 + lane, t);
  };
  load(0);
  const bool sorted = a.S <= kSortedSeqs;
  float units = (float)tiles() * (float)key_tiles();
  top = key_tiles();
  for (int s0 = 64; s0 < a.S; s0 += 64) {
    load(s0);
    units += (float)tiles() * (float)key_tiles();
    top = max(top, key_tiles());
  }
  if (a.target) {
    units = last_lane(wave_scan(units, [](float x, float y) { return x + y; }));
    chunk = max(a.min_tiles, (int)fminf(ceilf(units / (float)a.target), (float)(1 << 24)));
  }
  if (sorted) top = last_lane(wave_scan(top, [](int x, int y) { return max(x, y); }));
  int base = 0;
  for (int cls = 0; cls < (sorted ? 3 : 1); ++cls) {
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      if (a.S > 64) load(s0);
      const int nt = tiles(), kt = key_tiles(), parts = a.target ? max(1, (2 * kt + chunk) / (2 * chunk)) : 1;
      const int mine = !sorted || (2 * kt > top ? 0 : 4 * kt > top ? 1 : 2) == cls ? nt * parts : 0;
      const int incl = wave_scan(mine, [](int x, int y) { return x + y; });
      const int total = last_lane(incl);
      if (item < base + total) {
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + incl > item));
        const int within = item - base - __builtin_amdgcn_readlane(incl - mine, l);
        w.seq = s0 + l;
        w.q0 = __builtin_amdgcn_readlane(t.q0, l);
        w.m = __builtin_amdgcn_readlane(t.m, l);
        w.n = __builtin_amdgcn_readlane(t.n, l);
        w.k0 = __builtin_amdgcn_readlane(t.k0, l);
        w.before = __builtin_amdgcn_readlane(t.before, l);
        w.parts = __builtin_amdgcn_readlane(parts, l);
        const int from_last = w.parts == 1 ? within : within / w.parts;
        w.part = within - from_last * w.parts;
        const int last = __builtin_amdgcn_readlane(nt, l) - 1;
        w.tile = last - from_last;
        return within >= 0 && w.tile >= 0;  // (offsets that fall may let the counts wrap)
      }
      base += total;
    }
  }
  return false;
}

// The workgroup's item, found by its first wave (the others wait: the search is instructions that a neighbour on the
// CU could issue); false past the last. And what the merge has to do from this item on, which every workgroup of the
// grid says, those without an item too.
template <int R, int KT>
__device__ __forceinline__ bool take_item(const PackedAttn& a, int item, int h, Item& w) {
  __shared__ int shared[10];
  if (threadIdx.x < 64) {
    w = Item{};
    bool found = a.search ? search_item<R, KT>(a, item, w) : scan_item<R, KT>(a, item, w);
    // Offsets that fall may make more items than the grid has. A tile whose parts pass the last one is left out whole,
    // since the merge would read results that nothing wrote, past the workspace.
    found = found && w.parts - w.part <= a.items - item;
    if (threadIdx.x == 0) {
      if (a.target) {
        int4 x = make_int4(0, 0, 0, 0);
        if (found && w.part == 0 && w.parts > 1)
          x = make_int4(w.parts, w.q0, w.tile * R, min(R, w.m * a.G - w.tile * R));
        a.heads[(int64_t)item * a.Hk + h] = x;
      }
      shared[0] = w.seq;
      shared[1] = w.q0;
      shared[2] = w.m;
      shared[3] = w.n;
      shared[4] = w.k0;
      shared[5] = w.tile;
      shared[6] = w.part;
      shared[7] = w.parts;
      shared[8] = w.before;
      shared[9] = found;
    }
  }
  __syncthreads();
  auto get = [&](int i) { return __builtin_amdgcn_readfirstlane(shared[i]); };
  w = Item{get(0), get(1), get(2), get(3), get(4), get(8), get(5), get(6), get(7)};
  return get(9) != 0;
}

// Keys that token i of the sequence sees.
__device__ __forceinline__ int seen_keys(const PackedAttn& a, const Item& w, int i) {
  return a.causal ? min(w.n, max(0, w.before + i + 1)) : w.n;
}

// Floats of one part: reference and sum of R rows, then R rows of DH.
__host__ __device__ constexpr int64_t part_floats(int R, int DH) { return (int64_t)R * (DH + 2); }

__device__ __forceinline__ i16x8_t join8(i16x4_t lo, i16x4_t hi) {
  return i16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
__device__ __forceinline__ i16x4_t read_tr(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)p);
}

// exp2 arguments are finite or -inf: a reference of -inf (no key seen yet) is replaced by 0. References are compared by their
// difference, before the factor: 2^(c (m - m)) is 1, where m c with its product rounded would be off by up to half an ulp of
// it, once in every tile.
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }

// A score further out than this (log2) is compared with its reference by difference too: the rounding of the reference's
// product is whole exponents there (16 at 2^28), which gives infinite weights, or none at all.
static constexpr float kFarScore = 1048576.0f;

// Merge of the key parts of the items whose tile was split (workgroups of the others leave at once). With
// m = max_p m_p and f_p = 2^(c (m_p - m)): out = sum_p f_p o_p / sum_p f_p l_p; a part without a visible key has l_p = 0
// and is left out. DH / 8 lanes hold a row's dims; the other lanes of a wave take further parts of it (PL at a time,
// tiles of few rows and many parts) or further rows (PL = 1). A part's order in the sums is fixed.
//
// Rows of a workgroup: what its threads hold at once, or the tile of the keys kernel (3 chunks of up to 512 rows over 8 k
// keys, 256-row tiles: 40.3 -> 37.6 us against 32 rows a workgroup).
__host__ __device__ constexpr int merge_rows(int R, int DH) { return R == 16 ? 16 : 256 / (DH / 8); }
template <class E, int DH, int R>
__global__ __launch_bounds__(256) void packed_attn_merge_kernel(PackedAttn a) {
  constexpr int CPR = DH / 8, LANES = 64 / CPR, PL = R == 16 ? LANES : 1, U = 4;
  const int4 todo = a.heads[blockIdx.x];
  const int parts = todo.x;
  if (parts <= 1) return;
  const int item = a.by_hk(blockIdx.x), h = blockIdx.x - item * a.Hk;
  const int lane = threadIdx.x & 63, c = lane % CPR, pl = PL > 1 ? lane / CPR : 0;
  const int64_t stride = a.Hk * part_floats(R, DH);
  const float* base = a.ws + ((int64_t)item * a.Hk + h) * part_floats(R, DH);
  constexpr int STEP = 4 * (LANES / PL);  // rows of a workgroup at a time
  const int first = blockIdx.y * merge_rows(R, DH), end = min(todo.w, first + merge_rows(R, DH));
  if (first >= end) return;
  for (int r0 = first; r0 < end; r0 += STEP) {
    const int rr = r0 + (threadIdx.x / 64) * (LANES / PL) + (PL > 1 ? 0 : lane / CPR);
    const int r = min(rr, end - 1);  // lanes past the end repeat the last row, for the exchanges below
    float m = -INFINITY, l = 0.0f, x[8] = {};
    for (int p0 = pl; p0 < parts; p0 += PL * U) {
      float mp[U], lp[U];
      f32x4_t y[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* b = base + min(p0 + u * PL, parts - 1) * stride;
        mp[u] = b[r];
        lp[u] = p0 + u * PL < parts ? b[R + r] : 0.0f;
        const f32x4_t* src = reinterpret_cast<const f32x4_t*>(b + 2 * R + (int64_t)r * DH + 8 * c);
        y[u][0] = src[0];
        y[u][1] = src[1];
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lp[u] != 0.0f) top = fmaxf(top, mp[u]);
      const float ref = finite_ref(top);
      const float keep = __builtin_amdgcn_exp2f((m - ref) * a.scale_log2);
      m = top;
      l *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lp[u] != 0.0f) {
          const float f = __builtin_amdgcn_exp2f((mp[u] - ref) * a.scale_log2);
          l = fmaf(lp[u], f, l);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fmaf(y[u][e >> 2][e & 3], f, x[e]);
        }
    }
    if constexpr (PL > 1) {
#pragma unroll
      for (int s = CPR; s < 64; s <<= 1) {
        const float m2 = __shfl_xor(m, s, 64), top = fmaxf(m, m2), ref = finite_ref(top);
        const float f = __builtin_amdgcn_exp2f((m - ref) * a.scale_log2);
        const float f2 = __builtin_amdgcn_exp2f((m2 - ref) * a.scale_log2);
        m = top;
        l = l * f + __shfl_xor(l, s, 64) * f2;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * f + __shfl_xor(x[e], s, 64) * f2;
      }
    }
    if (rr >= end || pl) continue;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= inv;
    const int tok = a.by_g(todo.z + r), qh = todo.z + r - tok * a.G;
    *reinterpret_cast<typename E::v8*>(a.out + (int64_t)(todo.y + tok) * a.o_rs + (int64_t)(h * a.G + qh) * DH + 8 * c) =
        round8<E>(x);
  }
}

// Allows a kernel `lds` bytes of dynamic LDS on the current device, once.
inline int allow_lds(const void* fn, int lds, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error(OUDJAT_ERR_HIP, "%s: hipGetDevice: %s", what, hipGetErrorString(e));
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return OUDJAT_OK;
  e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return set_error(OUDJAT_ERR_HIP, "%s: hipFuncSetAttribute: %s", what, hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
  return OUDJAT_OK;
}

}  // namespace oudjat
