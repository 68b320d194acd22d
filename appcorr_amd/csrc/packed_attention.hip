// Grouped-head attention of packed query rows over the keys of their own sequences, causal or not.
//
// A sequence of m rows and n keys: its row i sees the keys j < n (causal: j <= n - m + i), as far as the buffers hold
// them,
//   out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - c mu),  c = scale log2 e,
// with an online softmax: mu is a reference that follows the running maximum, and sum and output are rescaled when it
// moves. Scores, statistics and outputs are fp32; the p_j are rounded to the element type for the second product, and
// the sum is of the rounded values, so that numerator and normaliser use the same weights. The matrix cores take 16-bit
// operands; a second product for the remainders would add half of a tile's matrix work for an error against 64 bits of
// 0.0016 instead of 0.0020 to 0.0023 (bf16, of the outputs' size; 0.0016 is the rounding of the output).
//
// The G query heads of a key head are packed into the query rows: packed row r of a sequence is token r / G, head
// r % G of the group, so that one pass over a key head's K and V serves the whole group, a single token fills G rows
// of a tile, and a causal tile spans few tokens.
//
// Work is dealt by the sequences' lengths, which only the device knows: a workgroup is one (item, key head), item =
// (tile of R packed rows, part of its keys), and finds its item from the lengths itself (scan_item, search_item: 1.2 us
// of an idle CU, 2 beside a busy neighbour; a launch that laid the items out would cost every call 3 us and more).
// Tiles are numbered from a sequence's last, the one with the most keys under causality. The grid is an upper bound
// from the numbers of rows and sequences; workgroups without an item leave.
//
// Few items are split by keys: parts of about units / target key tiles write their running reference, sum and
// unnormalised rows to the workspace, and a second launch merges them in part order.
//
// Two kernels. packed_attn_rows: R = 32 W rows, a wave owns 32, all waves of the workgroup share K/V tiles of 64 keys.
// packed_attn_keys, for few rows: R = 16, the waves share the rows and take 32 keys each in turn. Measured:
// prompts of up to 16384 tokens, 32 over 8 heads of 128, 3.32 to 3.52 ms by the card (977 to 1040 TF/s; a 16384^3 product
// of the library 1360); 32 tokens over caches of up to 16385 keys 155 us (5.0 TB/s); 24 crops of up to 1029 tokens, 16
// heads of 64, 43 us on a GPU that is busy, 47 on one that was idle. The steps' figures below were taken one against the
// other on one card.
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

// V^T fragment with its infinities and NaNs taken out (0) and told apart: plus / minus hold 1 where the element is
// +inf / -inf, both where it is NaN.
template <class E>
__device__ __forceinline__ void split_nonfinite(i16x8_t& v, i16x8_t& plus, i16x8_t& minus) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int b = (int)(uint16_t)v[e], mag = b & 0x7fff;
    const bool bad = mag >= E::kExp, nan = mag > E::kExp;
    v[e] = bad ? 0 : v[e];
    plus[e] = bad && (nan || !(b & 0x8000)) ? (short)E::kOne : 0;
    minus[e] = bad && (nan || (b & 0x8000)) ? (short)E::kOne : 0;
  }
}
template <class V>
__device__ __forceinline__ V add_nonfinite(V o, V plus, V minus, int n) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (e < n) {
      if (plus[e] > 0.0f) o[e] += INFINITY;
      if (minus[e] > 0.0f) o[e] -= INFINITY;
    }
  return o;
}

__device__ __forceinline__ i16x8_t join8(i16x4_t lo, i16x4_t hi) {
  return i16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
__device__ __forceinline__ i16x4_t read_tr(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)p);
}

// exp2 arguments are finite or -inf: a reference of -inf (no key seen yet) is replaced by 0.
__device__ __forceinline__ float ref_shift(float m, float scale_log2) { return m == -INFINITY ? 0.0f : m * scale_log2; }

// ------------------------------------------------------------------------------------------------
// Rows kernel. Each wave computes S^T = K . Q^T (two blocks of 32 keys x 32 rows on v_mfma_f32_32x32x16) and
// O^T += V^T . P^T: a row is one lane pair (l, l ^ 32), whose registers hold its scores, so that the softmax is a
// register reduction and one lane exchange, and P^T feeds the second product from registers. K and V tiles go from
// HBM to LDS by buffer loads, four stages deep, each through a descriptor of exactly the keys that its tile has
// left (built per tile from 64-bit addresses, so that a sequence may span more than 4 GiB): keys past the
// sequence's last load as zeros, whatever lies there. The scores of the next tile are issued before the softmax of
// this one. Bound by the softmax's VALU work and the matrix cores in about equal parts (about 140 VALU instructions per
// 32 x 64 scores, half of a tile's cycles), as the rectangular attention's kernels are; two waves per SIMD are stated in the
// launch bounds, without which the compiler keeps accumulators in the second register file and moves them (Dh = 64:
// 96 of 269 VALU instructions, 24 crops 92 -> 69 us). Three stages and three waves per SIMD at Dh = 64 spill (24 crops
// 46 -> 60 us). Beside the tiles a workgroup pays 4 to 5 us: its item, queries, first tiles and the output.
// Hidden keys inside a sequence (causal) have score -inf, weight 0; a non-finite value among them would still give
// 0 * inf = NaN in the second product. Only where a row came out non-finite is the item done again on a slow path
// that takes such values out of the product and adds them to the rows that see them. So are, without a mask too, value
// rows that lie closer than a row (one value for all keys, a cache of one token): the descriptor of a sequence's last
// tile shows visible values again behind the last key.
// ------------------------------------------------------------------------------------------------
template <class E, int DH, int W>
__global__ __launch_bounds__(W * 64, 2) void packed_attn_rows_kernel(PackedAttn a) {
  constexpr int R = 32 * W, QK_STEPS = DH / 16, OB = DH / 32, NST = 4;
  constexpr int ROWB = 2 * DH, CPR = DH / 8, TILEB = kKeyTile * ROWB, RPI = 1024 / ROWB, STAGE = 2 * TILEB;
  constexpr int LPW = kKeyTile / (RPI * W);
  static_assert(RPI * W % 16 == 0 && LPW >= 1, "the swizzle repeats every 16 rows");
  typedef typename E::v8 v8;
  extern __shared__ __align__(16) unsigned char smem[];

  const int item = a.by_hk(blockIdx.x), h = blockIdx.x - item * a.Hk;
  Item w;
  if (!take_item<R, kKeyTile>(a, item, h, w)) return;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int total = w.m * a.G;                       // packed rows of the sequence
  const int r0 = w.tile * R, rw = r0 + wave * 32;    // first row of the tile and of this wave
  const int row = rw + l32;
  const bool active = rw < total, mine = row < total;
  const int at = min(row, total - 1);  // rows past the last repeat it and are not stored
  const int tok = a.by_g(at), head = at - tok * a.G;
  const int lim = seen_keys(a, w, tok);
  // Keys: the tile's last row sees kend, its first lim_tile (all full tiles below need no mask); the same per wave.
  const int kend = seen_keys(a, w, a.by_g(min(r0 + R, total) - 1));
  const int lim_tile = seen_keys(a, w, a.by_g(r0));
  const int kend_wave = active ? seen_keys(a, w, a.by_g(min(rw + 32, total) - 1)) : 0;
  const int lim_wave = active ? seen_keys(a, w, a.by_g(rw)) : w.n;
  const int all_tiles = (kend + kKeyTile - 1) / kKeyTile;
  const int per = w.parts == 1 ? all_tiles : (all_tiles + w.parts - 1) / w.parts;
  const int tb = w.part * per;                       // first key tile of this part; tiles are numbered from it below
  const int ntiles = max(0, min(per, all_tiles - tb));
  const int nfull = lim_tile / kKeyTile - tb;

  const uint16_t* kbase = a.k + (a.batched ? (int64_t)w.seq * a.k_bs : (int64_t)w.k0 * a.k_rs) + (int64_t)h * a.k_hs;
  const uint16_t* vbase = a.v + (a.batched ? (int64_t)w.seq * a.v_bs : (int64_t)w.k0 * a.v_rs) + (int64_t)h * a.v_hs;

  v8 qf[QK_STEPS];  // lane: row l32, dims 16 ks + 8 g ..
  {
    const uint16_t* qp = a.q + (int64_t)(w.q0 + tok) * a.q_rs + (int64_t)(h * a.G + head) * a.q_hs + 8 * g;
#pragma unroll
    for (int ks = 0; ks < QK_STEPS; ++ks) qf[ks] = as8<E>(*reinterpret_cast<const uint4*>(qp + 16 * ks));
  }

  const int lrow = RPI * wave + lane / CPR;  // tile row that this lane loads, and rows RPI W further on
  const uint32_t chunk = (uint32_t)(((lane % CPR) ^ tile_swz<DH>(lrow)) << 4);
  const uint32_t koff0 = (uint32_t)lrow * (uint32_t)a.k_rs * 2u + chunk;
  const uint32_t voff0 = (uint32_t)lrow * (uint32_t)a.v_rs * 2u + chunk;
  // Tiles are issued in order: the next one's addresses and the keys left from it on (uniform).
  const uint16_t *knext, *vnext;
  int left;
  const int64_t kstep = kKeyTile * a.k_rs, vstep = kKeyTile * a.v_rs;
  const uint32_t krow = (uint32_t)a.k_rs * 2u, vrow = (uint32_t)a.v_rs * 2u;
  auto rewind = [&]() {
    knext = kbase + (int64_t)tb * kstep;
    vnext = vbase + (int64_t)tb * vstep;
    left = w.n - tb * kKeyTile;
  };
  rewind();
  auto issue = [&](int stage) __attribute__((always_inline)) {
    const uint32_t last = (uint32_t)(min(left, kKeyTile) - 1);
    const i32x4_t rk = make_buffer_rsrc(knext, last * krow + ROWB), rv = make_buffer_rsrc(vnext, last * vrow + ROWB);
    unsigned char* base = smem + stage * STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      buffer_load_lds16(rk, base + i * W * 1024, koff0 + (uint32_t)(i * RPI * W) * krow);
      buffer_load_lds16(rv, base + i * W * 1024 + TILEB, voff0 + (uint32_t)(i * RPI * W) * vrow);
    }
    knext += kstep;
    vnext += vstep;
    left -= kKeyTile;
  };
  auto wait_tiles = [&](int n) __attribute__((always_inline)) {  // tiles that may stay in flight
    if (n <= 0) wait_vmcnt<0>();
    else if (n == 1) wait_vmcnt<2 * LPW>();
    else wait_vmcnt<4 * LPW>();
  };

  f32x16_t o[OB];
  float m_i = -INFINITY, l_i = 0.0f;
#pragma unroll
  for (int d = 0; d < OB; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;

  int koff[QK_STEPS], voff[OB][2];
#pragma unroll
  for (int ks = 0; ks < QK_STEPS; ++ks) koff[ks] = tile_slot<DH>(l32, ks * 2 + g);
  {
    const int sl = lane & 15, hh = (lane >> 4) & 1, key = 4 * g + (sl >> 2);
#pragma unroll
    for (int db = 0; db < OB; ++db) {
      const int dcol = 32 * db + 16 * hh + 4 * (sl & 3);  // first of the 4 dims this lane addresses
      voff[db][0] = TILEB + tile_slot<DH>(key, dcol >> 3) + ((dcol >> 2) & 1) * 8;
      voff[db][1] = TILEB + tile_slot<DH>(key + 8, dcol >> 3) + ((dcol >> 2) & 1) * 8;
    }
  }

  struct Scores {
    f32x16_t s[2];  // s[kb][v]: key 32 kb + 8 (v / 4) + 4 g + v % 4, row l32
  };
  auto scores = [&](Scores& sc, const unsigned char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      v8 kf[QK_STEPS];
#pragma unroll
      for (int ks = 0; ks < QK_STEPS; ++ks)
        kf[ks] = as8<E>(*reinterpret_cast<const uint4*>(st + koff[ks] + kb * 32 * ROWB));
      const f32x16_t zero = {};
      sc.s[kb] = E::mfma32(kf[0], qf[0], zero);
#pragma unroll
      for (int ks = 1; ks < QK_STEPS; ++ks) sc.s[kb] = E::mfma32(kf[ks], qf[ks], sc.s[kb]);
    }
  };
  // MODE 0: no key of the tile is hidden from any row; 1: some may be; 2: and values may be non-finite.
  auto finish = [&](Scores& sc, const unsigned char* st, int t, auto mode) __attribute__((always_inline)) {
    constexpr int MODE = decltype(mode)::value;
    f32x16_t (&s)[2] = sc.s;
    const int key0 = (tb + t) * kKeyTile;
    if (MODE && key0 + kKeyTile > lim_wave) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (key0 + kb * 32 + 8 * (v >> 2) + 4 * g + (v & 3) >= lim) s[kb][v] = -INFINITY;
    }
    float mq[4];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      mq[q4] = s[q4 >> 1][8 * (q4 & 1)];
#pragma unroll
      for (int v = 1; v < 8; ++v) mq[q4] = fmaxf(mq[q4], s[q4 >> 1][8 * (q4 & 1) + v]);
    }
    const float mx = xor32_max(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])));
    const float m_new = softmax_ref_max(m_i, mx, a.scale_log2);
    const float mc = ref_shift(m_new, a.scale_log2);
    const float alpha = __builtin_amdgcn_exp2f(fmaf(m_i, a.scale_log2, -mc));
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[kb][v] = __builtin_amdgcn_exp2f(fmaf(s[kb][v], a.scale_log2, -mc));
    v8 pf[4];
    float rs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float tmp[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) tmp[e] = s[j >> 1][8 * (j & 1) + e];
      pf[j] = round8<E>(tmp);
      rs[j] = E::sum8(pf[j], 0.0f);
    }
    l_i = l_i * alpha + xor32_sum((rs[0] + rs[1]) + (rs[2] + rs[3]));
    m_i = m_new;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int d = 0; d < OB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
    }
#pragma unroll
    for (int db = 0; db < OB; ++db) {
      [[maybe_unused]] f32x16_t plus = {}, minus = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        i16x8_t vt = join8(read_tr(st + voff[db][0] + j * 16 * ROWB), read_tr(st + voff[db][1] + j * 16 * ROWB));
        if constexpr (MODE == 2) {
          i16x8_t vp, vm;
          split_nonfinite<E>(vt, vp, vm);
          plus = E::mfma32(__builtin_bit_cast(v8, vp), pf[j], plus);
          minus = E::mfma32(__builtin_bit_cast(v8, vm), pf[j], minus);
        }
        o[db] = E::mfma32(__builtin_bit_cast(v8, vt), pf[j], o[db]);
      }
      if constexpr (MODE == 2) o[db] = add_nonfinite(o[db], plus, minus, 16);
    }
  };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  // Iteration t: wait for tile t + 1, barrier (every wave is done with tile t - 1's stage), refill that stage with
  // tile t + 3, issue the scores of tile t + 1, then softmax and second product of tile t. All waves of the
  // workgroup pass the same barriers; waves without rows only load.
  auto pipeline = [&](auto work_c) __attribute__((always_inline)) {
    constexpr bool WORK = decltype(work_c)::value;
    Scores sa, sb;
    auto sees = [&](int t) { return WORK && (tb + t) * kKeyTile < kend_wave; };
    if (sees(0)) scores(sa, smem);
    auto step = [&](auto stage_c, int t, Scores& cur, Scores& nxt, auto mode) __attribute__((always_inline)) {
      constexpr int SG = decltype(stage_c)::value, MODE = decltype(mode)::value;
      if (!MODE || t + 1 < ntiles) {
        if (MODE) wait_tiles(min(NST - 3, ntiles - 2 - t));
        else wait_vmcnt<2 * LPW * (NST - 3)>();
        block_barrier();
        if (!MODE || t + NST - 1 < ntiles) issue((SG + NST - 1) % NST);
        if (MODE ? sees(t + 1) : WORK) scores(nxt, smem + ((SG + 1) % NST) * STAGE);
      }
      if (MODE ? sees(t) : WORK) finish(cur, smem + SG * STAGE, t, mode);
    };
    int t = 0;
    for (; t + 2 * NST - 2 < ntiles && t + NST <= nfull; t += NST) {  // nothing hidden in tiles t .. t + 3
      step(I0{}, t, sa, sb, I0{});
      step(I1{}, t + 1, sb, sa, I0{});
      step(I2{}, t + 2, sa, sb, I0{});
      step(I3{}, t + 3, sb, sa, I0{});
    }
    for (; t < ntiles; t += NST) {
      step(I0{}, t, sa, sb, I1{});
      if (t + 1 < ntiles) step(I1{}, t + 1, sb, sa, I1{});
      if (t + 2 < ntiles) step(I2{}, t + 2, sa, sb, I1{});
      if (t + 3 < ntiles) step(I3{}, t + 3, sb, sa, I1{});
    }
  };
  if (ntiles > 0) {
#pragma unroll
    for (int st = 0; st < NST - 1; ++st)
      if (st < ntiles) issue(st);
    wait_tiles(min(NST - 2, ntiles - 1));
    block_barrier();
    if (active) pipeline(std::true_type{});
    else pipeline(std::false_type{});
    if ((a.causal || a.values_overlap) && (tb + ntiles) * kKeyTile > lim_tile) {  // keys were hidden
      float z = 0.0f;
#pragma unroll
      for (int d = 0; d < OB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) z = fmaf(o[d][v], 0.0f, z);
      if (__syncthreads_or(mine && z != 0.0f)) {
        rewind();
        m_i = -INFINITY;
        l_i = 0.0f;
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
#pragma unroll 1
        for (int t = 0; t < ntiles; ++t) {
          __syncthreads();
          issue(0);
          wait_vmcnt<0>();
          __syncthreads();
          if ((tb + t) * kKeyTile < kend_wave) {
            Scores sc;
            scores(sc, smem);
            finish(sc, smem, t, I2{});
          }
        }
      }
    }
  }

  // O^T: lane l, register v of block db -> dim 32 db + 8 (v / 4) + 4 g + v % 4 of row l32.
  if (!mine) return;
  const int orow = w.q0 + tok, ohead = h * a.G + head;
  if (w.parts > 1) {
    float* ws = a.ws + ((int64_t)item * a.Hk + h) * part_floats(R, DH);
    const int r = row - r0;
    if (g == 0) {
      ws[r] = m_i;
      ws[R + r] = l_i;
    }
    float* wo = ws + 2 * R + (int64_t)r * DH + 4 * g;
#pragma unroll
    for (int d = 0; d < OB; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<f32x4_t*>(wo + 32 * d + 8 * r4) =
            f32x4_t{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
    return;
  }
  const float inv = l_i == 0.0f ? 0.0f : 1.0f / l_i;
  uint16_t* op = a.out + (int64_t)orow * a.o_rs + (int64_t)ohead * DH + 4 * g;
#pragma unroll
  for (int d = 0; d < OB; ++d)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x4_t x = {o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv};
      *reinterpret_cast<typename E::v4*>(op + 32 * d + 8 * r4) = __builtin_convertvector(x, typename E::v4);
    }
}

// ------------------------------------------------------------------------------------------------
// Keys kernel, for sequences of few packed rows (single tokens): 16 rows per workgroup, whose waves take 32 keys each
// in turn through rings of their own in LDS (two tiles of K and two of V, each refilled as soon as it is read), so that
// no barrier holds a wave and the loads of a CU (up to 96 KB) are never drained; the waves' results meet in LDS at the
// end. Bound by reading K and V once: 512 tokens over 1000 keys each, 32 over 8 heads of 128, 370 us, 5.7 TB/s.
// S^T per 16-key block on v_mfma_f32_16x16x32 (lane l, G = l / 16: keys 4 G + v of row l % 16), O^T per 16 dims
// (keys 4 G + {0..3} and 16 + 4 G + {0..3} per lane, V^T by the transposing LDS read).
// ------------------------------------------------------------------------------------------------
template <class E, int DH, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void packed_attn_keys_kernel(PackedAttn a) {
  constexpr int R = 16, KEYS = 32, NS = 2, QK_STEPS = DH / 32, DB = DH / 16;
  constexpr int ROWB = 2 * DH, CPR = DH / 8, TILEB = KEYS * ROWB, RPI = 1024 / ROWB, L = KEYS / RPI;
  typedef typename E::v8 v8;
  extern __shared__ __align__(16) unsigned char smem[];

  const int item = a.by_hk(blockIdx.x), h = blockIdx.x - item * a.Hk;
  Item w;
  if (!take_item<R, WAVES * KEYS>(a, item, h, w)) return;
  const int lane = threadIdx.x & 63, l16 = lane & 15, G = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int total = w.m * a.G, r0 = w.tile * R, row = r0 + l16;
  const bool mine = row < total;
  const int at = min(row, total - 1);  // rows past the last repeat it and are not stored
  const int tok = a.by_g(at), head = at - tok * a.G;
  const int lim = seen_keys(a, w, tok);
  const int kend = seen_keys(a, w, a.by_g(min(r0 + R, total) - 1));
  const int lim_tile = seen_keys(a, w, a.by_g(r0));
  constexpr int KT = WAVES * KEYS;
  const int all_tiles = (kend + KT - 1) / KT, per = w.parts == 1 ? all_tiles : (all_tiles + w.parts - 1) / w.parts;
  const int kfirst = min(w.part * per, all_tiles) * KT, klast = min(kend, kfirst + per * KT);  // this part's keys
  const int n32 = max(0, (klast - kfirst + KEYS - 1) / KEYS);
  const int cnt = (n32 - wave + WAVES - 1) / WAVES;  // tiles of this wave: wave, wave + 4, ...

  const uint16_t* kbase = a.k + (a.batched ? (int64_t)w.seq * a.k_bs : (int64_t)w.k0 * a.k_rs) + (int64_t)h * a.k_hs;
  const uint16_t* vbase = a.v + (a.batched ? (int64_t)w.seq * a.v_bs : (int64_t)w.k0 * a.v_rs) + (int64_t)h * a.v_hs;
  unsigned char* kring = smem + wave * (2 * NS * TILEB);
  unsigned char* vring = kring + NS * TILEB;

  v8 qf[QK_STEPS];  // lane: row l16, dims 32 ks + 8 G ..
  {
    const uint16_t* qp = a.q + (int64_t)(w.q0 + tok) * a.q_rs + (int64_t)(h * a.G + head) * a.q_hs + 8 * G;
#pragma unroll
    for (int ks = 0; ks < QK_STEPS; ++ks) qf[ks] = as8<E>(*reinterpret_cast<const uint4*>(qp + 32 * ks));
  }
  auto key_of = [&](int t) { return kfirst + (WAVES * t + wave) * KEYS; };
  auto issue = [&](unsigned char* ring, const uint16_t* base, int64_t rs, int t) __attribute__((always_inline)) {
    const int key0 = key_of(t), last = min(KEYS, w.n - key0) - 1;
    const i32x4_t rsrc = make_buffer_rsrc(base + (int64_t)key0 * rs, (uint32_t)last * (uint32_t)rs * 2u + ROWB);
    unsigned char* dst = ring + (t % NS) * TILEB;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int r = RPI * i + lane / CPR;
      buffer_load_lds16(rsrc, dst + i * 1024,
                        (uint32_t)r * (uint32_t)rs * 2u + (uint32_t)(((lane % CPR) ^ tile_swz<DH>(r)) << 4));
    }
  };
  // At most n of this wave's K or V tiles may stay in flight.
  auto wait_loads = [&](int n) __attribute__((always_inline)) {
    static_assert(NS == 2 && 3 * L < 64, "vmcnt range");
    if (n >= 3) wait_vmcnt<3 * L>();
    else if (n == 2) wait_vmcnt<2 * L>();
    else if (n == 1) wait_vmcnt<L>();
    else wait_vmcnt<0>();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto reads_done = [&]() __attribute__((always_inline)) {  // this wave's LDS reads, before their stage is refilled
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
    __builtin_amdgcn_sched_barrier(0);
  };

  int koff[QK_STEPS], voff[DB][2];
#pragma unroll
  for (int ks = 0; ks < QK_STEPS; ++ks) koff[ks] = tile_slot<DH>(l16, 4 * ks + G);
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int dcol = 16 * db + 4 * (l16 & 3), key = 4 * G + (l16 >> 2);
    voff[db][0] = tile_slot<DH>(key, dcol >> 3) + ((dcol >> 2) & 1) * 8;
    voff[db][1] = tile_slot<DH>(key + 16, dcol >> 3) + ((dcol >> 2) & 1) * 8;
  }

  f32x4_t o[DB];
  float m_i, l_i;
  auto reset = [&]() {
    m_i = -INFINITY;
    l_i = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  };
  reset();
  f32x4_t s[2];
  auto scores = [&](const unsigned char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < QK_STEPS; ++ks)
        s[kb] = E::mfma16(as8<E>(*reinterpret_cast<const uint4*>(st + koff[ks] + kb * 16 * ROWB)), qf[ks], s[kb]);
    }
  };
  v8 pf;
  auto softmax = [&](int key0) __attribute__((always_inline)) {
    if (key0 + KEYS > lim_tile) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (key0 + 16 * kb + 4 * G + v >= lim) s[kb][v] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
    mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = xor32_max(xor16_max(mx));
    const float m_new = softmax_ref_max(m_i, mx, a.scale_log2);
    const float mc = ref_shift(m_new, a.scale_log2);
    const float alpha = __builtin_amdgcn_exp2f(fmaf(m_i, a.scale_log2, -mc));
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], a.scale_log2, -mc));
    pf = round8<E>(p);
    l_i = l_i * alpha + xor32_sum(xor16_sum(E::sum8(pf, 0.0f)));
    m_i = m_new;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= alpha;
    }
  };
  auto values = [&](const unsigned char* st, auto safe) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      i16x8_t vt = join8(read_tr(st + voff[db][0]), read_tr(st + voff[db][1]));
      if constexpr (decltype(safe)::value) {
        i16x8_t vp, vm;
        split_nonfinite<E>(vt, vp, vm);
        const f32x4_t zero = {};
        const f32x4_t plus = E::mfma16(__builtin_bit_cast(v8, vp), pf, zero);
        const f32x4_t minus = E::mfma16(__builtin_bit_cast(v8, vm), pf, zero);
        o[db] = E::mfma16(__builtin_bit_cast(v8, vt), pf, o[db]);
        o[db] = add_nonfinite(o[db], plus, minus, 4);
      } else {
        o[db] = E::mfma16(__builtin_bit_cast(v8, vt), pf, o[db]);
      }
    }
  };

#pragma unroll
  for (int t = 0; t < NS; ++t)
    if (t < cnt) {
      issue(kring, kbase, a.k_rs, t);
      issue(vring, vbase, a.v_rs, t);
    }
#pragma unroll 1
  for (int t = 0; t < cnt; ++t) {
    const int ahead = 2 * min(NS - 1, cnt - 1 - t);  // loads of the tiles after this one
    wait_loads(ahead + 1);
    scores(kring + (t % NS) * TILEB);
    if (t + NS < cnt) {
      reads_done();
      issue(kring, kbase, a.k_rs, t + NS);
    }
    softmax(key_of(t));
    wait_loads(ahead + (t + NS < cnt ? 1 : 0));
    values(vring + (t % NS) * TILEB, std::false_type{});
    if (t + NS < cnt) {
      reads_done();
      issue(vring, vbase, a.v_rs, t + NS);
    }
  }
  // Keys were hidden: see the rows kernel. The last tile of 32 loads keys past kend, which hide even where
  // all rows of the tile see the same keys (16 query heads of one key head: one token).
  if ((a.causal || a.values_overlap) && kfirst + n32 * KEYS > lim_tile) {
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int v = 0; v < 4; ++v) z = fmaf(o[d][v], 0.0f, z);
    if (__builtin_amdgcn_ballot_w64(mine && z != 0.0f)) {
      reset();
#pragma unroll 1
      for (int t = 0; t < cnt; ++t) {
        reads_done();
        issue(kring, kbase, a.k_rs, t);
        issue(vring, vbase, a.v_rs, t);
        wait_loads(0);
        scores(kring + (t % NS) * TILEB);
        softmax(key_of(t));
        values(vring + (t % NS) * TILEB, std::true_type{});
      }
    }
  }

  // The waves' results: references and sums, then rows of DH + 4 floats (conflict-free writes of 16 rows).
  constexpr int OROW = DH + 4, WROWS = 2 * R + R * OROW;
  float* park = reinterpret_cast<float*>(smem);
  __syncthreads();
  {
    float* p = park + wave * WROWS;
    if (G == 0) {
      p[l16] = m_i;
      p[R + l16] = l_i;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4_t*>(p + 2 * R + l16 * OROW + 16 * d + 4 * G) = o[d];
  }
  __syncthreads();
  const int r = threadIdx.x / CPR, c = threadIdx.x % CPR;  // row, 8 dims
  if (r >= R || r0 + r >= total) return;
  float mp[WAVES], m = -INFINITY, l = 0.0f, x[8] = {};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    mp[i] = park[i * WROWS + r];
    m = fmaxf(m, mp[i]);
  }
  const float mc = ref_shift(m, a.scale_log2);
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const float f = __builtin_amdgcn_exp2f(fmaf(mp[i], a.scale_log2, -mc));
    l = fmaf(park[i * WROWS + R + r], f, l);
    const float* src = park + i * WROWS + 2 * R + r * OROW + 8 * c;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(src[e], f, x[e]);
  }
  const int otok = a.by_g(r0 + r), orow = w.q0 + otok, ohead = h * a.G + (r0 + r - otok * a.G);
  if (w.parts > 1) {
    float* ws = a.ws + ((int64_t)item * a.Hk + h) * part_floats(R, DH);
    if (c == 0) {
      ws[r] = m;
      ws[R + r] = l;
    }
    f32x4_t* wo = reinterpret_cast<f32x4_t*>(ws + 2 * R + (int64_t)r * DH + 8 * c);
    wo[0] = f32x4_t{x[0], x[1], x[2], x[3]};
    wo[1] = f32x4_t{x[4], x[5], x[6], x[7]};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= inv;
  const v8 y = round8<E>(x);
  *reinterpret_cast<v8*>(a.out + (int64_t)orow * a.o_rs + (int64_t)ohead * DH + 8 * c) = y;
}

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
      const float tc = ref_shift(top, a.scale_log2);
      const float keep = __builtin_amdgcn_exp2f(fmaf(m, a.scale_log2, -tc));
      m = top;
      l *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lp[u] != 0.0f) {
          const float f = __builtin_amdgcn_exp2f(fmaf(mp[u], a.scale_log2, -tc));
          l = fmaf(lp[u], f, l);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fmaf(y[u][e >> 2][e & 3], f, x[e]);
        }
    }
    if constexpr (PL > 1) {
#pragma unroll
      for (int s = CPR; s < 64; s <<= 1) {
        const float m2 = __shfl_xor(m, s, 64), top = fmaxf(m, m2), tc = ref_shift(top, a.scale_log2);
        const float f = __builtin_amdgcn_exp2f(fmaf(m, a.scale_log2, -tc));
        const float f2 = __builtin_amdgcn_exp2f(fmaf(m2, a.scale_log2, -tc));
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

}  // namespace oudjat

using namespace oudjat;

static constexpr int kPackedCus = 256;

// How a call is dealt, from what the host knows: rows per tile (16: the keys kernel, with its waves), the most items of
// a key head, and how many parts at the most its items are cut into beside their own number (0: never, no workspace).
struct PackedShape {
  int R, waves, target, min_tiles;
  bool search;
  int64_t items;
};

// Measured on one card, graphs of ten calls, us:
// R: up to 32 packed rows a sequence on the mean the keys kernel (4 x 12 rows of 4 heads each over 8 k keys: 17 by it, 32
//   by 128-row tiles with the limit at 16; 32 crops of 201 tokens: 8.7 by rows, 15.6 by keys with the limit at 64). Dh =
//   128: tiles of 256 rows, whose eight waves fill a CU (its LDS holds one workgroup), above 192 rows (4 x 32 heads,
//   414 of 4101: 142, by 128 rows 209; 64 tokens of 4 heads each over 8 k keys, 256 rows: 36, by 128 rows 33). Dh = 64: 128
//   rows, two workgroups on a CU (24 crops: 46, by 256 rows 52; causal 4101 of 16 heads: 61, 82).
// waves of the keys kernel at Dh = 64: eight, one workgroup on a CU, while there are no more tiles than CUs (4 tokens
//   over 1 k keys: 9.2 -> 7.9), else two workgroups of four (64 tokens, 16 heads: 18.6, by eight 26.7).
// target: with as many tiles as CUs (rows) or four times that (keys) nothing is split (64 tokens over 8 k keys, 8
//   key heads: 118 split, 139 not; 16 crops of up to 1029 tokens: 26 unsplit, 47 with twice the target and splits), nor
//   below 2049 keys (8 x 201 tokens of 6 heads: 8.7 unsplit, 10.6 with the merge launch). One part per CU: 1 token over 16 k
//   keys, 8 key heads: 19.2, two per CU 24.7.
// search (above): 256 tokens over 200 keys 17 by search, 26 by scan; 128 over up to 4 k keys 139 by search, 126 by scan.
// min_tiles: 6 x 100 rows over 3 k keys: 15.5 from 6, 20.8 from 12; 2 x 16 rows over 2 k keys: 9.8 from 2, 11.3 from 4.
// All go by the row buffer and the number of sequences, the host's upper bounds: single tokens in a buffer much longer
// than their number run on the rows kernel unsplit (32 tokens over up to 16 k keys 135 us, in 2048 rows 266).
static PackedShape packed_shape(int64_t rows, int64_t S, int64_t Hq, int64_t Hk, int64_t Dh, int64_t key_cap) {
  PackedShape s{};
  const int64_t G = Hq / Hk, seqs = std::max<int64_t>(1, std::min(S, rows));
  const int64_t mean = cdiv(rows * G, seqs);  // packed rows of a sequence
  s.R = mean <= 32 ? 16 : Dh == 128 && mean > 192 ? 256 : 128;
  s.min_tiles = s.R == 16 ? 2 : 6;
  const int64_t tiles = std::max(rows * G / s.R, seqs);  // about as many as there are
  s.waves = Dh == 64 && tiles * Hk <= kPackedCus ? 8 : 4;
  const int keys = s.R == 16 ? 32 * s.waves : kKeyTile;  // of a key tile
  const int64_t fill = s.R == 16 ? 4 * kPackedCus : kPackedCus;
  if (tiles * Hk < fill && key_cap > 2048) s.target = (int)cdiv(kPackedCus, Hk);
  // The most items: the ceil of every sequence's tiles is at most one more than its rows have; and the parts, with
  // room for the rounding of the units' fp32 sum, but no tile has more than the cache's length allows.
  s.search = S > 64 && !s.target && (S > kSortedSeqs || key_cap <= 2048);
  const int64_t most = rows * G / s.R + (s.search ? S : seqs), most_parts = cdiv(cdiv(key_cap, keys), s.min_tiles);
  s.items = s.target ? std::min(most + s.target + s.target / 16 + 1, most * most_parts) : most;
  return s;
}

static int64_t packed_part_elems(const PackedShape& s, int64_t Hk, int64_t Dh) {
  return s.items * Hk * (part_floats(s.R, (int)Dh) + 4);  // the results, then four ints each for the merge
}

extern "C" int64_t oudjat_packed_attention_workspace_elems(int64_t rows, int64_t S, int64_t Hq, int64_t Hk, int64_t Dh,
                                                           int64_t key_cap) {
  if (rows <= 0 || S <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || (Dh != 64 && Dh != 128) || rows * (Hq / Hk) >= 1 << 30)
    return 0;
  const PackedShape s = packed_shape(rows, S, Hq, Hk, Dh, key_cap);
  return s.target ? packed_part_elems(s, Hk, Dh) : 0;
}

// Allows a kernel `lds` bytes of dynamic LDS on the current device, once.
static int allow_lds(const void* fn, int lds, std::atomic<uint64_t>& done, const char* what) {
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

template <class E, int DH, int W>
static int launch_rows(const PackedAttn& a, hipStream_t st, const char* what) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = 4 * 2 * kKeyTile * 2 * DH;
  const int rc = allow_lds((const void*)packed_attn_rows_kernel<E, DH, W>, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  packed_attn_rows_kernel<E, DH, W><<<(unsigned)a.items * a.Hk, W * 64, lds, st>>>(a);
  return check_launch(what);
}

template <class E, int DH, int WAVES>
static int launch_keys(const PackedAttn& a, hipStream_t st, const char* what) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = WAVES * 2 * 2 * 32 * 2 * DH;  // a wave's rings: two tiles each of K and V
  const int rc = allow_lds((const void*)packed_attn_keys_kernel<E, DH, WAVES>, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  packed_attn_keys_kernel<E, DH, WAVES><<<(unsigned)a.items * a.Hk, WAVES * 64, lds, st>>>(a);
  return check_launch(what);
}

template <class E, int DH>
static int launch_packed(const PackedAttn& a, int R, int waves, hipStream_t st, const char* what) {
  constexpr int kHigh = DH == 128 ? 256 : 128;  // rows of the highest tile
  int rc;
  if (R == 16) {
    if constexpr (DH == 64) rc = waves == 8 ? launch_keys<E, DH, 8>(a, st, what) : launch_keys<E, DH, 4>(a, st, what);
    else rc = launch_keys<E, DH, 4>(a, st, what);
  }
  else rc = R == 128 ? launch_rows<E, DH, 4>(a, st, what) : launch_rows<E, DH, kHigh / 32>(a, st, what);
  if (rc != OUDJAT_OK || !a.target) return rc;
  const dim3 grid((unsigned)a.items * a.Hk, (unsigned)(R / merge_rows(R, DH)));
  if (R == 16) packed_attn_merge_kernel<E, DH, 16><<<grid, 256, 0, st>>>(a);
  else if (R == 128) packed_attn_merge_kernel<E, DH, 128><<<grid, 256, 0, st>>>(a);
  else packed_attn_merge_kernel<E, DH, kHigh><<<grid, 256, 0, st>>>(a);
  return check_launch("packed_attention (merge)");
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
  OUDJAT_REQUIRE(((q_rs | q_hs | k_bs | k_rs | k_hs | v_bs | v_rs | v_hs) % 8) == 0 && out_rs % 8 == 0 && aligned(q, 16) &&
                     aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(cu_q, cu_wide ? 8 : 4) &&
                     aligned(keys, keys_wide ? 8 : 4),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned q, k, v and out rows and heads required", what);
  OUDJAT_REQUIRE(entries_apart({{rows, out_rs}}, Hq * Dh), OUDJAT_ERR_UNSUPPORTED_LAYOUT,
                 "%s: the rows of out must not overlap", what);
  OUDJAT_REQUIRE(rows * (Hq / Hk) < (1 << 30) && Hq <= 65535 && S < (1 << 24) && key_cap < (1 << 30) &&
                     k_rs < (1 << 24) && v_rs < (1 << 24),
                 OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const PackedShape s = packed_shape(rows, S, Hq, Hk, Dh, key_cap);
  OUDJAT_REQUIRE(s.items * Hk < (1 << 23), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const int64_t parts = s.target ? packed_part_elems(s, Hk, Dh) : 0;
  OUDJAT_REQUIRE(!s.target || (workspace && aligned(workspace, 16) && workspace_elems >= parts),
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld elements is needed", what,
                 (long long)parts);
  const PackedAttn a{q, q_rs, q_hs, k, v, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, cu_q, keys, out, out_rs, (int)rows, (int)S,
                     (int)Hk, (int)(Hq / Hk), Divisor((uint32_t)Hk), Divisor((uint32_t)(Hq / Hk)), (int)key_cap,
                     cu_wide != 0, keys_wide != 0, batched != 0, causal != 0, s.search, v_rs < Dh, scale * 1.4426950408889634f,
                     s.target, s.min_tiles, (int)s.items, workspace,
                     s.target ? reinterpret_cast<int4*>(workspace + s.items * Hk * part_floats(s.R, (int)Dh)) : nullptr};
  hipStream_t st = as_stream(stream);
  if (dtype == OUDJAT_BF16)
    return Dh == 64 ? launch_packed<AttnBf16, 64>(a, s.R, s.waves, st, what)
                    : launch_packed<AttnBf16, 128>(a, s.R, s.waves, st, what);
  return Dh == 64 ? launch_packed<AttnFp16, 64>(a, s.R, s.waves, st, what)
                  : launch_packed<AttnFp16, 128>(a, s.R, s.waves, st, what);
}
