// Grouped-head attention of packed query rows over NVFP4 K/V caches (format: nvfp4_kv.hip): packed_attention.hip's
// operator, its packing of a group's heads into rows, its items, parts and merge, with other operands.
//
// A cached value is v = e2m1(code) e4m3(scale) h, h the head's tensor scale. x^ = e2m1 e4m3 has at most 6 significant
// bits and lies in 2^-10 .. 2688, so it is exact in fp16, two values in two instructions: a packed convert of the codes
// and a packed product with the block's scale (whose fp16 bits are its e4m3 bits shifted, 2^-8 of its value; the convert
// multiplies by 2^8). Both products run in fp16 for either type of the queries: a query row is scaled by a power of two
// that brings its largest value to 2^14 .. 2^15 (bf16 values keep all their bits down to 2^-28 of it), that power and
// the key head's h go into the row's factor of the scores, the value head's h into the output. Probabilities are kept
// 2^7 larger than their reference says, at most 2^15 with the 2^8 that the reference may lag (kFarScore: whatever the
// scores' size), so that weights down to 2^-21 of the largest are normal numbers of fp16 (rounded by at most 2^-11 of their value).
#include "elem.hpp"
#include "nvfp4_kv.hpp"

namespace oudjat {

struct Nvfp4Attn {
  PackedAttn p;  // (k and v unused)
  KvNvfp4 c;
  float scale_log2;
};

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));

static constexpr float kProbShift = 7.0f;

// The weight of score s is 2^(c s + shift), c the row's factor. With a reference of ordinary size one FMA takes it off,
// shift = 7 - c ref, rounded no more than the score itself would be in fp32. From 2^20 on the reference is taken off the
// scores first, exactly where they lie close, so that c (s - ref) is at most the 8 that it may lag: further out the rounding
// of the shift is whole exponents (16 at 2^28: infinite weights, or none at all). A trained model has no such row. The keys
// kernel looks at the reference in every tile; the rows kernel, where that costs 1 to 2 % at 64 dims, decides by the row's factor
// alone (scaled queries are below 2^15 and x^ is at most 6 * 480: Dh = 128, query values of 100 against keys of 450 at the usual
// scale are still near) and sends such rows through its masked tiles.
template <int DH>
__device__ __forceinline__ bool far_scores(float c) {
  return c > kFarScore / (DH * 32768.0f * 2880.0f);
}
// A reference as the exponent that the other waves' and parts' meet, kept finite (-inf, no key, too: its sum is 0).
__device__ __forceinline__ float ref_exponent(float m, float c) { return fminf(fmaxf(m * c, -3.40282347e38f), 3.40282347e38f); }
// A row's factor of its scores. Not 0 and not infinite, so that a hidden key's -inf stays what it is and a difference of 0 is 0.
__device__ __forceinline__ float score_factor(float c) { return fminf(fmaxf(c, 1.17549435e-38f), 3.40282347e38f); }

// Byte of 16-byte chunk `chunk` of key row `row` in a tile. Dh = 128: the chunks of row r lie at chunk ^ swz(r), swz a
// permutation of 0 .. 15 that puts four consecutive rows into four quarters of a row and the next four into the other
// halves of these, so that 16 rows at one chunk (fragment reads of keys, writes), four rows at four chunks and eight rows at
// two chunks (transposing reads of values for 32 and 16 dims) cover all banks.
template <int DH>
__device__ __forceinline__ int nv_slot(int row, int chunk) {
  if constexpr (DH == 128) {
    const int swz = ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
    return row * 2 * DH + ((chunk ^ swz) << 4);
  } else {
    return tile_slot<DH>(row, chunk);
  }
}

// fp16 pair of 2^-8 e4m3(byte i of s), twice.
__device__ __forceinline__ h2_t scale_pair(uint32_t s, int i) {
  return __builtin_bit_cast(h2_t, ((s >> (8 * i)) & 0x7fu) * 0x00800080u);
}
// Eight codes to x^.
__device__ __forceinline__ h8_t xhat8(uint32_t w, h2_t s) {
  const h2_t a = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 256.0f, 0)) * s;
  const h2_t b = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 256.0f, 1)) * s;
  const h2_t c = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 256.0f, 2)) * s;
  const h2_t d = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 256.0f, 3)) * s;
  return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's share of a query row, `N` chunks of 8 dims, as fp16 times 2^e; the inverse of that factor. `whole` combines a
// lane's value with those of the other lanes of the row (max or sum). A row with a NaN or an infinity is told by `bad`.
template <class E, int N, class Max, class Sum>
__device__ __forceinline__ float load_query(const uint16_t* p, int step, h8_t* q, bool& bad, Max&& row_max, Sum&& row_sum) {
  float f[N][8], top = 0.0f, z = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    E::to8(load16(p + i * step), f[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fabsf(f[i][e]));
      z = fmaf(f[i][e], 0.0f, z);
    }
  }
  top = row_max(top);
  bad = row_sum(z) != 0.0f;
  // Exponent fields: 14 + 127 - (top's - 127), kept where its inverse is a normal number too.
  const int field = clamp_idx(268 - (int)(__float_as_uint(top) >> 23), 1, 253);
  const float up = __uint_as_float((uint32_t)field << 23);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) q[i][e] = (_Float16)(f[i][e] * up);
  return __uint_as_float((uint32_t)(254 - field) << 23);
}

// ------------------------------------------------------------------------------------------------
// Keys kernel, for sequences of few packed rows (single tokens): 16 rows per workgroup, whose waves take 32 keys each in
// turn; the waves' results meet in LDS at the end. A lane loads its piece of a key row (four lanes a row) and its
// scales into registers, a tile ahead. Keys go from there to the first product (both of whose operands permute the
// dims alike: lane group G has dims G Dh / 4 ..), values through LDS in fp16, from where the transposing reads take
// them. Bound by reading the cache where there are enough waves: 512 tokens over 1000 keys each, 32 over 8 heads of 128,
// 121 to 125 us by the card (4.9 TB/s, a copy's rate; over a 16-bit cache 370 to 383).
// About 250 VALU instructions a tile of 32 keys, half of them the turning into fp16, are half of the SIMDs' cycles; a tile's
// chain (products, maximum, exponentials, products) is hidden by four waves a SIMD, for which the registers are stated
// (three: 126 us, two: 147).
// ------------------------------------------------------------------------------------------------
template <class E, int DH, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 ? 4 : 2) void nvfp4_attn_keys_kernel(Nvfp4Attn na) {
  constexpr int R = 16, KEYS = 32, QK_STEPS = DH / 32, DB = DH / 16, KT = WAVES * KEYS;
  constexpr int CW = DH / 32, ROWB = 2 * DH, CPR = DH / 8;  // a lane's words of codes
  const PackedAttn& a = na.p;
  extern __shared__ __align__(16) unsigned char smem[];

  const int item = a.by_hk(blockIdx.x), h = blockIdx.x - item * a.Hk;
  Item w;
  if (!take_item<R, KT>(a, item, h, w)) return;
  const int lane = threadIdx.x & 63, l16 = lane & 15, G = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int total = w.m * a.G, r0 = w.tile * R, row = r0 + l16;
  const int at = min(row, total - 1);  // rows past the last repeat it and are not stored
  const int tok = a.by_g(at), head = at - tok * a.G;
  const int lim = seen_keys(a, w, tok);
  const int kend = seen_keys(a, w, a.by_g(min(r0 + R, total) - 1));
  const int lim_tile = seen_keys(a, w, a.by_g(r0));
  const int all_tiles = (kend + KT - 1) / KT, per = w.parts == 1 ? all_tiles : (all_tiles + w.parts - 1) / w.parts;
  const int kfirst = min(w.part * per, all_tiles) * KT, klast = min(kend, kfirst + per * KT);  // this part's keys
  const int n32 = max(0, (klast - kfirst + KEYS - 1) / KEYS);
  const int cnt = (n32 - wave + WAVES - 1) / WAVES;  // tiles of this wave: wave, wave + WAVES, ...

  const uint8_t* kc = na.c.codes + (int64_t)w.seq * na.c.bs + (int64_t)h * na.c.hs;
  const uint8_t* ksc = na.c.scales + (int64_t)w.seq * na.c.sbs + (int64_t)h * na.c.shs;
  const uint8_t *vc = kc + na.c.cs, *vsc = ksc + na.c.scs;
  unsigned char* park16 = smem + wave * KEYS * ROWB;  // this wave's values in fp16

  h8_t qf[QK_STEPS];  // lane: row l16, dims G DH / 4 + 8 ks ..
  bool bad;
  const float down = load_query<E, QK_STEPS>(
      a.q + (int64_t)(w.q0 + tok) * a.q_rs + (int64_t)(h * a.G + head) * a.q_hs + G * (DH / 4), 8, qf, bad,
      [](float x) { return xor32_max(xor16_max(x)); }, [](float x) { return xor32_sum(xor16_sum(x)); });
  const float c = score_factor(na.scale_log2 * na.c.ts[h] * down);

  struct Tile {
    uint32_t k[2][CW], v[2][CW], ks[2], vs[2];
  };
  auto key_of = [&](int t) { return kfirst + (WAVES * t + wave) * KEYS; };
  auto load = [&](Tile& x, int t) __attribute__((always_inline)) {
    const int key0 = key_of(t), last = min(KEYS, w.n - key0) - 1;
    const uint8_t *kp = kc + (int64_t)key0 * na.c.ns, *vp = vc + (int64_t)key0 * na.c.ns;
    const uint8_t *ksp = ksc + (int64_t)key0 * na.c.sns, *vsp = vsc + (int64_t)key0 * na.c.sns;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t r = (uint32_t)min(l16 + 16 * i, last);  // keys past the last repeat it, their weight is 0
      const uint32_t off = r * (uint32_t)na.c.ns + (uint32_t)(G * 4 * CW);
      const uint32_t soff = r * (uint32_t)na.c.sns + (uint32_t)(G * (CW / 2));
      if constexpr (CW == 4) {
        const uint4 kk = *reinterpret_cast<const uint4*>(kp + off), vv = *reinterpret_cast<const uint4*>(vp + off);
        x.k[i][0] = kk.x; x.k[i][1] = kk.y; x.k[i][2] = kk.z; x.k[i][3] = kk.w;
        x.v[i][0] = vv.x; x.v[i][1] = vv.y; x.v[i][2] = vv.z; x.v[i][3] = vv.w;
        x.ks[i] = *reinterpret_cast<const uint16_t*>(ksp + soff);
        x.vs[i] = *reinterpret_cast<const uint16_t*>(vsp + soff);
      } else {
        const uint2 kk = *reinterpret_cast<const uint2*>(kp + off), vv = *reinterpret_cast<const uint2*>(vp + off);
        x.k[i][0] = kk.x; x.k[i][1] = kk.y;
        x.v[i][0] = vv.x; x.v[i][1] = vv.y;
        x.ks[i] = ksp[soff];
        x.vs[i] = vsp[soff];
      }
    }
  };

  // This lane's bytes in the wave's tile (16 keys further on: 16 rows): where it writes, and where it reads 4 dims of a key.
  const int put = nv_slot<DH>(l16, G * CW);
  const int get = nv_slot<DH>(4 * G + (l16 >> 2), (l16 & 3) >> 1) + (l16 & 1) * 8;
  // Chunk c of the same row: for aligned steps, the swizzle is an exclusive or.
  auto step_of = [](int base, int c) { return base ^ (c << 4); };

  f32x4_t o[DB];
  float m_i = -INFINITY, l_i = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto process = [&](const Tile& x, int t) __attribute__((always_inline)) {
    const int key0 = key_of(t);
    f32x4_t s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < QK_STEPS; ++ks)
        s[i] = AttnFp16::mfma16(xhat8(x.k[i][ks], scale_pair(x.ks[i], ks / 2)), qf[ks], s[i]);
#pragma unroll
      for (int ks = 0; ks < QK_STEPS; ++ks)
        *reinterpret_cast<h8_t*>(park16 + step_of(put, ks) + 16 * i * ROWB) =
            xhat8(x.v[i][ks], scale_pair(x.vs[i], ks / 2));
    }
    if (key0 + KEYS > lim_tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + 16 * i + 4 * G + e >= lim) s[i][e] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
    mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = xor32_max(xor16_max(mx));
    const float m_new = softmax_ref_max(m_i, mx, c);
    const float ref = finite_ref(m_new);
    const float alpha = __builtin_amdgcn_exp2f((m_i - ref) * c);
    float shift = kProbShift - ref * c;
    const bool far = fabsf(ref * c) > kFarScore;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(far) != 0, 0)) {
      const float off = far ? ref : 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] -= off;
      shift = far ? kProbShift : shift;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], c, shift));
    const h8_t pf = round8<AttnFp16>(p);
    l_i = l_i * alpha + xor32_sum(xor16_sum(AttnFp16::sum8(pf, 0.0f)));
    m_i = m_new;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= alpha;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const unsigned char* p = park16 + step_of(get, 2 * db);
      const i16x8_t vt = join8(read_tr(p), read_tr(p + 16 * ROWB));
      o[db] = AttnFp16::mfma16(__builtin_bit_cast(h8_t, vt), pf, o[db]);
    }
  };

  constexpr int AHEAD = 1;  // tiles (two or three more in flight: 2 to 10 % slower, their registers cost more than they hide)
  Tile x[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (i < cnt) load(x[i], i);
#pragma unroll 1
  for (int t0 = 0; t0 < cnt; t0 += AHEAD + 1) {
#pragma unroll
    for (int i = 0; i <= AHEAD; ++i) {
      const int t = t0 + i;
      if (t >= cnt) break;
      if (t + AHEAD < cnt) load(x[(i + AHEAD) % (AHEAD + 1)], t + AHEAD);
      process(x[i], t);
    }
  }
  if (bad && lim > 0) l_i = NAN;  // (its scores may all be -inf: 0 otherwise)

  // The waves' results: references and sums, then rows of DH + 4 floats (conflict-free writes of 16 rows).
  constexpr int OROW = DH + 4, WROWS = 2 * R + R * OROW;
  float* park = reinterpret_cast<float*>(smem);
  __syncthreads();
  {
    float* p = park + wave * WROWS;
    if (G == 0) {
      p[l16] = ref_exponent(m_i, c);
      p[R + l16] = l_i;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4_t*>(p + 2 * R + l16 * OROW + 16 * d + 4 * G) = o[d];
  }
  __syncthreads();
  const int r = threadIdx.x / CPR, ch = threadIdx.x % CPR;  // row, 8 dims
  if (r >= R || r0 + r >= total) return;
  float mp[WAVES], m = -INFINITY, l = 0.0f, z[8] = {};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    mp[i] = park[i * WROWS + r];
    m = fmaxf(m, mp[i]);
  }
  const float mc = finite_ref(m);
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const float f = __builtin_amdgcn_exp2f(mp[i] - mc);
    l = fmaf(park[i * WROWS + R + r], f, l);
    const float* src = park + i * WROWS + 2 * R + r * OROW + 8 * ch;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = fmaf(src[e], f, z[e]);
  }
  const float vts = na.c.ts[a.Hk + h];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] *= vts;
  const int otok = a.by_g(r0 + r), orow = w.q0 + otok, ohead = h * a.G + (r0 + r - otok * a.G);
  if (w.parts > 1) {
    float* ws = a.ws + ((int64_t)item * a.Hk + h) * part_floats(R, DH);
    if (ch == 0) {
      ws[r] = m;
      ws[R + r] = l;
    }
    f32x4_t* wo = reinterpret_cast<f32x4_t*>(ws + 2 * R + (int64_t)r * DH + 8 * ch);
    wo[0] = f32x4_t{z[0], z[1], z[2], z[3]};
    wo[1] = f32x4_t{z[4], z[5], z[6], z[7]};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] *= inv;
  store16(a.out + (int64_t)orow * a.o_rs + (int64_t)ohead * DH + 8 * ch, E::from8(z));
}

// ------------------------------------------------------------------------------------------------
// Rows kernel: R = 32 W packed rows, a wave owns 32, all waves of the workgroup share tiles of 64 keys in fp16 in LDS. S^T =
// K . Q^T and O^T += V^T . P^T on v_mfma_f32_32x32x16 as in packed_attention.hip: a row is one lane pair (l, l ^ 32), whose
// registers hold its scores. A thread turns pieces of 32 dims (16 bytes of codes, two scales) into fp16 once for the
// workgroup; a piece is loaded two tiles ahead and written one tile ahead, between the first product and the softmax of
// the tile before. 16 lanes write the same dims of 16 keys, which covers all banks. Neither the VALU nor the matrix cores are
// busy all the time, since a wave's softmax and products wait for one another and two waves a SIMD cover a part of it: 49 and 42 %
// of the SIMD cycles in one prompt of 8192 tokens, 32 over 8 heads of 128, 541 to 564 us by the card (1017 to 975 TF/s); 50 and
// 22 % in four prompts of up to 4101, 16 heads of 64; one of 4101 73 us, where 528 workgroups of different lengths leave CUs idle
// at the end (every other round of them backwards: 8 % faster to 10 % slower by the lengths). A block's fragments all read
// before its products: the same at 64 dims, 4 % slower at 128.
// ------------------------------------------------------------------------------------------------
template <class E, int DH, int W>
__global__ __launch_bounds__(W * 64, 2) void nvfp4_attn_rows_kernel(Nvfp4Attn na) {
  constexpr int R = 32 * W, QK_STEPS = DH / 16, OB = DH / 32, ROWB = 2 * DH;
  constexpr int TILEB = kKeyTile * ROWB, STAGE = 2 * TILEB;
  constexpr int PIECES = 2 * kKeyTile * (DH / 32) / (64 * W), PPW = 64 / (DH / 32);  // a thread's; keys of a wave's pieces
  static_assert(PIECES == 1 || PIECES == 2, "whole pieces");
  const PackedAttn& a = na.p;
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

  h8_t qf[QK_STEPS];  // lane: row l32, dims 16 ks + 8 g ..
  bool bad;
  const float down = load_query<E, QK_STEPS>(
      a.q + (int64_t)(w.q0 + tok) * a.q_rs + (int64_t)(h * a.G + head) * a.q_hs + 8 * g, 16, qf, bad,
      [](float x) { return xor32_max(x); }, [](float x) { return xor32_sum(x); });
  const float c = score_factor(na.scale_log2 * na.c.ts[h] * down);
  const bool far = far_scores<DH>(c), any_far = __builtin_amdgcn_ballot_w64(far) != 0;
  // Tiles that need neither a mask nor a reference taken off first (a wave's own: every tile has one barrier).
  const int nfull = any_far ? 0 : lim_tile / kKeyTile - tb;

  // This thread's pieces: with one a thread the waves' first half takes keys, the second values.
  const int pw = PIECES == 1 ? wave % (W / 2) : wave, pkey = pw * PPW + (lane & 15) + 16 * (lane / (16 * (DH / 32)));
  const int pc = (lane >> 4) % (DH / 32);
  const uint8_t *kc = na.c.codes + (int64_t)w.seq * na.c.bs + (int64_t)h * na.c.hs + 16 * pc;
  const uint8_t *ksc = na.c.scales + (int64_t)w.seq * na.c.sbs + (int64_t)h * na.c.shs + 2 * pc;
  const bool second = PIECES == 1 && wave >= W / 2;
  if (second) {
    kc += na.c.cs;
    ksc += na.c.scs;
  }
  struct Pieces {
    uint4 codes[PIECES];
    uint32_t scales[PIECES];
  };
  auto load = [&](Pieces& x, int t) __attribute__((always_inline)) {
    const int key0 = (tb + t) * kKeyTile;
    const uint32_t r = (uint32_t)min(pkey, w.n - 1 - key0);  // keys past the last repeat it, their weight is 0
    const uint8_t *kp = kc + (int64_t)key0 * na.c.ns, *ksp = ksc + (int64_t)key0 * na.c.sns;
    const uint32_t off = r * (uint32_t)na.c.ns, soff = r * (uint32_t)na.c.sns;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      x.codes[i] = *reinterpret_cast<const uint4*>(kp + (i ? na.c.cs : 0) + off);
      x.scales[i] = *reinterpret_cast<const uint16_t*>(ksp + (i ? na.c.scs : 0) + soff);
    }
  };
  int slot[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) slot[j] = nv_slot<DH>(pkey, 4 * pc + j) + (second ? TILEB : 0);
  auto expand = [&](const Pieces& x, unsigned char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint32_t word[4] = {x.codes[i].x, x.codes[i].y, x.codes[i].z, x.codes[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<h8_t*>(st + slot[j] + i * TILEB) = xhat8(word[j], scale_pair(x.scales[i], j / 2));
    }
  };

  f32x16_t o[OB];
  float m_i = -INFINITY, l_i = 0.0f;
#pragma unroll
  for (int d = 0; d < OB; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
  int koff[QK_STEPS], voff[OB][2];
#pragma unroll
  for (int ks = 0; ks < QK_STEPS; ++ks) koff[ks] = nv_slot<DH>(l32, ks * 2 + g);
  {
    const int sl = lane & 15, hh = (lane >> 4) & 1, key = 4 * g + (sl >> 2);
#pragma unroll
    for (int db = 0; db < OB; ++db) {
      const int dcol = 32 * db + 16 * hh + 4 * (sl & 3);  // first of the 4 dims this lane addresses
      voff[db][0] = TILEB + nv_slot<DH>(key, dcol >> 3) + ((dcol >> 2) & 1) * 8;
      voff[db][1] = TILEB + nv_slot<DH>(key + 8, dcol >> 3) + ((dcol >> 2) & 1) * 8;
    }
  }
  f32x16_t s[2];  // s[kb][v]: key 32 kb + 8 (v / 4) + 4 g + v % 4, row l32
  auto scores = [&](const unsigned char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      h8_t kf[QK_STEPS];
#pragma unroll
      for (int ks = 0; ks < QK_STEPS; ++ks) kf[ks] = *reinterpret_cast<const h8_t*>(st + koff[ks] + kb * 32 * ROWB);
      const f32x16_t zero = {};
      s[kb] = AttnFp16::mfma32(kf[0], qf[0], zero);
#pragma unroll
      for (int ks = 1; ks < QK_STEPS; ++ks) s[kb] = AttnFp16::mfma32(kf[ks], qf[ks], s[kb]);
    }
  };
  auto finish = [&](const unsigned char* st, int t, auto masked) __attribute__((always_inline)) {
    const int key0 = (tb + t) * kKeyTile;
    if (decltype(masked)::value && key0 + kKeyTile > lim_wave) {
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
    const float m_new = softmax_ref_max(m_i, mx, c);
    const float ref = finite_ref(m_new);
    const float alpha = __builtin_amdgcn_exp2f((m_i - ref) * c);
    float shift = kProbShift - ref * c;
    if (decltype(masked)::value && any_far) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kb][v] -= far ? ref : 0.0f;
      if (far) shift = kProbShift;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[kb][v] = __builtin_amdgcn_exp2f(fmaf(s[kb][v], c, shift));
    h8_t pf[4];
    float rs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float tmp[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) tmp[e] = s[j >> 1][8 * (j & 1) + e];
      pf[j] = round8<AttnFp16>(tmp);
      rs[j] = AttnFp16::sum8(pf[j], 0.0f);
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
    for (int db = 0; db < OB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const i16x8_t vt = join8(read_tr(st + voff[db][0] + j * 16 * ROWB), read_tr(st + voff[db][1] + j * 16 * ROWB));
        o[db] = AttnFp16::mfma32(__builtin_bit_cast(h8_t, vt), pf[j], o[db]);
      }
  };

  // Iteration t: barrier (tile t is in its stage, and every wave is done with tile t - 1's), first product of tile t, tile
  // t + 1 into the other stage, loads of tile t + 2, softmax and second product of tile t. All waves of the workgroup
  // pass the same barriers; waves without rows only load and expand.
  if (ntiles > 0) {
    Pieces x;
    load(x, 0);
    expand(x, smem);
    if (ntiles > 1) load(x, 1);
    auto pipeline = [&](auto work_c) __attribute__((always_inline)) {
      constexpr bool WORK = decltype(work_c)::value;
      auto step = [&](int t, auto masked) __attribute__((always_inline)) {
        unsigned char* st = smem + (t & 1) * STAGE;
        const bool sees = WORK && (!decltype(masked)::value || (tb + t) * kKeyTile < kend_wave);
        block_barrier();
        if (sees) scores(st);
        if (t + 1 < ntiles) {
          expand(x, smem + (~t & 1) * STAGE);
          if (t + 2 < ntiles) load(x, t + 2);
        }
        if (sees) finish(st, t, masked);
      };
      int t = 0;
      for (; t < min(nfull, ntiles); ++t) step(t, std::false_type{});
      for (; t < ntiles; ++t) step(t, std::true_type{});
    };
    if (active) pipeline(std::true_type{});
    else pipeline(std::false_type{});
  }
  if (bad && lim > 0) l_i = NAN;  // (its scores may all be -inf: 0 otherwise)

  // O^T: lane l, register v of block db -> dim 32 db + 8 (v / 4) + 4 g + v % 4 of row l32.
  if (!mine) return;
  const float vts = na.c.ts[a.Hk + h];
  const int orow = w.q0 + tok, ohead = h * a.G + head;
  if (w.parts > 1) {
    float* ws = a.ws + ((int64_t)item * a.Hk + h) * part_floats(R, DH);
    const int r = row - r0;
    if (g == 0) {
      ws[r] = ref_exponent(m_i, c);
      ws[R + r] = l_i;
    }
    float* wo = ws + 2 * R + (int64_t)r * DH + 4 * g;
#pragma unroll
    for (int d = 0; d < OB; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<f32x4_t*>(wo + 32 * d + 8 * r4) =
            f32x4_t{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]} * vts;
    return;
  }
  const float inv = l_i == 0.0f ? 0.0f : vts / l_i;
  uint16_t* op = a.out + (int64_t)orow * a.o_rs + (int64_t)ohead * DH + 4 * g;
#pragma unroll
  for (int d = 0; d < OB; ++d)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const float y[8] = {o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv};
      const uint4 b = E::from8(y);
      *reinterpret_cast<uint2*>(op + 32 * d + 8 * r4) = make_uint2(b.x, b.y);
    }
}

}  // namespace oudjat

using namespace oudjat;

static constexpr int kNvfp4Cus = 256;

// How a call is dealt, as packed_attention.hip's packed_shape. Measured on one card, graphs of calls, us:
// waves of the keys kernel: eight while there are at most two tiles for each CU and nothing is split (32 tokens over up to
//   2000 keys, 32 over 8 heads of 128: 17.7 by eight, 21.3 by four; 64: 20.7, 22.6; 128: 38.9, 31.1).
// target: keys are split while there are fewer than four tiles for each CU. Parts for each CU, keys kernel: four, whose waves
//   are all that hides a tile's chain of steps (32 tokens over up to 16 k keys, 32 over 8 heads of 128: 59 with one, 50 with
//   two, 41 with four; 1 token 14.5, 15.5, 15.7). Tiles of 256 rows, one workgroup on a CU: one (512 rows over 8 k keys, 32 over
//   8 heads: 85, with two 102); of 128 rows: two (8 x 512 rows over up to 8 k keys, 16 heads of 64: 82 with one, 70 with two,
//   129 unsplit; as many keys for all: 101 split, 99 not). 8 x 256 rows over up to 8 k keys, 32 over 8 heads: 106, 243 unsplit.
struct Nvfp4Shape {
  int R, waves, target, min_tiles;
  bool search;
  int64_t items;
};
static Nvfp4Shape nvfp4_shape(int64_t rows, int64_t S, int64_t Hq, int64_t Hk, int64_t Dh, int64_t key_cap) {
  Nvfp4Shape s{};
  const int64_t G = Hq / Hk, seqs = std::max<int64_t>(1, std::min(S, rows));
  const int64_t mean = cdiv(rows * G, seqs);  // packed rows of a sequence
  s.R = mean <= 32 ? 16 : Dh == 128 && mean > 192 ? 256 : 128;
  s.min_tiles = s.R == 16 ? 2 : 6;
  const int64_t tiles = std::max(rows * G / s.R, seqs);  // about as many as there are
  const int64_t parts = s.R == 16 ? 4 : s.R == 128 ? 2 : 1;  // for each CU
  if (tiles * Hk < 4 * kNvfp4Cus && key_cap > 2048) s.target = (int)cdiv(parts * kNvfp4Cus, Hk);
  s.waves = !s.target && tiles * Hk <= 2 * kNvfp4Cus ? 8 : 4;
  const int keys = s.R == 16 ? 32 * s.waves : kKeyTile;  // of a key tile
  s.search = S > 64 && !s.target && (S > kSortedSeqs || key_cap <= 2048);
  const int64_t most = rows * G / s.R + (s.search ? S : seqs), most_parts = cdiv(cdiv(key_cap, keys), s.min_tiles);
  s.items = s.target ? std::min(most + s.target + s.target / 16 + 1, most * most_parts) : most;
  return s;
}

static int64_t nvfp4_part_elems(const Nvfp4Shape& s, int64_t Hk, int64_t Dh) {
  return s.items * Hk * (part_floats(s.R, (int)Dh) + 4);  // the results, then four ints each for the merge
}

extern "C" int64_t oudjat_packed_attention_nvfp4_workspace_elems(int64_t rows, int64_t S, int64_t Hq, int64_t Hk,
                                                                 int64_t Dh, int64_t key_cap) {
  if (rows <= 0 || S <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || (Dh != 64 && Dh != 128) || rows * (Hq / Hk) >= 1 << 30)
    return 0;
  const Nvfp4Shape s = nvfp4_shape(rows, S, Hq, Hk, Dh, key_cap);
  return s.target ? nvfp4_part_elems(s, Hk, Dh) : 0;
}

template <class E, int DH, int WAVES>
static int launch_nvfp4_keys(const Nvfp4Attn& a, hipStream_t st, const char* what) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = WAVES * std::max(32 * 2 * DH, (2 * 16 + 16 * (DH + 4)) * 4);
  const int rc = allow_lds((const void*)nvfp4_attn_keys_kernel<E, DH, WAVES>, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  nvfp4_attn_keys_kernel<E, DH, WAVES><<<(unsigned)a.p.items * a.p.Hk, WAVES * 64, lds, st>>>(a);
  return check_launch(what);
}

template <class E, int DH, int W>
static int launch_nvfp4_rows(const Nvfp4Attn& a, hipStream_t st, const char* what) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = 2 * 2 * kKeyTile * 2 * DH;
  const int rc = allow_lds((const void*)nvfp4_attn_rows_kernel<E, DH, W>, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  nvfp4_attn_rows_kernel<E, DH, W><<<(unsigned)a.p.items * a.p.Hk, W * 64, lds, st>>>(a);
  return check_launch(what);
}

template <class E, class A, int DH>
static int launch_nvfp4(const Nvfp4Attn& a, int R, int waves, hipStream_t st, const char* what) {
  constexpr int kHigh = DH == 128 ? 256 : 128;  // rows of the highest tile
  const int rc = R == 16    ? (waves == 8 ? launch_nvfp4_keys<E, DH, 8>(a, st, what) : launch_nvfp4_keys<E, DH, 4>(a, st, what))
                 : R == 128 ? launch_nvfp4_rows<E, DH, 4>(a, st, what)
                            : launch_nvfp4_rows<E, DH, kHigh / 32>(a, st, what);
  if (rc != OUDJAT_OK || !a.p.target) return rc;
  const dim3 grid((unsigned)a.p.items * a.p.Hk, (unsigned)(R / merge_rows(R, DH)));
  if (R == 16) packed_attn_merge_kernel<A, DH, 16><<<grid, 256, 0, st>>>(a.p);
  else if (R == 128) packed_attn_merge_kernel<A, DH, 128><<<grid, 256, 0, st>>>(a.p);
  else packed_attn_merge_kernel<A, DH, kHigh><<<grid, 256, 0, st>>>(a.p);
  return check_launch("packed_attention_nvfp4 (merge)");
}

extern "C" int oudjat_packed_attention_nvfp4(const uint16_t* q, int64_t q_rs, int64_t q_hs, int64_t rows, int64_t Hq,
                                             int64_t Dh, const uint8_t* codes, int64_t c_bs, int64_t c_ns, int64_t c_cs,
                                             int64_t c_hs, const uint8_t* scales, int64_t s_bs, int64_t s_ns,
                                             int64_t s_cs, int64_t s_hs, const float* tensor_scale, int64_t Hk,
                                             int64_t key_cap, const void* cu_q, int cu_wide, const void* keys,
                                             int keys_wide, int64_t S, float scale, int causal, int dtype,
                                             uint16_t* out, int64_t out_rs, float* workspace, int64_t workspace_elems,
                                             oudjat_stream_t stream) {
  const char* what = "packed_attention_nvfp4";
  OUDJAT_REQUIRE(rows >= 0 && S >= 0 && Hq > 0 && Hk > 0 && Dh > 0 && key_cap >= 0 && workspace_elems >= 0,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad size", what);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(std::isfinite(scale) && scale > 0.0f, OUDJAT_ERR_INVALID_ARGUMENT, "%s: scale must be positive", what);
  OUDJAT_REQUIRE(Dh == 64 || Dh == 128, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (64 or 128)", what, (long long)Dh);
  OUDJAT_REQUIRE(Hq % Hk == 0, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: %lld query heads over %lld key heads", what,
                 (long long)Hq, (long long)Hk);
  if (rows == 0 || S == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE(q && cu_q && keys && out && tensor_scale && (key_cap == 0 || (codes && scales)),
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(q_rs >= 0 && q_hs >= 0 && out_rs >= 0, OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: negative stride", what);
  OUDJAT_REQUIRE(((q_rs | q_hs | out_rs) % 8) == 0 && aligned(q, 16) && aligned(out, 16) &&
                     aligned(cu_q, cu_wide ? 8 : 4) && aligned(keys, keys_wide ? 8 : 4),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned q and out rows and heads required", what);
  const KvNvfp4 c{const_cast<uint8_t*>(codes), c_bs, c_ns, c_cs, c_hs, const_cast<uint8_t*>(scales), s_bs, s_ns, s_cs,
                  s_hs, tensor_scale, S, key_cap, (int)Hk};
  int rc = check_kv_nvfp4(c, Dh, what);
  if (rc != OUDJAT_OK) return rc;
  OUDJAT_REQUIRE(entries_apart({{rows, out_rs}}, Hq * Dh), OUDJAT_ERR_UNSUPPORTED_LAYOUT,
                 "%s: the rows of out must not overlap", what);
  OUDJAT_REQUIRE(rows * (Hq / Hk) < (1 << 30) && Hq <= 65535 && S < (1 << 24) && key_cap < (1 << 30) &&
                     c_ns < (1 << 24) && s_ns < (1 << 24),
                 OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const Nvfp4Shape s = nvfp4_shape(rows, S, Hq, Hk, Dh, key_cap);
  OUDJAT_REQUIRE(s.items * Hk < (1 << 23), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const int64_t parts = s.target ? nvfp4_part_elems(s, Hk, Dh) : 0;
  OUDJAT_REQUIRE(!s.target || (workspace && aligned(workspace, 16) && workspace_elems >= parts),
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld elements is needed", what,
                 (long long)parts);
  // The parts' references are exponents of 2 already: the merge takes them times 1.
  const Nvfp4Attn a{PackedAttn{q, q_rs, q_hs, nullptr, nullptr, 0, 0, 0, 0, 0, 0, cu_q, keys, out, out_rs, (int)rows,
                               (int)S, (int)Hk, (int)(Hq / Hk), Divisor((uint32_t)Hk), Divisor((uint32_t)(Hq / Hk)),
                               (int)key_cap, cu_wide != 0, keys_wide != 0, true, causal != 0, s.search, false, 1.0f,
                               s.target, s.min_tiles, (int)s.items, workspace,
                               s.target ? reinterpret_cast<int4*>(workspace + s.items * Hk * part_floats(s.R, (int)Dh))
                                        : nullptr},
                    c, scale * 1.4426950408889634f};
  hipStream_t st = as_stream(stream);
  if (dtype == OUDJAT_BF16)
    return Dh == 64 ? launch_nvfp4<ElemBf16, AttnBf16, 64>(a, s.R, s.waves, st, what)
                    : launch_nvfp4<ElemBf16, AttnBf16, 128>(a, s.R, s.waves, st, what);
  return Dh == 64 ? launch_nvfp4<ElemFp16, AttnFp16, 64>(a, s.R, s.waves, st, what)
                  : launch_nvfp4<ElemFp16, AttnFp16, 128>(a, s.R, s.waves, st, what);
}
