// INT8 products with a scale for each token and each output channel: the quantiser of rows and the product.
//
//   quantise:  s = max |x| / 127 (fp32),  c = rint(x / s) (nearest even; 0 where s = 0), c in -127 .. 127;
//   product:   y[m, n] = (sum_k a[m, k] w[n, k]) (s_a[m] s_w[n]) + bias[n], the sum exact in int32 (K < 2^17),
// then the epilogue in fp32 and one rounding to the output's type.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "elem.hpp"
#include "packed_attn.hpp"

namespace oudjat {

typedef int i32x4v_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------
// Quantiser. A row is held in registers by 64 LANES / 64 waves, CH chunks of 8 values a lane, between its maximum and its
// codes, so that it is read once; longer rows are read again. The maximum is taken on the bits without their sign, where
// infinities and NaNs are above all others: such a row gets the scale NaN and the codes 0, so that its products are NaN.
// Quotients are the IEEE ones: with y = RN(1 / s), q0 = RN(x y), r = x - q0 s (exact by an FMA), RN(q0 + r y) is the
// correctly rounded quotient (Markstein); where s is so small that y overflows or r underflows, x and s are scaled by 2^100 first.
// Adding 1.5 2^23 leaves the nearest whole number (ties to even) in the low byte.
// Bound by HBM: 16404 rows of 8192 in 60 to 73 us (5.5 TB/s and more, VALU 74 % busy), 1656 of 4096 in 7.2; few rows by a launch
// and a round of loads (2.2 to 3.4).
// ------------------------------------------------------------------------------------------------
struct QuantRow {
  float s, t, y, up;  // scale; the scale and its inverse as they are used, the factor between
};
__device__ __forceinline__ QuantRow quant_row(float top) {
  QuantRow r;
  r.s = top / 127.0f;
  r.up = r.s < 1e-24f ? 1.2676506002282294e30f : 1.0f;  // 2^100
  r.t = r.s * r.up;
  r.y = r.t > 0.0f ? 1.0f / r.t : 0.0f;
  return r;
}
__device__ __forceinline__ uint32_t quant_byte(float x, const QuantRow& r) {
  x *= r.up;
  const float q0 = x * r.y;
  const float rem = __builtin_fmaf(-q0, r.t, x);
  const float q = fminf(fmaxf(__builtin_fmaf(rem, r.y, q0), -127.0f), 127.0f);
  return __float_as_uint(q + 12582912.0f) & 0xffu;
}
template <class E>
__device__ __forceinline__ uint2 quant8(const uint4& v, const QuantRow& r) {
  float f[8];
  E::to8(v, f);
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = quant_byte(f[e], r);
  return make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
}
__device__ __forceinline__ uint32_t top_bits(const uint4& v, uint32_t top) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t w = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
    top = max(top, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
  }
  return top;
}
struct QuantBf16 : ElemBf16 {
  static constexpr uint32_t kExp = 0x7f80u;
  static __device__ __forceinline__ float value(uint32_t b) { return bf16_to_f32(b); }
};
struct QuantFp16 : ElemFp16 {
  static constexpr uint32_t kExp = 0x7c00u;
  static __device__ __forceinline__ float value(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
};

static constexpr int kWaveRow = 1024;  // the longest row of one wave

template <class E, int LANES, int CH, bool LONG>
__global__ __launch_bounds__(256) void quantize_int8_kernel(const uint16_t* __restrict__ x, int64_t rows, int K,
                                                            int64_t x_rs, int8_t* __restrict__ codes, int64_t c_rs,
                                                            float* __restrict__ scale) {
  constexpr int RPW = 256 / LANES;  // rows of a workgroup
  __shared__ uint32_t tops[4];
  const int l = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / LANES;
  const bool there = row < rows;  // uniform over a row's lanes
  const uint16_t* p = x + (there ? row : 0) * x_rs;
  const int chunks = K / 8;
  uint4 v[CH];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (l + i * LANES < chunks) v[i] = load16(p + 8 * (l + i * LANES));
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) top = top_bits(v[i], top);
  if constexpr (LONG)
    for (int i = l + CH * LANES; i < chunks; i += LANES) top = top_bits(load16(p + 8 * (int64_t)i), top);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  if (!there) return;
  QuantRow r = quant_row(E::value(top));
  const bool bad = top >= E::kExp;
  if (l == 0) scale[row] = bad ? NAN : r.s;
  int8_t* c = codes + row * c_rs;
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (l + i * LANES < chunks)
      *reinterpret_cast<uint2*>(c + 8 * (l + i * LANES)) = bad ? make_uint2(0, 0) : quant8<E>(v[i], r);
  if constexpr (LONG)
    for (int i = l + CH * LANES; i < chunks; i += LANES)
      *reinterpret_cast<uint2*>(c + 8 * (int64_t)i) = bad ? make_uint2(0, 0) : quant8<E>(load16(p + 8 * (int64_t)i), r);
}

// ------------------------------------------------------------------------------------------------
// Product
// ------------------------------------------------------------------------------------------------
struct Int8Gemm {
  const int8_t* a;
  int64_t lda;
  const float* sa;
  const int8_t* w;
  int64_t ldw;
  const float* sw;
  const uint16_t *bias, *gamma, *resid;
  int64_t ldr;
  uint16_t* c;
  int64_t ldc;
  int M, N, K, tiles_m, tiles_n;
};

// y / (1 + e^-y) on the hardware's exponential and reciprocal, an ulp each: within 2^-20 of its value for |y| < 8 (in units of
// 2^-24: 1.22 |y| by the exponent's product and constant, 2 each by the two functions, 1 each by the sum and the last product),
// and of y elsewhere (library exponential and division: 16404 x 8192 x 4096 618 us, this 551).
__device__ __forceinline__ float silu(float y) {
  return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.44269504f));
}

// Four outputs of one row, columns n .. n + 3, with the roundings of the tile kernel, where y gamma goes through LDS before the
// residual is added: no contraction of the two, so that a row's bits do not depend on the kernel.
template <class E, int EPI>
__device__ __forceinline__ void int8_store4(const Int8Gemm& g, int m, int n, const i32x4v_t& acc) {
#pragma clang fp contract(off)
  typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));
  auto four = [&](const uint16_t* p, float* f) {
    const u16x4_t v = *reinterpret_cast<const u16x4_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = E::value(v[e]);
  };
  const float sa = g.sa[m];
  const float4 sw4 = *reinterpret_cast<const float4*>(g.sw + n);
  const float sw[4] = {sw4.x, sw4.y, sw4.z, sw4.w};
  float y[8] = {}, bias[4] = {}, t[4];
  if (g.bias) four(g.bias + n, bias);
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf((float)acc[e], sa * sw[e], bias[e]);
  if constexpr (EPI == OUDJAT_EPI_BIAS_LS || EPI == OUDJAT_EPI_BIAS_LS_RESID) {
    four(g.gamma + n, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= t[e];
  }
  if constexpr (EPI == OUDJAT_EPI_BIAS_LS_RESID || EPI == OUDJAT_EPI_BIAS_SILU_MUL) {
    four(g.resid + (int64_t)m * g.ldr + n, t);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = EPI == OUDJAT_EPI_BIAS_LS_RESID ? y[e] + t[e] : silu(y[e]) * t[e];
  }
  const uint4 o = E::from8(y);
  *reinterpret_cast<uint2*>(g.c + (int64_t)m * g.ldc + n) = make_uint2(o.x, o.y);
}

// Direct kernel, for few rows: 16 x 16 outputs a workgroup, whose eight waves take 128 bytes of K each in turn, straight
// from memory to registers (a weight is used by one workgroup, or by few), four such chunks in flight, and add their
// sums up in LDS. Bound by the latency of a launch and two rounds of loads, then by reading the weight: 1 x 4096 x 4096
// 5.9 us (2.8 TB/s; one chunk more or fewer in flight, 16 waves, 16 x 32 outputs: 5.8 to 7.3).
static constexpr int kDirectWaves = 8;
template <class E, int EPI>
__global__ __launch_bounds__(kDirectWaves * 64) void int8_direct_kernel(Int8Gemm g) {
  constexpr int WAVES = kDirectWaves, U = 4;  // chunks in flight
  __shared__ i32x4v_t park[WAVES * 64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, G = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tm = blockIdx.x % g.tiles_m, tn = blockIdx.x / g.tiles_m;
  const int m0 = tm * 16, n0 = tn * 16;
  const int8_t *A = g.a + (int64_t)m0 * g.lda, *W = g.w + (int64_t)n0 * g.ldw;
  // (rows past the last repeat it and are not stored)
  const uint32_t oa = (uint32_t)min(l16, g.M - 1 - m0) * (uint32_t)g.lda + 16u * G;
  const uint32_t ow = (uint32_t)min(l16, g.N - 1 - n0) * (uint32_t)g.ldw + 16u * G;
  struct Unit {
    i32x4v_t a[2], w[2];
  };
  const int chunks = (g.K + 127) / 128;
  auto both = [&](int c) { return c * 128 + 64 < g.K; };  // K = 64 mod 128: the last chunk is half a one
  auto load = [&](Unit& u, int c) __attribute__((always_inline)) {
    const int8_t *a = A + (int64_t)c * 128, *w = W + (int64_t)c * 128;
    const uint32_t second = both(c) ? 64u : 0u;
    u.w[0] = *reinterpret_cast<const i32x4v_t*>(w + ow);
    u.w[1] = *reinterpret_cast<const i32x4v_t*>(w + (ow + second));
    u.a[0] = *reinterpret_cast<const i32x4v_t*>(a + oa);
    u.a[1] = *reinterpret_cast<const i32x4v_t*>(a + (oa + second));
  };
  i32x4v_t acc = {0, 0, 0, 0};
  auto products = [&](const Unit& u, int c) __attribute__((always_inline)) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.w[0], u.a[0], acc, 0, 0, 0);
    if (both(c)) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.w[1], u.a[1], acc, 0, 0, 0);
  };
  Unit u[U];
  int c = wave;
#pragma unroll
  for (int i = 0; i < U - 1; ++i)
    if (c + i * WAVES < chunks) load(u[i], c + i * WAVES);
  while (c < chunks) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (c >= chunks) break;
      if (c + (U - 1) * WAVES < chunks) load(u[(i + U - 1) % U], c + (U - 1) * WAVES);
      products(u[i], c);
      c += WAVES;
    }
  }
  park[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) acc += park[w * 64 + lane];
  if (m0 + l16 < g.M && n0 + 4 * G < g.N) int8_store4<E, EPI>(g, m0 + l16, n0 + 4 * G, acc);
}

// Eight outputs of a tile. Large tiles store past the caches, which then keep the operands that other tiles read. Us of the
// product alone, through the caches -> past them, one card, both in turn: 16404 x 8192 x 4096 470 -> 460 (with a residual 533 ->
// 514), 16404 x 4096 x 8192 437 -> 428 (474 -> 468), 16404 x 4096 x 4096 241 -> 237 (269 -> 249), 4176 x 4096 x 1024 29.6 -> 26.9,
// 1656 x 12288 x 4096 86.6 -> 85.2; in place of the residual, whose lines the caches hold: the same. What reads the output next
// gives some of it back: with a quantiser behind it, 570 -> 550 (with a residual 619 -> 634), 479 -> 481 (514 -> 510), 269 -> 272
// (306 -> 312), 39.8 -> 38.7, 99 -> 100. Small tiles make outputs that are still in the caches when they are read (40 x 4096 x 4096
// with the quantiser: 12.9, past them 13.2).
template <bool PAST>
__device__ __forceinline__ void store_row(uint16_t* p, const uint4& v) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t*>(p));
  else store16(p, v);
}

// Tile kernel: BM x BN outputs, WGM x WGN waves of WM x WN each, K in tiles of 128 bytes through NST stages of LDS that
// buffer loads fill (descriptors of the tile's rows that exist: others load as zeros). LDS row r keeps its 16-byte chunk
// c in slot c ^ (r / 2) % 8, so that 16 rows at one chunk cover all banks. v_mfma_i32_16x16x64_i8 with the weight as its
// first operand: lane l holds row l % 16, columns 4 (l / 16) .. + 3 of a 16 x 16 block.
// A tile of K is two steps. While the matrix cores work on the fragments of one step, those of the next are read; a
// barrier in the middle of the tile says that all waves have read it, so that the loads of the K tile NST further on may
// go to its stage, and that the next tile has landed.
// 256 x 256: eight waves of 128 x 64, two on a SIMD (four of 128 x 128 with twice the accumulators need both register files,
// and moves between them: 571 us against 433 at 8192^3). 8192^3: 417 to 466 us by the card, 2635 TOP/s at best, matrix cores
// busy 65 % (the library's product 1824 TOP/s on the card of the 417, 2347 at 16384^3).
// Small tiles are bound by their fragments' way through LDS and by the two rounds of its latency in each K tile, which
// deeper stages do not shorten.
template <class E, int EPI, int BM, int BN, int WGM, int WGN, int NST>
__global__ __launch_bounds__(WGM * WGN * 64) void int8_tile_kernel(Int8Gemm g) {
  constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16;
  constexpr int STAGE = (BM + BN) * 128, L = (BM + BN) / (8 * NW);  // a wave's loads of a tile
  static_assert(WM % 16 == 0 && WN % 16 == 0 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole blocks and loads");
  static_assert(NST >= 2 && NST <= 4 && (NST - 1) * L < 64, "wait_tiles, vmcnt range");
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, l16 = lane & 15, G = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  // Tiles of one XCD (workgroups b, b + 8, ..) lie side by side, in groups of 8 rows of tiles.
  const int tiles = gridDim.x, b = blockIdx.x, xcd = b & 7, q = tiles >> 3, rest = tiles & 7;
  const int tile = xcd * q + min(xcd, rest) + (b >> 3);
  const int group = tile / (8 * g.tiles_n), first = group * 8, in = tile - group * 8 * g.tiles_n;
  const int high = min(8, g.tiles_m - first), tm = first + in % high, tn = in / high;
  const int m0 = tm * BM, n0 = tn * BN;

  const i32x4_t ra = make_buffer_rsrc(g.a + (int64_t)m0 * g.lda,
                                      (uint32_t)(min(BM, g.M - m0) - 1) * (uint32_t)g.lda + (uint32_t)g.K);
  const i32x4_t rw = make_buffer_rsrc(g.w + (int64_t)n0 * g.ldw,
                                      (uint32_t)(min(BN, g.N - n0) - 1) * (uint32_t)g.ldw + (uint32_t)g.K);
  const int lrow = 8 * wave + (lane >> 3);  // of the 8 rows that one load fills
  const uint32_t chunk = (uint32_t)((lane & 7) ^ ((lrow >> 1) & 7)) << 4;
  const uint32_t va = (uint32_t)lrow * (uint32_t)g.lda + chunk, vw = (uint32_t)lrow * (uint32_t)g.ldw + chunk;
  auto load = [&](int kt, int i) __attribute__((always_inline)) {  // load i of L: rows of A, then of W
    unsigned char* st = smem + (kt % NST) * STAGE + (i * NW + wave) * 1024;
    const uint32_t k0 = (uint32_t)kt * 128u;
    if (i * 8 * NW < BM) buffer_load_lds16(ra, st, va + (uint32_t)(i * 8 * NW) * (uint32_t)g.lda + k0);
    else buffer_load_lds16(rw, st, vw + (uint32_t)(i * 8 * NW - BM) * (uint32_t)g.ldw + k0);
  };

  struct Frags {
    i32x4v_t a[FM], w[FN];
  };
  const int swz = (l16 >> 1) & 7;
  const int aoff = (wm * WM + l16) * 128, woff = (BM + wn * WN + l16) * 128;
  const int slot[2] = {(G ^ swz) << 4, ((4 + G) ^ swz) << 4};
  // Fragment f of a step: the weight's first, which the step's first products all need.
  auto read = [&](Frags& x, const unsigned char* st, int s, int f) __attribute__((always_inline)) {
    if (f < FN) x.w[f] = *reinterpret_cast<const i32x4v_t*>(st + woff + slot[s] + f * 2048);
    else x.a[f - FN] = *reinterpret_cast<const i32x4v_t*>(st + aoff + slot[s] + (f - FN) * 2048);
  };
  i32x4v_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4v_t{0, 0, 0, 0};
  // One step: the products of `cur`, one row of blocks at a time, with the reads of `nxt` (step s of stage `st`) and the
  // loads of K tile kt spread over them. PART: a wave whose last rows are past M leaves those blocks out.
  constexpr int RPR = (FM + FN + FM - 1) / FM, LPR = (L + FM - 1) / FM;  // reads and loads for each row of blocks
  const int blocks = min(FM, (g.M - m0 - wm * WM + 15) / 16);
  auto step = [&](const Frags& cur, Frags& nxt, const unsigned char* st, int s, int kt, auto reads, auto loads, auto part)
      __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (decltype(reads)::value)
#pragma unroll
        for (int f = i * RPR; f < (i + 1) * RPR; ++f)
          if (f < FM + FN) read(nxt, st, s, f);
      if constexpr (decltype(loads)::value)
#pragma unroll
        for (int f = i * LPR; f < (i + 1) * LPR; ++f)
          if (f < L) load(kt, f);
      if (!decltype(part)::value || i < blocks) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.w[j], cur.a[i], acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using Yes = std::true_type;
  using No = std::false_type;
  const int KT = (g.K + 127) / 128;
  auto wait_tiles = [&](int n) __attribute__((always_inline)) {  // the loads of n tiles, NST - 2 at most, may stay in flight
    if constexpr (NST > 3) {
      if (n >= 2) return wait_vmcnt<2 * L>();
    }
    if constexpr (NST > 2) {
      if (n >= 1) return wait_vmcnt<L>();
    }
    wait_vmcnt<0>();
  };
  Frags x, y;
  auto run = [&](auto part) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < FM + FN; ++f) read(x, smem, 0, f);
    int kt = 0, st = 0;
    auto middle = [&](int n) __attribute__((always_inline)) {
      wait_tiles(n);
      block_barrier();
    };
    auto next = [&]() { return st + 1 == NST ? 0 : st + 1; };
    for (; kt + NST < KT; ++kt) {
      step(x, y, smem + st * STAGE, 1, 0, Yes{}, No{}, part);
      middle(NST - 2);
      st = next();
      step(y, x, smem + st * STAGE, 0, kt + NST, Yes{}, Yes{}, part);
    }
    for (; kt + 1 < KT; ++kt) {
      step(x, y, smem + st * STAGE, 1, 0, Yes{}, No{}, part);
      middle(KT - 2 - kt);
      st = next();
      step(y, x, smem + st * STAGE, 0, 0, Yes{}, No{}, part);
    }
    step(x, y, smem + st * STAGE, 1, 0, Yes{}, No{}, part);
    if (g.K % 128 == 0) step(y, x, smem, 0, 0, No{}, No{}, part);  // K = 64 mod 128: that half holds other rows' bytes
  };
#pragma unroll
  for (int t = 0; t < NST; ++t)
    if (t < KT)
#pragma unroll
      for (int f = 0; f < L; ++f) load(t, f);
  wait_tiles(min(NST, KT) - 1);
  block_barrier();
  run(std::integral_constant<bool, (BM >= 128)>{});

  // Epilogue. A wave writes its outputs in fp32, bias and gamma applied, to LDS, RB rows at a time, and takes them up again
  // in rows, 8 columns a lane, for the residual and the stores.
  constexpr int RB = WM % 32 ? 16 : 32, LD = WN + 4, CL = WN / 8, RPP = 64 / CL;  // rows of a pass over the lanes
  static_assert(WM % RB == 0 && 64 % CL == 0 && RB % RPP == 0, "rows of the epilogue");
  block_barrier();  // (every wave is done with the stages)
  float* park = reinterpret_cast<float*>(smem) + wave * RB * LD;
  typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));
  auto four = [&](const uint16_t* p, float* f) __attribute__((always_inline)) {
    const u16x4_t v = *reinterpret_cast<const u16x4_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = E::value(v[e]);
  };
  constexpr bool LS = EPI == OUDJAT_EPI_BIAS_LS || EPI == OUDJAT_EPI_BIAS_LS_RESID;
  constexpr bool RESID = EPI == OUDJAT_EPI_BIAS_LS_RESID || EPI == OUDJAT_EPI_BIAS_SILU_MUL;
  float sw[FN][4], bias[FN][4], gamma[FN][4];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int n = min(n0 + wn * WN + 16 * j + 4 * G, g.N - 4);  // (columns past the last are not stored)
    const float4 s4 = *reinterpret_cast<const float4*>(g.sw + n);
    sw[j][0] = s4.x; sw[j][1] = s4.y; sw[j][2] = s4.z; sw[j][3] = s4.w;
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[j][e] = 0.0f;
    if (g.bias) four(g.bias + n, bias[j]);
    if constexpr (LS) four(g.gamma + n, gamma[j]);
  }
  const int cl = lane % CL, n = n0 + wn * WN + 8 * cl;
#pragma unroll
  for (int h = 0; h < WM / RB; ++h) {
    const int mh = m0 + wm * WM + h * RB;
    if (mh >= g.M) break;  // uniform over the wave
    uint4 resid[RESID ? RB / RPP : 1];  // (on their way while the outputs go through LDS)
    if constexpr (RESID)
#pragma unroll
      for (int r = 0; r < RB / RPP; ++r)
        resid[r] = load16(g.resid + (int64_t)min(mh + r * RPP + lane / CL, g.M - 1) * g.ldr + min(n, g.N - 8));
    float sa[RB / 16];
#pragma unroll
    for (int i = 0; i < RB / 16; ++i) sa[i] = g.sa[min(mh + 16 * i + l16, g.M - 1)];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < RB / 16; ++i) {
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = __builtin_fmaf((float)acc[h * (RB / 16) + i][j][e], sa[i] * sw[j][e], bias[j][e]);
          if constexpr (LS) v[e] *= gamma[j][e];
        }
        *reinterpret_cast<f32x4_t*>(park + (16 * i + l16) * LD + 16 * j + 4 * G) = v;
      }
#pragma unroll
    for (int r = 0; r < RB / RPP; ++r) {
      const int row = r * RPP + lane / CL, m = mh + row;
      const float* src = park + row * LD + 8 * cl;
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(src), hi = *reinterpret_cast<const f32x4_t*>(src + 4);
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if constexpr (RESID) {
        float t[8];
        E::to8(resid[r], t);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = EPI == OUDJAT_EPI_BIAS_LS_RESID ? v[e] + t[e] : silu(v[e]) * t[e];
      }
      if (m < g.M && n < g.N) store_row<(BM >= 128)>(g.c + (int64_t)m * g.ldc + n, E::from8(v));
    }
  }
}

}  // namespace oudjat

using namespace oudjat;

extern "C" int oudjat_quantize_int8(const uint16_t* x, int64_t rows, int64_t K, int64_t x_rs, int dtype, int8_t* codes,
                                    int64_t c_rs, float* scale, oudjat_stream_t stream) {
  const char* what = "quantize_int8";
  OUDJAT_REQUIRE(rows >= 0 && K >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(K % 16 == 0, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: K=%lld (a multiple of 16)", what, (long long)K);
  if (rows == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE(scale && (K == 0 || (x && codes)), OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(aligned(scale, 4) && (K == 0 || (x_rs >= 0 && x_rs % 8 == 0 && c_rs % 16 == 0 && aligned(x, 16) &&
                                                  aligned(codes, 16))),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned rows required", what);
  OUDJAT_REQUIRE(entries_apart({{rows, c_rs}}, K), OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: the rows of codes must not overlap",
                 what);
  // (a launch holds less than 2^32 threads)
  OUDJAT_REQUIRE(cdiv(rows, K <= kWaveRow ? 4 : 1) < (1 << 24) && K < (1 << 30), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  auto go = [&](auto e, auto lanes, auto ch, auto lng) {
    constexpr int L = decltype(lanes)::value;
    quantize_int8_kernel<decltype(e), L, decltype(ch)::value, decltype(lng)::value>
        <<<(unsigned)cdiv(rows, 256 / L), 256, 0, as_stream(stream)>>>(x, rows, (int)K, x_rs, codes, c_rs, scale);
  };
  using std::integral_constant;
  auto by_len = [&](auto e) {
    if (K <= kWaveRow) go(e, integral_constant<int, 64>{}, integral_constant<int, 2>{}, std::false_type{});
    else if (K <= 4096) go(e, integral_constant<int, 256>{}, integral_constant<int, 2>{}, std::false_type{});
    else if (K <= 8192) go(e, integral_constant<int, 256>{}, integral_constant<int, 4>{}, std::false_type{});
    else go(e, integral_constant<int, 256>{}, integral_constant<int, 4>{}, std::true_type{});
  };
  if (dtype == OUDJAT_BF16) by_len(QuantBf16{});
  else by_len(QuantFp16{});
  return check_launch(what);
}

template <class E, int EPI, int BM, int BN, int WGM, int WGN, int NST>
static int launch_tile(Int8Gemm g, hipStream_t st, const char* what) {
  static std::atomic<uint64_t> done{0};
  g.tiles_m = (int)cdiv(g.M, BM);
  g.tiles_n = (int)cdiv(g.N, BN);
  constexpr int RB = BM / WGM % 32 ? 16 : 32;  // rows of a wave that the epilogue stages
  constexpr int lds = std::max(NST * (BM + BN) * 128, WGM * WGN * RB * (BN / WGN + 4) * 4);
  const auto fn = int8_tile_kernel<E, EPI, BM, BN, WGM, WGN, NST>;
  const int rc = allow_lds((const void*)fn, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  fn<<<(unsigned)g.tiles_m * g.tiles_n, WGM * WGN * 64, lds, st>>>(g);
  return check_launch(what);
}

template <class E, int EPI>
static int launch_direct(Int8Gemm g, hipStream_t st, const char* what) {
  g.tiles_m = (int)cdiv(g.M, 16);
  g.tiles_n = (int)cdiv(g.N, 16);
  int8_direct_kernel<E, EPI><<<(unsigned)g.tiles_m * g.tiles_n, kDirectWaves * 64, 0, st>>>(g);
  return check_launch(what);
}

// The kernels, and the time of a call in us: start + rounds of tiles over the CUs x (K tiles x per_k + per_tile), fitted to
// 74 shapes (1 .. 16404 rows, N 64 .. 12288, K 64 .. 8192) that ran with each of them on one card; the kernel that this
// chooses is 1 % slower than the fastest on the mean, 16 % at most (668 x 256 x 1088: 5.2 us by 64 x 64 tiles, 4.5 directly).
// Where the others lie, us by 16 x 16 directly / 64 x 64 / 64 x 128 / 128 x 128 / 192 x 256 / 256 x 256:
//   1 x 4096 x 4096: 5.9 / 9.4 / 12 / 21 / 28 / 30;  32 x 8192 x 4096: 17 / 9.8 / 13 / 22 / 28 / 30;
//   512 x 4096 x 4096: 114 / 16 / 14 / 25 / 40 / 47;  1656 x 4096 x 8192: 727 / 90 / 78 / 60 / 76 / 87;
//   1656 x 12288 x 4096: 1090 / 134 / 110 / 97 / 91 / 101;  16404 x 4096 x 8192: - / 833 / 671 / 547 / 504 / 499 (452 in
//   two launches, below). These and the figures of splits below were taken when all tiles stored through the caches.
struct Int8Tile {
  int bm, bn, threads;
  float start, per_k, per_tile;
};
static const Int8Tile kInt8Tiles[] = {
    {16, 16, kDirectWaves * 64, 2.29f, 0.088f, 0.2f}, {64, 64, 256, 2.27f, 0.189f, 0.91f},
    {64, 128, 512, 1.97f, 0.292f, 1.39f},             {128, 128, 256, 2.5f, 0.479f, 2.39f},
    {192, 256, 512, 1.0f, 1.18f, 6.87f},              {256, 256, 512, 1.0f, 1.346f, 9.13f},
};
static constexpr int kInt8Kinds = sizeof(kInt8Tiles) / sizeof(kInt8Tiles[0]);
static constexpr int kInt8Large = 4;  // from here on a CU holds one tile at a time
// (a launch holds less than 2^32 threads: a kernel that needs more is never the one)
static constexpr float kInt8Never = 3.40282347e38f;
static float int8_time(const Int8Tile& t, int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = cdiv(M, t.bm) * cdiv(N, t.bn);
  if (tiles * t.threads >= (int64_t)1 << 32) return kInt8Never;
  return t.start + (float)cdiv(tiles, 256) * ((float)K / 128.0f * t.per_k + t.per_tile);
}
static int choose_int8(int64_t M, int64_t N, int64_t K, float& least) {
  int best = 0;
  least = int8_time(kInt8Tiles[0], M, N, K);
  for (int i = 1; i < kInt8Kinds; ++i) {
    const float us = int8_time(kInt8Tiles[i], M, N, K);
    if (us < least) best = i, least = us;
  }
  return best;
}

// Rows of a plan: all by one kernel, or those that fill whole rounds of large tiles and then the rest by smaller ones in a
// second launch. The rest reads the weight once more; a split is taken where the model says that it spares a
// twentieth or more, and only for tiles that a CU holds one at a time, whose rounds are real ones (128 x 128 for 1024 of
// 1300 rows, 4096 x 4096: 39 us, in one launch 33). us in one launch and in two: 4116 x 4096 x 4096: 84, 68;
// 16404 x 1024 x 1024: 34, 28; 4600 x 4096 x 8192: 159, 139; 16404 x 4096 x 8192: 493, 452; 33000 x 4096 x 1024: 201, 197;
// 16404 x 8192 x 4096: 506, 499; not taken, by the twentieth: 5000 x 8192 x 8192: 288, 282; 1656 x 12288 x 4096: 88, 89.
static bool int8_size(int64_t M, int64_t N) {
  return M < (1 << 30) && N < (1 << 30) && cdiv(M, 16) * cdiv(N, 16) < (int64_t)1 << 31;
}
struct Int8Plan {
  int tile, rest;
  int64_t first;  // rows of the first launch
};
static bool plan_int8(int64_t M, int64_t N, int64_t K, Int8Plan& p) {  // false: no kernel's launch holds the call
  float least, rest_us;
  p = Int8Plan{choose_int8(M, N, K, least), 0, M};
  if (least == kInt8Never) return false;
  const float again = (float)N * (float)K / 5e6f;  // the weight at 5 TB/s
  least *= 0.95f;
  for (int i = kInt8Large; i < kInt8Kinds; ++i) {
    const Int8Tile& t = kInt8Tiles[i];
    const int64_t across = cdiv(N, t.bn), rounds = cdiv(cdiv(M, t.bm) * across, 256) - 1;
    const int64_t first = rounds * 256 / across * t.bm;
    if (first <= 0 || first >= M) continue;
    const int rest = choose_int8(M - first, N, K, rest_us);
    const float us = int8_time(t, first, N, K) + again + rest_us;
    if (us < least) least = us, p = Int8Plan{i, rest, first};
  }
  return true;
}

template <class E, int EPI>
static int launch_one(int tile, const Int8Gemm& g, hipStream_t st, const char* what) {
  switch (tile) {
    case 0: return launch_direct<E, EPI>(g, st, what);
    case 1: return launch_tile<E, EPI, 64, 64, 2, 2, 4>(g, st, what);
    case 2: return launch_tile<E, EPI, 64, 128, 2, 4, 3>(g, st, what);
    case 3: return launch_tile<E, EPI, 128, 128, 2, 2, 2>(g, st, what);
    case 4: return launch_tile<E, EPI, 192, 256, 2, 4, 2>(g, st, what);
    default: return launch_tile<E, EPI, 256, 256, 2, 4, 2>(g, st, what);
  }
}
template <class E, int EPI>
static int launch_int8(Int8Gemm g, hipStream_t st, const char* what) {
  Int8Plan p;
  if (!plan_int8(g.M, g.N, g.K, p)) return set_error(OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const int rest = g.M - (int)p.first;
  g.M = (int)p.first;
  const int rc = launch_one<E, EPI>(p.tile, g, st, what);
  if (rc != OUDJAT_OK || !rest) return rc;
  g.a += p.first * g.lda;
  g.sa += p.first;
  if (g.resid) g.resid += p.first * g.ldr;
  g.c += p.first * g.ldc;
  g.M = rest;
  return launch_one<E, EPI>(p.rest, g, st, what);
}

extern "C" int oudjat_linear_int8_tile(int64_t M, int64_t N, int64_t K, int* rows, int* columns, int64_t* first) {
  const char* what = "linear_int8_tile";
  OUDJAT_REQUIRE(M > 0 && N > 0 && K > 0 && rows && columns && first, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad argument", what);
  Int8Plan p;
  OUDJAT_REQUIRE(int8_size(M, N) && plan_int8(M, N, K, p), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  *rows = kInt8Tiles[p.tile].bm;
  *columns = kInt8Tiles[p.tile].bn;
  *first = p.first;
  return OUDJAT_OK;
}

extern "C" int oudjat_linear_int8(const int8_t* A, int64_t M, int64_t K, int64_t lda, const float* a_scale,
                                  const int8_t* W, int64_t N, int64_t ldw, const float* w_scale, const uint16_t* bias,
                                  int epi, const uint16_t* gamma, const uint16_t* resid, int64_t ldr, uint16_t* C,
                                  int64_t ldc, int dtype, oudjat_stream_t stream) {
  const char* what = "linear_int8";
  OUDJAT_REQUIRE(M >= 0 && N >= 0 && K >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  OUDJAT_REQUIRE(epi == OUDJAT_EPI_BIAS || epi == OUDJAT_EPI_BIAS_LS_RESID || epi == OUDJAT_EPI_BIAS_LS ||
                     epi == OUDJAT_EPI_BIAS_SILU_MUL,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: unsupported epilogue %d", what, epi);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(K > 0 && K % 64 == 0 && N % 8 == 0, OUDJAT_ERR_UNSUPPORTED_SHAPE,
                 "%s: need K %% 64 == 0 and N %% 8 == 0 (K=%lld, N=%lld)", what, (long long)K, (long long)N);
  OUDJAT_REQUIRE(K < (1 << 17), OUDJAT_ERR_TOO_LARGE, "%s: K=%lld: sums of 2^17 products may pass 32 bits", what,
                 (long long)K);
  if (M == 0 || N == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE(A && a_scale && W && w_scale && C, OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE((epi != OUDJAT_EPI_BIAS_LS && epi != OUDJAT_EPI_BIAS_LS_RESID) || gamma, OUDJAT_ERR_INVALID_ARGUMENT,
                 "%s: epilogue needs gamma", what);
  OUDJAT_REQUIRE((epi != OUDJAT_EPI_BIAS_LS_RESID && epi != OUDJAT_EPI_BIAS_SILU_MUL) || resid,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: epilogue needs resid", what);
  OUDJAT_REQUIRE(lda >= 0 && ldw >= 0 && ldr >= 0 && lda % 16 == 0 && ldw % 16 == 0 && ldc % 8 == 0 && ldr % 8 == 0 &&
                     aligned(A, 16) && aligned(W, 16) && aligned(C, 16) && aligned(resid, 16) && aligned(bias, 16) &&
                     aligned(gamma, 16) && aligned(w_scale, 16) && aligned(a_scale, 4),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned operands and rows required", what);
  OUDJAT_REQUIRE(entries_apart({{M, ldc}}, N), OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: the rows of the output must not overlap",
                 what);
  OUDJAT_REQUIRE(int8_size(M, N) && lda < (1 << 22) && ldw < (1 << 22), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  const Int8Gemm g{A, lda, a_scale, W, ldw, w_scale, bias, gamma, resid, ldr, C, ldc, (int)M, (int)N, (int)K, 0, 0};
  hipStream_t st = as_stream(stream);
  auto by_epi = [&](auto e) {
    using E = decltype(e);
    switch (epi) {
      case OUDJAT_EPI_BIAS: return launch_int8<E, OUDJAT_EPI_BIAS>(g, st, what);
      case OUDJAT_EPI_BIAS_LS: return launch_int8<E, OUDJAT_EPI_BIAS_LS>(g, st, what);
      case OUDJAT_EPI_BIAS_LS_RESID: return launch_int8<E, OUDJAT_EPI_BIAS_LS_RESID>(g, st, what);
      default: return launch_int8<E, OUDJAT_EPI_BIAS_SILU_MUL>(g, st, what);
    }
  };
  return dtype == OUDJAT_BF16 ? by_epi(QuantBf16{}) : by_epi(QuantFp16{});
}
