// INT8 products with a scale for each token and each output channel: the quantiser of rows and the product.
//
//   quantise:  s = max |x| / 127 (fp32),  c = rint(x / s) (nearest even; 0 where s = 0), c in -127 .. 127;
//   product:   y[m, n] = (sum_k a[m, k] w[n, k]) (s_a[m] s_w[n]) + bias[n], the sum exact in int32 (K < 2^17),
// then the epilogue in fp32 and one rounding to the output's type.
#include <algorithm>
#include <atomic>

#include "elem.hpp"
#include "packed_attn.hpp"

namespace oudjat {

typedef int i32x4v_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------
// Quantiser. A row is held in registers by 64 LANES / 64 waves, CH chunks of 8 values a lane, between its maximum and its
// codes, so that it is read once; longer rows are read again. The maximum is taken on the bits without their sign, where
// infinities and NaNs are above all others: such a row gets the scale NaN and the codes 0, so that its products are NaN.
// Quotients are the IEEE ones: with y = RN(1 / s), q0 = RN(x y), r = x - q0 s (exact by an FMA), RN(q0 + r y) is the
// correctly rounded quotient; where s is so small that y overflows or r underflows, x and s are scaled by 2^100 first.
// Adding 1.5 2^23 leaves the nearest whole number (ties to even) in the low byte.
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

// Four outputs of one row, columns n .. n + 3.
template <class E, int EPI>
__device__ __forceinline__ void int8_store4(const Int8Gemm& g, int m, int n, const i32x4v_t& acc) {
  typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));
  const float sa = g.sa[m];
  const float4 sw = *reinterpret_cast<const float4*>(g.sw + n);
  float y[4] = {(float)acc[0] * (sa * sw.x), (float)acc[1] * (sa * sw.y), (float)acc[2] * (sa * sw.z),
                (float)acc[3] * (sa * sw.w)};
  auto four = [&](const uint16_t* p, float* f) {
    const u16x4_t b = *reinterpret_cast<const u16x4_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = E::value(b[e]);
  };
  float t[4];
  if (g.bias) {
    four(g.bias + n, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += t[e];
  }
  if constexpr (EPI == OUDJAT_EPI_BIAS_LS || EPI == OUDJAT_EPI_BIAS_LS_RESID) {
    four(g.gamma + n, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= t[e];
  }
  if constexpr (EPI == OUDJAT_EPI_BIAS_LS_RESID || EPI == OUDJAT_EPI_BIAS_SILU_MUL) {
    four(g.resid + (int64_t)m * g.ldr + n, t);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = EPI == OUDJAT_EPI_BIAS_LS_RESID ? y[e] + t[e] : y[e] / (1.0f + expf(-y[e])) * t[e];
  }
  const float out[8] = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
  const uint4 o = E::from8(out);
  *reinterpret_cast<uint2*>(g.c + (int64_t)m * g.ldc + n) = make_uint2(o.x, o.y);
}

// Tile kernel: BM x BN outputs, WGM x WGN waves, K in steps of 128 bytes through NST stages of LDS, filled by buffer
// loads (descriptors of the tile's rows that exist: others load as zeros). LDS row r keeps its 16-byte chunk c in slot
// c ^ (r / 2) % 8, so that 16 rows at one chunk cover all banks. v_mfma_i32_16x16x64_i8 with the weight as its first
// operand: lane l holds row l % 16, columns 4 (l / 16) .. + 3 of a 16 x 16 block.
template <class E, int EPI, int BM, int BN, int WGM, int WGN, int NST>
__global__ __launch_bounds__(WGM * WGN * 64) void int8_tile_kernel(Int8Gemm g) {
  constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16;
  constexpr int STAGE = (BM + BN) * 128, LA = BM / (8 * NW), LW = BN / (8 * NW), L = LA + LW;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole loads");
  static_assert((NST - 1) * L < 64, "vmcnt range");
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

  const int8_t* A = g.a + (int64_t)m0 * g.lda;
  const int8_t* W = g.w + (int64_t)n0 * g.ldw;
  const i32x4_t ra = make_buffer_rsrc(A, (uint32_t)(min(BM, g.M - m0) - 1) * (uint32_t)g.lda + (uint32_t)g.K);
  const i32x4_t rw = make_buffer_rsrc(W, (uint32_t)(min(BN, g.N - n0) - 1) * (uint32_t)g.ldw + (uint32_t)g.K);
  const int lrow = lane >> 3;  // of the 8 rows that one load fills
  const uint32_t chunk = (uint32_t)(((lane & 7) ^ ((8 * wave + lrow) >> 1)) & 7) << 4;
  const uint32_t va = (uint32_t)(8 * wave + lrow) * (uint32_t)g.lda + chunk;
  const uint32_t vw = (uint32_t)(8 * wave + lrow) * (uint32_t)g.ldw + chunk;
  auto issue = [&](int kt) __attribute__((always_inline)) {
    unsigned char* st = smem + (kt % NST) * STAGE + wave * 1024;
    const uint32_t k0 = (uint32_t)kt * 128u;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      buffer_load_lds16(ra, st + i * NW * 1024, va + (uint32_t)(i * 8 * NW) * (uint32_t)g.lda + k0);
#pragma unroll
    for (int i = 0; i < LW; ++i)
      buffer_load_lds16(rw, st + BM * 128 + i * NW * 1024, vw + (uint32_t)(i * 8 * NW) * (uint32_t)g.ldw + k0);
  };
  auto at = [&](int row, int c) { return row * 128 + ((c ^ ((row >> 1) & 7)) << 4); };

  i32x4v_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4v_t{0, 0, 0, 0};
  const int KT = (g.K + 127) / 128;
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (s < KT) issue(s);
  for (int kt = 0; kt < KT; ++kt) {
    // Tile kt has landed when only the loads of the tiles after it are in flight.
    if (NST == 2 || kt + 1 >= KT) wait_vmcnt<0>();
    else if (NST == 3 || kt + 2 >= KT) wait_vmcnt<L>();
    else wait_vmcnt<2 * L>();
    block_barrier();
    if (kt + NST - 1 < KT) issue(kt + NST - 1);
    const unsigned char* st = smem + (kt % NST) * STAGE;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s == 1 && kt * 128 + 64 >= g.K) break;  // K = 64 mod 128: the last half tile holds other rows' bytes
      i32x4v_t fa[FM], fw[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i)
        fa[i] = *reinterpret_cast<const i32x4v_t*>(st + at(wm * WM + 16 * i + l16, 4 * s + G));
#pragma unroll
      for (int j = 0; j < FN; ++j)
        fw[j] = *reinterpret_cast<const i32x4v_t*>(st + BM * 128 + at(wn * WN + 16 * j + l16, 4 * s + G));
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * WM + 16 * i + l16;
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn * WN + 16 * j + 4 * G;
      if (n < g.N) int8_store4<E, EPI>(g, m, n, acc[i][j]);
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
  OUDJAT_REQUIRE(rows < (1 << 26) && K < (1 << 30), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  auto go = [&](auto e, auto lanes, auto ch, auto lng) {
    constexpr int L = decltype(lanes)::value;
    quantize_int8_kernel<decltype(e), L, decltype(ch)::value, decltype(lng)::value>
        <<<(unsigned)cdiv(rows, 256 / L), 256, 0, as_stream(stream)>>>(x, rows, (int)K, x_rs, codes, c_rs, scale);
  };
  using std::integral_constant;
  auto by_len = [&](auto e) {
    if (K <= 1024) go(e, integral_constant<int, 64>{}, integral_constant<int, 2>{}, std::false_type{});
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
  constexpr int lds = NST * (BM + BN) * 128;
  const auto fn = int8_tile_kernel<E, EPI, BM, BN, WGM, WGN, NST>;
  const int rc = allow_lds((const void*)fn, lds, done, what);
  if (rc != OUDJAT_OK) return rc;
  g.tiles_m = (int)cdiv(g.M, BM);
  g.tiles_n = (int)cdiv(g.N, BN);
  fn<<<(unsigned)g.tiles_m * g.tiles_n, WGM * WGN * 64, lds, st>>>(g);
  return check_launch(what);
}

template <class E, int EPI>
static int launch_int8(const Int8Gemm& g, hipStream_t st, const char* what) {
  return launch_tile<E, EPI, 128, 128, 2, 2, 2>(g, st, what);
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
  OUDJAT_REQUIRE(M < (1 << 30) && N < (1 << 30) && lda < (1 << 22) && ldw < (1 << 22) &&
                     cdiv(M, 16) * cdiv(N, 16) < ((int64_t)1 << 31),
                 OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
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
