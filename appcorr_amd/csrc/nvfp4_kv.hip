// K/V caches in NVFP4: rows of keys and values written into one, and rows of it read back in 16 bits.
//
// A block is 16 consecutive dims of one head of one token. With h the head's tensor scale (fp32, one each for keys and
// values), a = max |x| over the block:
//   s8 = e4m3(clamp((a / 6) / h, 2^-16, 448)),   code_i = e2m1(x_i / (h s8)),   value_i = e2m1(code_i) e4m3(s8) h,
// the element arithmetic of nvfp4.hpp (IEEE quotients, nearest even, saturating). A block whose scale rounds to 0 holds
// zeros; a NaN counts as 0 and an infinity as the largest value, for which the format has nothing else: what a cache
// holds is finite. Element 2i lies in the low nibble of byte i. The scale bytes are read without their sign bit, and
// 0x7f (never written) as 480, so that memory that nobody has written cannot give a NaN either.
#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "nvfp4_kv.hpp"

namespace oudjat {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

static constexpr int kKvThreads = 256;

// Reciprocal of a normal b whose reciprocal is normal too: one Newton step on the hardware's, which is within an ulp, gives
// the correctly rounded one, for all significands but all ones by the theory, where it hangs on the hardware's own rounding. On
// gfx950 it is IEEE's 1 / b for each of the 2^23 significands with each of 250 exponents.
__device__ __forceinline__ float rcp_rn(float b) {
  const float y = __builtin_amdgcn_rcpf(b);
  return __builtin_fmaf(__builtin_fmaf(-b, y, 1.0f), y, y);
}
// a / b correctly rounded, y = RN(1 / b), where nothing leaves the normal range: a - q0 b is exact.
__device__ __forceinline__ float quotient(float a, float b, float y) {
  const float q0 = a * y;
  return __builtin_fmaf(__builtin_fmaf(-q0, b, a), y, q0);
}

// Workgroups of one XCD (b, b + 8, ..) take consecutive rows, whose slots mostly lie side by side: a line of codes holds two
// tokens of a head, one of scales 16, and it is in one L2.
__device__ __forceinline__ int64_t xcd_group() {
  const int n = gridDim.x, b = blockIdx.x, xcd = b & 7, q = n >> 3, rest = n & 7;
  return xcd * q + min(xcd, rest) + (b >> 3);
}

// A block's scale byte and codes. The usual block is finite, its values and the tensor scale are of ordinary size, and the
// scale is neither cut off nor rounded to 0; any other takes IEEE divisions and the limits that the format needs.
template <class E>
__device__ __forceinline__ uint2 quantize_block(const uint4& lo, const uint4& hi, float ts, uint32_t& s8) {
  float f[16];
  E::to8(lo, f);
  E::to8(hi, f + 8);
  float am = 0.0f, z = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    am = fmaxf(am, fabsf(f[e]));
    z = __builtin_fmaf(f[e], 0.0f, z);  // NaN if any value is not finite
  }
  const float scaled = quotient(quotient(am, kE2m1Max, 1.0f / kE2m1Max), ts, rcp_rn(ts));
  if (__builtin_expect(z == 0.0f && am > 1e-18f && ts > 1e-18f && ts < 1e18f && scaled > 0.001f && scaled <= kE4m3Max, 1)) {
    s8 = e4m3_encode_pos(scaled);
    const float unit = ts * e4m3_decode(s8), y = rcp_rn(unit);
    return make_uint2(nvfp4_codes8(f, unit, y), nvfp4_codes8(f + 8, unit, y));
  }
  am = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    f[e] = f[e] == f[e] ? f[e] : 0.0f;
    am = fmaxf(am, fabsf(f[e]));
  }
  float unit;
  nvfp4_block_scale(am, ts, s8, unit);
  if (!s8) return make_uint2(0, 0);
  // (values past 8 units saturate all the same, and their quotients stay finite)
  const float most = 8.0f * unit, y = 1.0f / unit;
#pragma unroll
  for (int e = 0; e < 16; ++e) f[e] = fminf(fmaxf(f[e], -most), most);
  return make_uint2(nvfp4_codes8(f, unit, y), nvfp4_codes8(f + 8, unit, y));
}

// UNI: a row is whole waves of items, so that what belongs to the row alone (its slot, its addresses) is the scalar unit's
// (reads of 16404 rows of 32 heads of 128: 195 -> 189 us as they were then, of 4116 of 16 of 64 13.3 -> 12.6).
template <bool UNI>
__device__ __forceinline__ int row_of(int r) {
  return UNI ? __builtin_amdgcn_readfirstlane(r) : r;
}

// Write. An item is a block, 16 dims of a head: the wave reads and writes consecutive pieces of a row, and one lane in four
// stores four scales. A workgroup takes `per_wg` rows. Bound by HBM and by the pieces' ends: a token of a head is 64 or 32
// bytes of codes and 8 or 4 of scales. 16404 rows of 32 heads of 128, 344 MB, us: in slot order 73 (4.7 TB/s; without the
// order by XCD 77), shuffled 87; 4116 of 16 of 64: 7.9 and 8.7 (8.4 and 9.0 with two rounds of items a workgroup). The
// quantisation's VALU instructions take 80 % of the SIMDs' cycles (with IEEE divisions for every block and value: 114 us).
template <class E, bool UNI>
__global__ __launch_bounds__(kKvThreads) void kv_nvfp4_write_kernel(
    const uint16_t* __restrict__ k, int64_t k_rs, int64_t k_hs, const uint16_t* __restrict__ v, int64_t v_rs,
    int64_t v_hs, int64_t rows, int blocks, Divisor by_row, Divisor by_head, const int64_t* __restrict__ batch_idx,
    const int64_t* __restrict__ token_idx, KvNvfp4 c, int per_wg) {
  const int64_t row0 = xcd_group() * per_wg;
  const int n = (int)min((int64_t)per_wg, rows - row0), per_row = 2 * c.Hk * blocks;
  for (int i = threadIdx.x; i < n * per_row; i += kKvThreads) {
    const int r = row_of<UNI>(by_row(i)), j = i - r * per_row;
    const int kh = by_head(j), d16 = j - kh * blocks;  // key heads, then value heads; 16 dims
    const bool val = kh >= c.Hk;
    const int h = val ? kh - c.Hk : kh;
    const int64_t row = row0 + r;
    const uint16_t* src = (val ? v + row * v_rs + h * v_hs : k + row * k_rs + h * k_hs) + 16 * d16;
    const uint4 lo = load16(src), hi = load16(src + 8);
    const int64_t b = batch_idx[row], t = token_idx[row];
    uint32_t s8;
    const uint2 codes = quantize_block<E>(lo, hi, c.ts[kh], s8);
    uint32_t four = s8 << (8 * (d16 & 3));  // four blocks' scales into one word
    four |= __shfl_xor(four, 1, 64);
    four |= __shfl_xor(four, 2, 64);
    if (b < 0 || b >= c.B || t < 0 || t >= c.N) continue;
    *reinterpret_cast<uint2*>(c.codes + b * c.bs + t * c.ns + (val ? c.cs : 0) + h * c.hs + 8 * d16) = codes;
    if ((d16 & 3) == 0)
      *reinterpret_cast<uint32_t*>(c.scales + b * c.sbs + t * c.sns + (val ? c.scs : 0) + h * c.shs + d16) = four;
  }
}

// The value of the lane next to this one (l ^ 1).
__device__ __forceinline__ uint32_t swap_lanes(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true);
}

// Read. An item is a block: 8 bytes of codes and a scale byte in, 32 bytes out. Two lanes exchange halves of their blocks, so
// that a wave's store is one piece of memory, and the stores bypass the caches, which then keep the lines of the cache
// that neighbouring tokens share. 16404 rows of 32 heads of 128 written and as many others, 690 MB in all, us: in slot order
// 120 (5.7 TB/s), shuffled 168; through the caches 181 and 193; pieces of 16 bytes of two lanes' blocks past the caches 271,
// 263; two blocks a thread 125, 214. What reads the rows next fetches them from memory: with a copy of them behind the read 32 rows
// of 8 heads of 128 take 8.1 us (7.5 if stored through the caches), 512 9 to 10 (9), 4096 21.5 (21.3), 8192 31 (29), 32296 of 32
// heads 360 (383); with one token's attention over 512 of them 14.4 (12.2).
template <class E, bool UNI>
__global__ __launch_bounds__(kKvThreads) void kv_nvfp4_read_kernel(KvNvfp4 c, int blocks, Divisor by_row, Divisor by_head,
                                                                   const int64_t* __restrict__ batch_idx,
                                                                   const int64_t* __restrict__ token_idx, int64_t rows,
                                                                   uint16_t* __restrict__ k_out,
                                                                   uint16_t* __restrict__ v_out, int per_wg) {
  const int64_t row0 = xcd_group() * per_wg;
  const int n = (int)min((int64_t)per_wg, rows - row0), per_row = 2 * c.Hk * blocks;
  const bool odd = threadIdx.x & 1;
  for (int i = threadIdx.x; i < n * per_row; i += kKvThreads) {
    const int r = row_of<UNI>(by_row(i)), j = i - r * per_row;
    const int kh = by_head(j), d16 = j - kh * blocks;
    const bool val = kh >= c.Hk;
    const int h = val ? kh - c.Hk : kh;
    const int64_t row = row0 + r, b = batch_idx[row], t = token_idx[row];
    uint2 w = make_uint2(0, 0);  // a slot outside the cache: zeros, whatever the tensor scale is
    uint32_t s8 = 0;
    float ts = 0.0f;
    if (b >= 0 && b < c.B && t >= 0 && t < c.N) {
      w = *reinterpret_cast<const uint2*>(c.codes + b * c.bs + t * c.ns + (val ? c.cs : 0) + h * c.hs + 8 * d16);
      s8 = c.scales[b * c.sbs + t * c.sns + (val ? c.scs : 0) + h * c.shs + d16];
      ts = c.ts[kh];
    }
    const float s = e4m3_decode(s8 & 0x7f);
    float f[16];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t x = half ? w.y : w.x;
      const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 0);
      const auto v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 1);
      const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 2);
      const auto v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 3);
      const float e2[8] = {v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[8 * half + e] = (e2[e] * s) * ts;  // (the first product is exact)
    }
    const u32x4_t lo = __builtin_bit_cast(u32x4_t, E::from8(f)), hi = __builtin_bit_cast(u32x4_t, E::from8(f + 8));
    u32x4_t first, second;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t got = swap_lanes(odd ? lo[e] : hi[e]);  // (a row has an even number of blocks: both lanes are here)
      first[e] = odd ? got : lo[e];
      second[e] = odd ? hi[e] : got;
    }
    uint16_t* dst = (val ? v_out : k_out) + (row * c.Hk + h) * (16 * blocks) + 16 * (d16 & ~1) + (odd ? 8 : 0);
    __builtin_nontemporal_store(first, reinterpret_cast<u32x4_t*>(dst));
    __builtin_nontemporal_store(second, reinterpret_cast<u32x4_t*>(dst + 16));
  }
}

// Rows of a workgroup: as many whole ones as its threads, one at the least.
static int kv_rows_per_wg(int64_t per_row) { return (int)std::max<int64_t>(1, kKvThreads / per_row); }

int check_kv_nvfp4(const KvNvfp4& c, int64_t Dh, const char* what) {
  OUDJAT_REQUIRE(c.bs >= 0 && c.ns >= 0 && c.cs >= 0 && c.hs >= 0 && c.sbs >= 0 && c.sns >= 0 && c.scs >= 0 && c.shs >= 0,
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: negative stride", what);
  OUDJAT_REQUIRE(((c.bs | c.ns | c.cs | c.hs) % 16) == 0 && ((c.sbs | c.sns | c.scs | c.shs) % (Dh / 16)) == 0 &&
                     aligned(c.codes, 16) && aligned(c.scales, Dh / 16) && aligned(c.ts, 4),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: a head's codes must be 16-byte aligned, its scales by their own size",
                 what);
  return OUDJAT_OK;
}

}  // namespace oudjat

using namespace oudjat;

extern "C" int oudjat_kv_nvfp4_write(const uint16_t* k, int64_t k_rs, int64_t k_hs, const uint16_t* v, int64_t v_rs,
                                     int64_t v_hs, int64_t rows, int64_t Hk, int64_t Dh, int dtype,
                                     const int64_t* batch_idx, const int64_t* token_idx, uint8_t* codes, int64_t c_bs,
                                     int64_t c_ns, int64_t c_cs, int64_t c_hs, uint8_t* scales, int64_t s_bs,
                                     int64_t s_ns, int64_t s_cs, int64_t s_hs, const float* tensor_scale, int64_t B,
                                     int64_t N, oudjat_stream_t stream) {
  const char* what = "kv_nvfp4_write";
  OUDJAT_REQUIRE(rows >= 0 && Hk > 0 && Dh > 0 && B >= 0 && N >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad size", what);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(Dh == 64 || Dh == 128, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (64 or 128)", what, (long long)Dh);
  OUDJAT_REQUIRE(Hk <= 65535, OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  if (rows == 0) return OUDJAT_OK;
  const bool empty = B == 0 || N == 0;  // a cache without slots: every row is skipped
  OUDJAT_REQUIRE(k && v && batch_idx && token_idx && ((codes && scales) || empty) && tensor_scale,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(k_rs >= 0 && k_hs >= 0 && v_rs >= 0 && v_hs >= 0 && ((k_rs | k_hs | v_rs | v_hs) % 8) == 0 &&
                     aligned(k, 16) && aligned(v, 16) && aligned(batch_idx, 8) && aligned(token_idx, 8),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned rows and heads of k and v required", what);
  const KvNvfp4 c{codes, c_bs, c_ns, c_cs, c_hs, scales, s_bs, s_ns, s_cs, s_hs, tensor_scale, B, N, (int)Hk};
  const int rc = check_kv_nvfp4(c, Dh, what);
  if (rc != OUDJAT_OK) return rc;
  OUDJAT_REQUIRE(entries_apart({{B, c_bs}, {N, c_ns}, {2, c_cs}, {Hk, c_hs}}, Dh / 2) &&
                     entries_apart({{B, s_bs}, {N, s_ns}, {2, s_cs}, {Hk, s_hs}}, Dh / 16),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: the rows of the cache must not overlap", what);
  const int64_t per_row = 2 * Hk * Dh / 16;
  const int per = kv_rows_per_wg(per_row);
  OUDJAT_REQUIRE(cdiv(rows, per) < (1 << 24), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  if (empty) return OUDJAT_OK;
  auto go = [&](auto e, auto uni) {
    kv_nvfp4_write_kernel<decltype(e), decltype(uni)::value><<<(unsigned)cdiv(rows, per), kKvThreads, 0, as_stream(stream)>>>(
        k, k_rs, k_hs, v, v_rs, v_hs, rows, (int)(Dh / 16), Divisor((uint32_t)per_row), Divisor((uint32_t)(Dh / 16)),
        batch_idx, token_idx, c, per);
  };
  auto by_row = [&](auto e) { per_row % 64 ? go(e, std::false_type{}) : go(e, std::true_type{}); };
  if (dtype == OUDJAT_BF16) by_row(ElemBf16{});
  else by_row(ElemFp16{});
  return check_launch(what);
}

extern "C" int oudjat_kv_nvfp4_read(const uint8_t* codes, int64_t c_bs, int64_t c_ns, int64_t c_cs, int64_t c_hs,
                                    const uint8_t* scales, int64_t s_bs, int64_t s_ns, int64_t s_cs, int64_t s_hs,
                                    const float* tensor_scale, int64_t B, int64_t N, int64_t Hk, int64_t Dh,
                                    const int64_t* batch_idx, const int64_t* token_idx, int64_t rows, int dtype,
                                    uint16_t* k_out, uint16_t* v_out, oudjat_stream_t stream) {
  const char* what = "kv_nvfp4_read";
  OUDJAT_REQUIRE(rows >= 0 && Hk > 0 && Dh > 0 && B >= 0 && N >= 0, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad size", what);
  OUDJAT_REQUIRE(dtype == OUDJAT_BF16 || dtype == OUDJAT_FP16, OUDJAT_ERR_INVALID_ARGUMENT, "%s: bad element type %d",
                 what, dtype);
  OUDJAT_REQUIRE(Dh == 64 || Dh == 128, OUDJAT_ERR_UNSUPPORTED_SHAPE, "%s: Dh=%lld (64 or 128)", what, (long long)Dh);
  OUDJAT_REQUIRE(Hk <= 65535, OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  if (rows == 0) return OUDJAT_OK;
  OUDJAT_REQUIRE(batch_idx && token_idx && ((codes && scales) || B == 0 || N == 0) && tensor_scale && k_out && v_out,
                 OUDJAT_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  OUDJAT_REQUIRE(k_out != v_out, OUDJAT_ERR_INVALID_ARGUMENT, "%s: k_out and v_out are the same buffer", what);
  const KvNvfp4 c{const_cast<uint8_t*>(codes), c_bs, c_ns, c_cs, c_hs, const_cast<uint8_t*>(scales), s_bs, s_ns, s_cs,
                  s_hs, tensor_scale, B, N, (int)Hk};
  const int rc = check_kv_nvfp4(c, Dh, what);
  if (rc != OUDJAT_OK) return rc;
  OUDJAT_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16) && aligned(batch_idx, 8) && aligned(token_idx, 8),
                 OUDJAT_ERR_UNSUPPORTED_LAYOUT, "%s: 16-byte aligned outputs required", what);
  const int64_t per_row = 2 * Hk * Dh / 16;
  const int per = kv_rows_per_wg(per_row);
  OUDJAT_REQUIRE(cdiv(rows, per) < (1 << 24), OUDJAT_ERR_TOO_LARGE, "%s: too large", what);
  auto go = [&](auto e, auto uni) {
    kv_nvfp4_read_kernel<decltype(e), decltype(uni)::value><<<(unsigned)cdiv(rows, per), kKvThreads, 0, as_stream(stream)>>>(
        c, (int)(Dh / 16), Divisor((uint32_t)per_row), Divisor((uint32_t)(Dh / 16)), batch_idx, token_idx, rows, k_out,
        v_out, per);
  };
  auto by_row = [&](auto e) { per_row % 64 ? go(e, std::false_type{}) : go(e, std::true_type{}); };
  if (dtype == OUDJAT_BF16) by_row(ElemBf16{});
  else by_row(ElemFp16{});
  return check_launch(what);
}
