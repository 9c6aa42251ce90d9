// The MXFP4 format on the device: E2M1 packing, block scales, the scale tiles
// and the loads of 16-bit activations that the MXFP4 kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/mxfp4.h"

namespace w8a8 {
namespace mx {

enum DType { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

constexpr int kBlock = 32;          // values per scale
constexpr int kTileBytes = 512;     // one scale tile: 128 rows x 4 blocks
constexpr int kNanScale = 255;

// Scale tiles per 128 rows: K is padded to a multiple of 256 values (two
// tiles), the k block of the GEMMs.
__host__ __device__ constexpr int64_t k_tiles(int64_t K) { return 2 * ((K + 255) / 256); }
__host__ __device__ constexpr int64_t row_tiles(int64_t rows) { return (rows + 127) / 128; }

// Byte offset of (row, first block of k tile `kt`) in the scale tiles.
__device__ __forceinline__ int64_t scale_offset(int64_t row, int64_t kt, int64_t ktiles) {
  const int r = static_cast<int>(row & 127);
  return ((row >> 7) * ktiles + kt) * kTileBytes + (r & 31) * 16 + (r >> 5) * 4;
}

// E8M0 byte of a block from the bit pattern of its largest magnitude (compared
// as unsigned integers, which orders NaN above infinity above every number):
// floor(log2 amax) - 2 is the fp32 exponent field less 2, since E2M1's largest
// binade is [4, 8).  Magnitudes below 2^-125 (subnormals among them) get the
// smallest scale, infinities and NaN the NaN scale.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23);
  return e == 255 ? kNanScale : max(e - 2, 0);
}

// 2^(127 - byte), the exact factor that brings a block into E2M1's range; 0
// for the NaN scale (its codes are zero).  byte <= 252 for finite blocks, so
// the exponent field 254 - byte is that of a normal number.
__device__ __forceinline__ float inv_scale(int byte) {
  return byte == kNanScale ? 0.0f : __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// max(|a|, |b|, |c|) and max(|a|, |b|), NaN if one is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ float max2_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// Eight values as four pairs, the operands of the packed fp32 instructions.
struct Vec8 {
  float2 p[4];
};

__device__ __forceinline__ float amax8(const Vec8& v) {
  const float a = max3_abs(v.p[0].x, v.p[0].y, v.p[1].x);
  const float b = max3_abs(v.p[1].y, v.p[2].x, v.p[2].y);
  return max3_abs(max3_abs(v.p[3].x, v.p[3].y, a), b, b);
}

// v * f to eight E2M1 codes (nearest, ties to even, saturating), value j in
// bits [4j, 4j + 4).
__device__ __forceinline__ uint32_t pack8_scaled(const Vec8& v, float f) {
  const float2 ff = make_float2(f, f);
  float2 t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = __fmul2_rn(v.p[j], ff);
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(t[0].x), "f"(t[0].y), "f"(t[1].x), "f"(t[1].y), "f"(t[2].x), "f"(t[2].y), "f"(t[3].x), "f"(t[3].y));
  return w;
}

// ---- computed values (fp32, relative error below `d`): their scale and codes,
// from both ends of that error's interval.
// The scale of a block whose largest magnitude is m; false where the ends differ
// or it is the NaN scale.
__device__ __forceinline__ bool scale_fast(float m, float d, int& byte) {
  const uint32_t l = abs_bits(m * (1.0f - d)), h = abs_bits(m * (1.0f + d));
  byte = scale_byte(l);
  return ((l ^ h) >> 23) == 0 && byte != kNanScale;
}

// Codes of eight values; the result has a bit set in each code whose ends differ.
__device__ __forceinline__ uint32_t codes_fast(const Vec8& y, int byte, float d, uint32_t& w) {
  const float f = inv_scale(byte);
  w = pack8_scaled(y, f * (1.0f - d));
  return w ^ pack8_scaled(y, f * (1.0f + d));
}

// ---- 64-bit forms, for the values next to a border
// E2M1 code of t (already divided by the block's scale).
__device__ inline uint32_t code_of(double t) {
  const double a = fabs(t);
  // the nearest code: borders between neighbours, an even code wins its tie
  uint32_t c = 0;
  c += a > 0.25;
  c += a >= 0.75;
  c += a > 1.25;
  c += a >= 1.75;
  c += a > 2.5;
  c += a >= 3.5;
  c += a > 5.0;
  return c | (signbit(t) ? 8u : 0u);
}

// E8M0 byte from the exact largest magnitude of a block.
__device__ inline int scale_byte(double amax) {
  if (!(amax <= 3.4028234663852886e38)) return kNanScale;
  const int e = static_cast<int>(__double2hiint(amax) >> 20) - 1023;  // floor(log2 amax); -1023 for 0
  return max(e - 2 + 127, 0);
}

// ---- 16-bit activations
template <typename T>
__device__ __forceinline__ Vec8 unpack8(const uint4& raw);

template <>
__device__ __forceinline__ Vec8 unpack8<__nv_bfloat16>(const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  Vec8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.p[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  return v;
}

template <>
__device__ __forceinline__ Vec8 unpack8<__half>(const uint4& raw) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
  Vec8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.p[j] = __half22float2(h[j]);
  return v;
}

// Largest magnitude of eight 16-bit values, as a pair still to be joined (NaN
// if one is): four-lane reductions work on the pair.
template <typename T>
struct Pair16;
template <>
struct Pair16<__nv_bfloat16> {
  using V = __nv_bfloat162;
};
template <>
struct Pair16<__half> {
  using V = __half2;
};

template <typename T>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  using V = typename Pair16<T>::V;
  const V m = __hmax2_nan(reinterpret_cast<const V&>(a), reinterpret_cast<const V&>(b));
  return reinterpret_cast<const uint32_t&>(m);
}

template <typename T>
__device__ __forceinline__ uint32_t amax8_pair(const uint4& raw) {
  constexpr uint32_t k = 0x7fff7fffu;
  return max_pair<T>(max_pair<T>(raw.x & k, raw.y & k), max_pair<T>(raw.z & k, raw.w & k));
}

// fp32 bits of the larger of a pair of magnitudes.
template <typename T>
__device__ __forceinline__ uint32_t pair_bits(uint32_t m);
template <>
__device__ __forceinline__ uint32_t pair_bits<__nv_bfloat16>(uint32_t m) {
  return max(m << 16, m & 0xffff0000u);
}
template <>
__device__ __forceinline__ uint32_t pair_bits<__half>(uint32_t m) {
  const float2 f = __half22float2(reinterpret_cast<const __half2&>(m));
  return max(__float_as_uint(f.x), __float_as_uint(f.y)) & 0x7fffffffu;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);

template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}

template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

// silu(g) * u in fp32 on the ex2 and rcp units, as (g u) / (1 + exp(-g)).  For
// g in [-40, inf) the relative error is below 2^-18 = 3.8e-6: the argument
// t = -g log2(e), below 58, is off by its own rounding (2^-19) and by the
// constant's (40 x 2e-8), 2.7e-6 together, which is 1.9e-6 relative in 2^t;
// ex2 adds 2^-22, the sum, rcp and two products about 2^-22 together.  (g u
// taken first keeps subnormal gates exact where a large up lifts them; where it
// overflows although the quotient would not, the result is not finite.)
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 silu_mul_fast(float2 g, float2 u) {
  constexpr float c = -1.4426950408889634f;
  const float2 t = __fmul2_rn(g, make_float2(c, c));
  const float2 d = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.0f, 1.0f));
  return __fmul2_rn(__fmul2_rn(g, u), make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}

constexpr float kSiluDelta = 3.814697265625e-6f;  // 2^-18

// The same with the rounding of t and of the constant put back, 2^t (1 + ln 2
// lo): what is left is ex2's 2^-22, rcp's 2^-23, three additions and products'
// 2^-24 each and that of the factor with which the result is packed, 6.6e-7
// together for g in [-40, inf): below 2^-20 = 9.5e-7.  (In results below 2^-126
// fp32's spacing adds up to 2^-149; the smallest border is 2^-129.)
__device__ __forceinline__ float2 silu_mul_close(float2 g, float2 u) {
  constexpr float c = -1.44269502162933349609375f, cl = -1.925962991e-8f, ln2 = 0.693147180559945f;
  const float2 cc = make_float2(c, c);
  const float2 t = __fmul2_rn(g, cc);
  float2 lo = __ffma2_rn(g, cc, make_float2(-t.x, -t.y));
  lo = __fmul2_rn(__ffma2_rn(g, make_float2(cl, cl), lo), make_float2(ln2, ln2));
  float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
  e = __ffma2_rn(e, lo, e);
  const float2 d = __fadd2_rn(e, make_float2(1.0f, 1.0f));
  return __fmul2_rn(__fmul2_rn(g, u), make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}
constexpr float kSiluCloseDelta = 9.5367431640625e-7f;  // 2^-20

// The same for g < -40, where the sigmoid is 2^-t (1 + 2^-t is 1 to 2^-57) and
// neither 2^t nor its reciprocal need fit fp32 although the product with a large u
// does: four factors 2^(-t/4), u first, so that no partial product is larger than
// u or smaller than the result.  Their 2^-22 each and the products' 2^-24 stay
// below 2^-18.  (Below -1000 the result is zero for every u.)
__device__ __forceinline__ float silu_mul_far(float g, float u) {
  constexpr float c = 1.44269502162933349609375f, cl = 1.925962991e-8f, ln2 = 0.693147180559945f;
  const float x = fmaxf(g, -1000.0f);
  const float t = x * c, lo = fmaf(x, cl, fmaf(x, c, -t)) * ln2;
  const float h = ex2_approx(0.25f * t);
  const float y = u * h * g * h * h * h;
  return fmaf(y, lo, y);
}
constexpr float kSiluFar = -40.0f;

// silu(g) * u in 64 bits.
__device__ inline double silu_mul_exact(float g, float u) {
  const double x = g;
  return x / (1.0 + exp(-x)) * static_cast<double>(u);
}

// Pairs of fp32 numbers hi + lo, about 2^-46 relative.
__device__ __forceinline__ float2 pair_sum(float a, float b) {  // exact
  const float s = a + b, t = s - a;
  return make_float2(s, (a - (s - t)) + (b - t));
}
__device__ __forceinline__ float2 pair_mul(float2 a, float2 b) {
  const float h = a.x * b.x;
  return make_float2(h, fmaf(a.x, b.x, -h) + fmaf(a.x, b.y, a.y * b.x));
}
__device__ __forceinline__ float2 pair_add(float2 c, float2 a) {  // |c.x| >= |a.x|
  const float s = c.x + a.x;
  return make_float2(s, (a.x - (s - c.x)) + (a.y + c.y));
}

// exp(-g) as 2^n times a pair (exp(80) for g beyond 80): e^z, with z / 8 in a
// Taylor polynomial and that squared three times.  Relative errors add up to 2^-41
// (2^-40 for g = -185, by the argument).
__device__ __forceinline__ float2 exp_neg(float g, int& n) {
  constexpr float c = 1.44269502162933349609375f, cl = 1.925962991e-8f;  // log2(e)
  constexpr float k = 0.0866433978080749512f, kl = -2.380817875e-10f;    // ln(2) / 8
  constexpr float sixth = 0.16666667163372039795f, sixth_l = -4.967053731e-9f;
  const float x = fmaxf(-g, -80.0f);
  const float t = x * c, r = rintf(t);
  n = static_cast<int>(r);
  const float2 z = pair_mul(pair_sum(t - r, fmaf(x, cl, fmaf(x, c, -t))), make_float2(k, kl));
  float2 e = make_float2(fmaf(z.x, fmaf(z.x, fmaf(z.x, 1.0f / 5040.0f, 1.0f / 720.0f), 1.0f / 120.0f), 1.0f / 24.0f), 0.0f);
  e = pair_add(make_float2(sixth, sixth_l), pair_mul(z, e));
  e = pair_add(make_float2(0.5f, 0.0f), pair_mul(z, e));
  e = pair_add(make_float2(1.0f, 0.0f), pair_mul(z, e));
  e = pair_add(make_float2(1.0f, 0.0f), pair_mul(z, e));
#pragma unroll
  for (int i = 0; i < 3; ++i) e = pair_mul(e, e);
  return e;
}

// 2^n for n in [-126, 127].
__device__ __forceinline__ float power2(int n) { return __int_as_float((n + 127) << 23); }

// On which side of `border` |silu(g) u| / 2^scale lies (1 above, -1 below), for a
// value within 2^-16 of it; 0 where this does not tell (within 2^-38, or factors
// out of the range that it is made for): compares |g u| / 2^scale with border (1 +
// exp(-g)), below kSiluFar both over 2^n.  It takes no 64-bit instruction: while
// tcgen05.mma runs the first of those waits for some 5000 clocks (170 otherwise).
__device__ __forceinline__ int silu_mul_side(float g, float u, int scale, float border) {
  const float ag = fabsf(g);
  if (!(ag > 8.67361738e-19f && g > -185.0f && g < 1.15292150e18f)) return 0;  // 2^-60, 2^60
  int n;
  float2 d = exp_neg(g, n);
  int up = -scale;
  if (g < kSiluFar) {
    up -= n;
  } else {
    const float s = power2(n);  // n is in [-116, 58]
    const float2 sum = pair_sum(1.0f, d.x * s);
    d = make_float2(sum.x, fmaf(d.y, s, sum.y));
  }
  if (up < -250) return 0;
  const float au = fabsf(u) * power2(up >> 1) * power2(up - (up >> 1));
  if (!(au > 8.67361738e-19f && au < 3.402823466e38f)) return 0;
  const float p = ag * au, pl = fmaf(ag, au, -p);
  const float diff = fmaf(-border, d.x, p) + fmaf(-border, d.y, pl);  // (the first is exact)
  return fabsf(diff) <= p * 3.6379788e-12f ? 0 : diff > 0.0f ? 1 : -1;  // 2^-38
}

// Border between the E2M1 magnitudes c and c + 1.
__device__ __forceinline__ float border_above(uint32_t c) {
  return c < 4 ? 0.25f + 0.5f * static_cast<float>(c) : c == 4 ? 2.5f : c == 5 ? 3.5f : 5.0f;
}

}  // namespace mx
}  // namespace w8a8
