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

// Eight values to eight E2M1 codes (nearest, ties to even, saturating), value
// j in bits [4j, 4j + 4).
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}

__device__ __forceinline__ uint32_t pack8_scaled(const float (&v)[8], float f) {
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = v[j] * f;
  return pack8(t);
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
__device__ __forceinline__ void unpack8(const uint4& raw, float (&f)[8]);

template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(w[j] << 16);
    f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}

template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& raw, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = __half22float2(h[j]);
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
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

// silu(g) * u in fp32 on the ex2 and rcp units.  For g in [-40, inf) the
// relative error is below 2^-18: the argument -g log2(e) carries at most
// 58 (2^-24 + 2^-25.9) absolute error, i.e. 3e-6 relative in exp, ex2 and rcp
// about 2^-22 each, and three roundings.  Below that see the callers.
__device__ __forceinline__ float silu_mul_fast(float g, float u) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
  return g * s * u;
}

}  // namespace mx
}  // namespace w8a8
