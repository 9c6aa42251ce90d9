// MXFP4 quantisers of the linear path's activations: plain, fused with
// SiLU*mul, fused with residual add + RMSNorm; and the inverse.
//
// Thread mapping, shared by the three: a lane holds 8 consecutive values (one
// 16-byte load), so four lanes share a block of 32 and a warp covers 256
// values of a row, which is exactly two scale tiles of that row.  The block's
// largest magnitude takes two shuffles; the 8 codes of a lane are one 4-byte
// store (128 contiguous bytes per warp); lanes 0 and 16 collect their tile's
// four scale bytes and store them as one word.  Lanes beyond the row's end
// hold zeros, whose scale byte is 0, so the padding blocks of the last tiles
// come out as the format asks without a case of their own.
//
// The plain quantiser is exact: the scale is a power of two, so x / s has no
// rounding and the only rounding is E2M1's own.  The fused ones quantise a
// computed y, for which they first work in fp32 with a relative error below
// `d`: if y (1 - d) and y (1 + d) round to the same code and the block's
// largest magnitude has the same exponent at both ends, that code and scale
// are those of the exact value.  Where they differ (of the order of one value in 10^5, the interval's width)
// the block is evaluated again in 64 bits, out of line.  Two conversions
// instead of one per value, and the result does not depend on how exp or the
// row's sum were evaluated.
#include "common.cuh"
#include "mxfp4.cuh"
#include "sm100.cuh"

namespace w8a8 {
namespace mx {
namespace {

constexpr int kThreads = 256;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery): the row of
// a warp's task; a 64-bit division would be a quarter of the instructions that
// a warp spends on its values.
struct Divisor {
  uint32_t d, mul, shift;
  explicit Divisor(uint32_t d_) : d(d_) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    shift = l;
    mul = static_cast<uint32_t>((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return (__umulhi(n, mul) + n) >> shift;  // n < 2^31: the sum does not wrap
  }
};

// A warp's share: VPT groups of 256 values from group g0 of a row.
struct Task {
  int64_t row;
  int g0;
  __device__ __forceinline__ Task(const Divisor& segs, int vpt) {
    const uint32_t t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const uint32_t r = segs.quotient(t);
    row = r;
    g0 = static_cast<int>(t - r * segs.d) * vpt;
  }
};

// A lane's place in the scale tiles for 256-value group 0 of a row: the word of
// its k tile (lanes 0-15 the even one, 16-31 the odd one).  Group g is 1024
// bytes further on.
__device__ __forceinline__ int64_t scale_word(int64_t row, int64_t ktiles, int lane) {
  return scale_offset(row, lane >> 4, ktiles);
}

// Stores a warp's scale bytes (one per block, in every lane of the block) of a
// group whose words start at `word`.
__device__ __forceinline__ void store_scales(uint8_t* word, int lane, int byte) {
  uint32_t w = static_cast<uint32_t>(byte);
  w |= __shfl_down_sync(0xffffffffu, w, 4) << 8;
  w |= __shfl_down_sync(0xffffffffu, w, 8) << 16;
  if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(word) = w;
}

// Largest magnitude over the four lanes of a block, NaN if one is.
__device__ __forceinline__ float quad_max(float v) {
  v = max2_nan(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return max2_nan(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// ------------------------------------------------------------------- plain
// A warp takes VPT consecutive groups of 256 values of one row.
template <typename T, int VPT>
__global__ void __launch_bounds__(kThreads) quant_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ data,
                                                         uint8_t* __restrict__ scales, int64_t M, int K, Divisor segs) {
  const int lane = threadIdx.x & 31;
  const Task t(segs, VPT);
  const int nvec = K >> 3;
  const int64_t kt = k_tiles(K);
  dev::griddep_launch();
  dev::griddep_wait();
  if (t.row >= M) return;
  const int v0 = t.g0 * 32 + lane;
  const uint4* xr = reinterpret_cast<const uint4*>(x + t.row * ldx) + v0;
  uint32_t* qr = reinterpret_cast<uint32_t*>(data + t.row * (K >> 1)) + v0;
  uint8_t* sw = scales + scale_word(t.row, kt, lane) + static_cast<int64_t>(t.g0) * 1024;
  uint4 raw[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) raw[j] = v0 + 32 * j < nvec ? __ldcs(xr + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if ((t.g0 + j) * 32 >= nvec) break;  // the whole warp is beyond the row
    uint32_t m = amax8_pair<T>(raw[j]);
    m = max_pair<T>(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_pair<T>(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int byte = scale_byte(pair_bits<T>(m));
    const uint32_t w = byte == kNanScale ? 0u : pack8_scaled(unpack8<T>(raw[j]), inv_scale(byte));
    if (v0 + 32 * j < nvec) qr[32 * j] = w;
    store_scales(sw + 1024 * j, lane, byte);
  }
}

// The quantisation of a computed block: codes and scale byte of a lane's eight
// values `y` (fp32, relative error below `d`; m: the largest magnitude over the
// block's four lanes).  False where that error could change either: then
// block_exact gives them.  (scale_fast and codes_fast spelled out: called from
// here they cost the SiLU kernel, which is held to 48 registers, two more spills.)
__device__ __forceinline__ bool block_fast(const Vec8& y, float m, float d, uint32_t& w, int& byte) {
  const uint32_t l = abs_bits(m * (1.0f - d)), h = abs_bits(m * (1.0f + d));
  byte = scale_byte(l);
  const float f = inv_scale(byte);
  w = pack8_scaled(y, f * (1.0f - d));
  const uint32_t hi = pack8_scaled(y, f * (1.0f + d));
  return ((l ^ h) >> 23) == 0 && byte != kNanScale && w == hi;
}

// The same from eight exact values; all four lanes of the block come here.
template <typename Value>
__device__ __forceinline__ uint2 block_exact(int lane, Value value) {
  double v[8], m = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = value(j);
    const double a = fabs(v[j]);
    m = (a > m || isnan(a)) ? a : m;
  }
  const uint32_t quad = 15u << (lane & 28);
#pragma unroll
  for (int o = 1; o <= 2; o *= 2) {
    const double other = __shfl_xor_sync(quad, m, o);
    m = (other > m || isnan(other)) ? other : m;
  }
  const int byte = scale_byte(m);
  uint32_t w = 0;
  if (byte != kNanScale) {
    const double f = ldexp(1.0, 127 - byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= code_of(v[j] * f) << (4 * j);
  }
  return make_uint2(w, static_cast<uint32_t>(byte));
}

// Whether one of the four lanes of this lane's block says so.
__device__ __forceinline__ bool quad_any(bool x, int lane) {
  return (__ballot_sync(0xffffffffu, x) >> (lane & 28)) & 15u;
}

template <typename T>
__device__ inline float element(const uint4& raw, int j) {
  return to_float(reinterpret_cast<const T*>(&raw)[j]);
}

// -------------------------------------------------------------- SiLU * mul
template <typename T>
__device__ __noinline__ uint2 silu_exact(uint4 graw, uint4 uraw, int lane) {
  return block_exact(lane, [&](int j) { return silu_mul_exact(element<T>(graw, j), element<T>(uraw, j)); });
}

// Smallest of eight gates.  Below -40 the fast form's argument error grows (and
// its reciprocal flushes further down); those blocks are taken in 64 bits, as are
// blocks with a NaN.  (4096 x 12288: 45.6 us without any; with a gate at -50 in 1,
// 10 and 100 % of the blocks of each row 57, 159 and 217 us, with a NaN 67, 124 and
// 192.)
template <typename T>
__device__ __forceinline__ float min8(const uint4& raw);

template <>
__device__ __forceinline__ float min8<__nv_bfloat16>(const uint4& raw) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
  const __nv_bfloat162 m = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
  return fminf(__low2float(m), __high2float(m));
}

template <>
__device__ __forceinline__ float min8<__half>(const uint4& raw) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
  const __half2 m = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
  return fminf(__low2float(m), __high2float(m));
}

template <typename T, int VPT>
__global__ void __launch_bounds__(kThreads, 5) silu_kernel(const T* __restrict__ gate_up, int64_t ld,
                                                           uint8_t* __restrict__ data, uint8_t* __restrict__ scales,
                                                           int64_t M, int I, Divisor segs) {
  const int lane = threadIdx.x & 31;
  const Task t(segs, VPT);
  const int nvec = I >> 3;
  const int64_t kt = k_tiles(I);
  dev::griddep_launch();
  dev::griddep_wait();
  if (t.row >= M) return;
  const int v0 = t.g0 * 32 + lane;
  const uint4* gr = reinterpret_cast<const uint4*>(gate_up + t.row * ld) + v0;
  const uint4* ur = gr + nvec;
  uint4 graw[VPT], uraw[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const bool in = v0 + 32 * j < nvec;
    graw[j] = in ? __ldcs(gr + 32 * j) : make_uint4(0, 0, 0, 0);
    uraw[j] = in ? __ldcs(ur + 32 * j) : make_uint4(0, 0, 0, 0);
  }
  uint32_t w[VPT];
  int byte[VPT];
  uint32_t open = 0;  // bit j: vector j's block is to be taken in 64 bits
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const Vec8 g = unpack8<T>(graw[j]), u = unpack8<T>(uraw[j]);
    Vec8 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.p[e] = silu_mul_fast(g.p[e], u.p[e]);
    const bool ok = block_fast(y, quad_max(amax8(y)), kSiluDelta, w[j], byte[j]);
    if (!ok || min8<T>(graw[j]) < -40.0f) open |= 1u << j;
  }
  if (__any_sync(0xffffffffu, open != 0)) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (quad_any(open >> j & 1u, lane)) {
        const uint2 r = silu_exact<T>(graw[j], uraw[j], lane);
        w[j] = r.x;
        byte[j] = static_cast<int>(r.y);
      }
  }
  uint32_t* qr = reinterpret_cast<uint32_t*>(data + t.row * (I >> 1)) + v0;
  uint8_t* sw = scales + scale_word(t.row, kt, lane) + static_cast<int64_t>(t.g0) * 1024;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if ((t.g0 + j) * 32 >= nvec) break;  // the whole warp is beyond the row
    if (v0 + 32 * j < nvec) qr[32 * j] = w[j];
    store_scales(sw + 1024 * j, lane, byte[j]);
  }
}

// ----------------------------------------------------------------- RMSNorm
// One CTA per row, thread t holding vectors t + blockDim * j of v = x +
// residual in fp32.  The sum of squares is taken in 64 bits, where a square is
// exact: blocks next to a border need it so (with fp32 sums of four squares one
// value in 3 10^8 got the neighbouring code), and it takes no time, as the
// 64-bit unit and the conversions run beside the rest (4097 x 5120, when
// changed: 29.4 us, 29.3 with the fp32 sums).  y = v (r w) in fp32: errors of r
// (2.5e-7) and of the two products stay below 2^-20.  r w may leave fp32's
// range.  Above, y is not finite, and its block is taken in 64 bits.  Below, it
// is off by 2^-150, and y by that times |v| <= sqrt(K) rms: less than 2^-45 of
// the block's first border (m / 32 or more) as long as the block's largest
// magnitude m is at least 2^-92 rms; a block of less, in a row that is not all
// zeros, is taken in 64 bits too.  That includes blocks whose values or weights are
// all zero (padded or pruned channels), whose codes need no such look: 4097 x 5120
// takes 30 us without any, 35, 59 and 77 us with 1, 10 and 50 % of the weight's
// blocks zero, 104 us with 10 % of x and residual.
constexpr float kNormDelta = 9.5367431640625e-7f;  // 2^-20

struct NormRow {
  double ss;  // sum of v^2 over the row
  int K;
  float eps;
};

template <typename T>
__device__ __noinline__ uint2 norm_exact(Vec8 v, uint4 wr, NormRow n, int lane) {
  const double root = sqrt(n.ss / n.K + static_cast<double>(n.eps));
  return block_exact(lane, [&](int j) {
    return static_cast<double>(j & 1 ? v.p[j >> 1].y : v.p[j >> 1].x) / root * static_cast<double>(element<T>(wr, j));
  });
}

// Sum over the CTA, in every thread and in an order that does not vary.
__device__ __forceinline__ double block_sum(double x, double* part, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (warps == 1) return x;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.0;
  for (int i = 0; i < warps; ++i) x += part[i];
  return x;
}

template <typename T, int VPT, int MAX_THREADS, int MIN_CTAS, bool ADD>
__global__ void __launch_bounds__(MAX_THREADS, MIN_CTAS)
    rmsnorm_kernel(const T* x, int64_t ldx, T* residual, int64_t ldr, const T* __restrict__ weight,
                   float eps, uint8_t* __restrict__ data, uint8_t* __restrict__ scales, int K) {
  __shared__ double part[MAX_THREADS / 32];
  const int lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  const int nvec = K >> 3;
  const int64_t kt = k_tiles(K);
  dev::griddep_launch();
  dev::griddep_wait();
  const int64_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * ldx);
  uint4* rr = ADD ? reinterpret_cast<uint4*>(residual + row * ldr) : nullptr;
  const uint4* wr = reinterpret_cast<const uint4*>(weight);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  Vec8 v[VPT];
  uint4 wa[VPT];
  {
    uint4 xa[VPT], ra[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vi = threadIdx.x + j * blockDim.x;
      xa[j] = vi < nvec ? __ldcs(xr + vi) : zero;
      if (ADD) ra[j] = vi < nvec ? __ldcs(rr + vi) : zero;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vi = threadIdx.x + j * blockDim.x;
      wa[j] = vi < nvec ? __ldg(wr + vi) : zero;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vi = threadIdx.x + j * blockDim.x;
      v[j] = unpack8<T>(xa[j]);
      if constexpr (ADD) {
        const Vec8 r = unpack8<T>(ra[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j].p[e] = __fadd2_rn(v[j].p[e], r.p[e]);
        if (vi < nvec)
          rr[vi] = make_uint4(pack2<T>(v[j].p[0].x, v[j].p[0].y), pack2<T>(v[j].p[1].x, v[j].p[1].y),
                              pack2<T>(v[j].p[2].x, v[j].p[2].y), pack2<T>(v[j].p[3].x, v[j].p[3].y));
      }
    }
  }
  double s0 = 0.0, s1 = 0.0;  // two chains
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double a = v[j].p[e].x, b = v[j].p[e].y;
      s0 = fma(a, a, s0);
      s1 = fma(b, b, s1);
    }
  const double ss = block_sum(s0 + s1, part, warps);
  const double mean = ss * (1.0 / K) + static_cast<double>(eps);
  // A row with an infinity or a NaN needs no second look: r is 0 or NaN, and y
  // zero or NaN as it is by the definition.
  const bool finite = ss < __longlong_as_double(0x7ff0000000000000LL);
  // rows whose mean square is beyond the fp32 form: all in 64 bits
  const bool far = finite && !(mean > 1e-25 && mean < 1e25);
  const NormRow n = {ss, K, eps};
  const float root = sqrtf(static_cast<float>(mean));
  const float r = 1.0f / root;
  const float limit = finite && ss > 0.0 ? root * 2.0194839173657902e-28f : 0.0f;  // 2^-92 rms
  const float2 r2 = make_float2(r, r);
  uint8_t* sw = scales + scale_word(row, kt, lane);
  uint32_t* qr = reinterpret_cast<uint32_t*>(data + row * (K >> 1));
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int base = (threadIdx.x & ~31) + j * blockDim.x;
    if (base >= nvec) break;
    const int vi = base + lane;
    const Vec8 w = unpack8<T>(wa[j]);
    Vec8 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.p[e] = __fmul2_rn(v[j].p[e], __fmul2_rn(w.p[e], r2));
    uint32_t code;
    int byte;
    // (a lane beyond the row may hold 0 times an infinite r: no value of the block)
    const float m = quad_max(vi < nvec ? amax8(y) : 0.0f);
    bool ok = block_fast(y, m, kNormDelta, code, byte) && m >= limit;
    if (!finite) {
      ok = true;
      if (byte == kNanScale) code = 0;
    }
    if (quad_any(far || (!ok && vi < nvec), lane)) {
      const uint2 e = norm_exact<T>(v[j], wa[j], n, lane);
      code = e.x;
      byte = vi < nvec ? static_cast<int>(e.y) : 0;
    }
    if (vi < nvec) qr[vi] = code;
    store_scales(sw + base * 32, lane, byte);
  }
}

// ----------------------------------------------------------------- inverse
template <typename O>
__device__ __forceinline__ void store8(O* out, const Vec8& v) {
  if constexpr (sizeof(O) == 4) {
    reinterpret_cast<float4*>(out)[0] = make_float4(v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y);
    reinterpret_cast<float4*>(out)[1] = make_float4(v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y);
  } else {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<O>(v.p[0].x, v.p[0].y), pack2<O>(v.p[1].x, v.p[1].y),
                                                pack2<O>(v.p[2].x, v.p[2].y), pack2<O>(v.p[3].x, v.p[3].y));
  }
}

template <typename O, int VPT>
__global__ void __launch_bounds__(kThreads) dequant_kernel(const uint8_t* __restrict__ data,
                                                           const uint8_t* __restrict__ scales, O* __restrict__ out,
                                                           int64_t M, int K, Divisor segs) {
  const int lane = threadIdx.x & 31;
  const Task t(segs, VPT);
  const int nvec = K >> 3;
  const int64_t kt = k_tiles(K);
  dev::griddep_launch();
  dev::griddep_wait();
  if (t.row >= M) return;
  const int v0 = t.g0 * 32 + lane;
  const uint32_t* qr = reinterpret_cast<const uint32_t*>(data + t.row * (K >> 1)) + v0;
  const uint8_t* sr = scales + scale_word(t.row, kt, lane) + ((lane >> 2) & 3) + static_cast<int64_t>(t.g0) * 1024;
  O* dst = out + t.row * K + static_cast<int64_t>(v0) * 8;
  uint32_t w[VPT], s[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const bool in = v0 + 32 * j < nvec;
    w[j] = in ? __ldcs(qr + 32 * j) : 0u;
    s[j] = in ? sr[1024 * j] : 0u;
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (v0 + 32 * j >= nvec) break;
    // 2^(s - 127): a subnormal for s = 0, NaN for s = 255
    const float f = s[j] == kNanScale ? __uint_as_float(0x7fffffffu)
                    : s[j] == 0       ? __uint_as_float(0x00400000u)
                                      : __uint_as_float(s[j] << 23);
    Vec8 v;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint32_t h;
      asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}"
          : "=r"(h)
          : "r"((w[j] >> (8 * b)) & 255u));
      v.p[b] = __fmul2_rn(__half22float2(reinterpret_cast<const __half2&>(h)), make_float2(f, f));
    }
    store8(dst + 256 * j, v);
  }
}

// -------------------------------------------------------------------- host
int check_shape(const char* what, int64_t M, int64_t K) {
  W8A8_REQUIRE(M >= 0 && K >= 0, W8A8_ERR_INVALID_ARG, "%s: negative shape", what);
  W8A8_REQUIRE(K > 0 && K % kBlock == 0, W8A8_ERR_INVALID_ARG, "%s: the last dimension (%lld) must be a positive multiple of 32",
               what, (long long)K);
  W8A8_REQUIRE(K <= (1LL << 30) && M <= (1LL << 30), W8A8_ERR_UNSUPPORTED, "%s: shape too large", what);
  return W8A8_OK;
}

int check_device(const char* what) {
  W8A8_REQUIRE(device_cc_major() == 10, W8A8_ERR_UNSUPPORTED,
               "%s: the kernels need an sm_100 (B200) device; found compute capability %d.x", what, device_cc_major());
  return W8A8_OK;
}

// Groups of 256 values per warp: 4 (64 bytes in flight per lane) once that
// still gives every SM 16 warps, else 1.
int pick_vpt(int64_t M, int64_t K) {
  const int64_t groups = M * ((K + 255) / 256);
  return groups >= 4 * 16 * static_cast<int64_t>(sm_count()) ? 4 : 1;
}

int grid_of(const char* what, int64_t M, int64_t K, int vpt, uint32_t* segs, unsigned* grid) {
  const int64_t groups = (K + 255) / 256;
  *segs = static_cast<uint32_t>((groups + vpt - 1) / vpt);
  const int64_t ctas = (M * *segs + kThreads / 32 - 1) / (kThreads / 32);
  // (Divisor and Task count a launch's warps in 31 bits)
  W8A8_REQUIRE(ctas < (1LL << 31) / (kThreads / 32), W8A8_ERR_UNSUPPORTED, "%s: %lld x %lld is too large for one launch",
               what, (long long)M, (long long)K);
  *grid = static_cast<unsigned>(ctas);
  return W8A8_OK;
}

template <typename T>
int run_quant(const void* x, int64_t ldx, uint8_t* data, uint8_t* scales, int64_t M, int64_t K, cudaStream_t s) {
  const int vpt = pick_vpt(M, K);
  uint32_t segs;
  unsigned grid;
  if (int rc = grid_of("mxfp4_quant", M, K, vpt, &segs, &grid)) return rc;
  auto kern = vpt == 4 ? quant_kernel<T, 4> : quant_kernel<T, 1>;
  W8A8_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(kThreads), 0, s, static_cast<const T*>(x), ldx, data, scales, M,
                           static_cast<int>(K), Divisor(segs)));
  return W8A8_OK;
}

template <typename T>
int run_silu(const void* gu, int64_t ld, uint8_t* data, uint8_t* scales, int64_t M, int64_t I, cudaStream_t s) {
  // (4096 x 12288 fp16: 41.9 us with two groups per warp and five CTAs per SM;
  // 43.0 with four and three, 53.4 with one)
  const int vpt = pick_vpt(M, I) == 4 ? 2 : 1;
  uint32_t segs;
  unsigned grid;
  if (int rc = grid_of("mxfp4_silu_mul_quant", M, I, vpt, &segs, &grid)) return rc;
  auto kern = vpt == 2 ? silu_kernel<T, 2> : silu_kernel<T, 1>;
  W8A8_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(kThreads), 0, s, static_cast<const T*>(gu), ld, data, scales, M,
                           static_cast<int>(I), Divisor(segs)));
  return W8A8_OK;
}

// Threads and vectors per thread of a row: with few rows one vector per thread
// (the shortest chain), with many four, so that a CTA is small and an SM holds
// rows at different stages (4097 x 5120, when chosen: 32.8 us; with two 34.8,
// with one 69.6).  The kernel asks for 98 registers; held to 80 and 64, so that
// 768 to 1024 threads fit an SM, some are spilled but more rows are under way
// (4097 x 5120: 28.1 us, 29.4 unbound; 4096 x 8192: 43.4, 52.4; 2048 x 16384:
// 47.8, 59.7).
template <typename T, bool ADD>
int run_norm(const void* x, int64_t ldx, void* residual, int64_t ldr, const void* weight, float eps, uint8_t* data,
             uint8_t* scales, int64_t M, int64_t K, cudaStream_t s) {
  const int nvec = static_cast<int>(K / 8);
  const int vpt = M >= 2 * sm_count() || nvec > 2048 ? 4 : nvec > 1024 ? 2 : 1;
  const int threads = ((nvec + vpt - 1) / vpt + 31) / 32 * 32;
#define MXFP4_NORM(V, THREADS, CTAS)                                                                              \
  W8A8_CUDA_TRY(launch_pdl(rmsnorm_kernel<T, V, THREADS, CTAS, ADD>, dim3(static_cast<unsigned>(M)), dim3(threads), \
                           0, s, static_cast<const T*>(x), ldx, static_cast<T*>(residual), ldr,                   \
                           static_cast<const T*>(weight), eps, data, scales, static_cast<int>(K)))
  if (vpt == 1) MXFP4_NORM(1, 1024, 1);
  else if (vpt == 2) MXFP4_NORM(2, 1024, 1);
  else if (threads <= 160) MXFP4_NORM(4, 160, 5);
  else if (threads <= 256) MXFP4_NORM(4, 256, 3);
  else if (threads <= 512) MXFP4_NORM(4, 512, 2);
  else MXFP4_NORM(4, 1024, 1);
#undef MXFP4_NORM
  return W8A8_OK;
}

template <typename O>
int run_dequant(const uint8_t* data, const uint8_t* scales, void* out, int64_t M, int64_t K, cudaStream_t s) {
  const int vpt = pick_vpt(M, K);
  uint32_t segs;
  unsigned grid;
  if (int rc = grid_of("mxfp4_dequant", M, K, vpt, &segs, &grid)) return rc;
  auto kern = vpt == 4 ? dequant_kernel<O, 4> : dequant_kernel<O, 1>;
  W8A8_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(kThreads), 0, s, data, scales, static_cast<O*>(out), M,
                           static_cast<int>(K), Divisor(segs)));
  return W8A8_OK;
}

}  // namespace
}  // namespace mx
}  // namespace w8a8

extern "C" {

int64_t mxfp4_scale_bytes(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || K % w8a8::mx::kBlock) return 0;
  return w8a8::mx::row_tiles(rows) * w8a8::mx::k_tiles(K) * w8a8::mx::kTileBytes;
}

int mxfp4_quant(const void* x, int64_t ldx, int dtype, uint8_t* data, uint8_t* scales, int64_t M, int64_t K,
                void* stream) {
  using namespace w8a8;
  if (M == 0) return W8A8_OK;
  if (int rc = mx::check_shape("mxfp4_quant", M, K)) return rc;
  W8A8_REQUIRE(x && data && scales, W8A8_ERR_INVALID_ARG, "mxfp4_quant: null pointer");
  W8A8_REQUIRE(dtype == mx::kBf16 || dtype == mx::kFp16, W8A8_ERR_INVALID_ARG, "mxfp4_quant: bf16 or fp16 input");
  W8A8_REQUIRE(ldx >= K && ldx % 8 == 0, W8A8_ERR_INVALID_ARG, "mxfp4_quant: the row stride must be a multiple of 8, at least K");
  W8A8_REQUIRE(W8A8_ALIGNED16(x) && W8A8_ALIGNED16(data) && W8A8_ALIGNED16(scales), W8A8_ERR_ALIGNMENT,
               "mxfp4_quant: pointers must be 16-byte aligned");
  if (int rc = mx::check_device("mxfp4_quant")) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return dtype == mx::kBf16 ? mx::run_quant<__nv_bfloat16>(x, ldx, data, scales, M, K, s)
                            : mx::run_quant<__half>(x, ldx, data, scales, M, K, s);
}

int mxfp4_dequant(const uint8_t* data, const uint8_t* scales, void* out, int dtype, int64_t M, int64_t K,
                  void* stream) {
  using namespace w8a8;
  if (M == 0) return W8A8_OK;
  if (int rc = mx::check_shape("mxfp4_dequant", M, K)) return rc;
  W8A8_REQUIRE(data && scales && out, W8A8_ERR_INVALID_ARG, "mxfp4_dequant: null pointer");
  W8A8_REQUIRE(dtype >= mx::kBf16 && dtype <= mx::kFp32, W8A8_ERR_INVALID_ARG, "mxfp4_dequant: bf16, fp16 or fp32 output");
  W8A8_REQUIRE(W8A8_ALIGNED16(data) && W8A8_ALIGNED16(scales) && W8A8_ALIGNED16(out), W8A8_ERR_ALIGNMENT,
               "mxfp4_dequant: pointers must be 16-byte aligned");
  if (int rc = mx::check_device("mxfp4_dequant")) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case mx::kBf16: return mx::run_dequant<__nv_bfloat16>(data, scales, out, M, K, s);
    case mx::kFp16: return mx::run_dequant<__half>(data, scales, out, M, K, s);
    default: return mx::run_dequant<float>(data, scales, out, M, K, s);
  }
}

int mxfp4_silu_mul_quant(const void* gate_up, int64_t ld, int dtype, uint8_t* data, uint8_t* scales, int64_t M,
                         int64_t I, void* stream) {
  using namespace w8a8;
  if (M == 0) return W8A8_OK;
  if (int rc = mx::check_shape("mxfp4_silu_mul_quant", M, I)) return rc;
  W8A8_REQUIRE(gate_up && data && scales, W8A8_ERR_INVALID_ARG, "mxfp4_silu_mul_quant: null pointer");
  W8A8_REQUIRE(dtype == mx::kBf16 || dtype == mx::kFp16, W8A8_ERR_INVALID_ARG,
               "mxfp4_silu_mul_quant: bf16 or fp16 input");
  W8A8_REQUIRE(ld >= 2 * I && ld % 8 == 0, W8A8_ERR_INVALID_ARG,
               "mxfp4_silu_mul_quant: the row stride must be a multiple of 8, at least 2I");
  W8A8_REQUIRE(W8A8_ALIGNED16(gate_up) && W8A8_ALIGNED16(data) && W8A8_ALIGNED16(scales), W8A8_ERR_ALIGNMENT,
               "mxfp4_silu_mul_quant: pointers must be 16-byte aligned");
  if (int rc = mx::check_device("mxfp4_silu_mul_quant")) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return dtype == mx::kBf16 ? mx::run_silu<__nv_bfloat16>(gate_up, ld, data, scales, M, I, s)
                            : mx::run_silu<__half>(gate_up, ld, data, scales, M, I, s);
}

int mxfp4_rmsnorm_quant(const void* x, int64_t ldx, void* residual, int64_t ldr, const void* weight, float eps,
                        int dtype, uint8_t* data, uint8_t* scales, int64_t M, int64_t K, void* stream) {
  using namespace w8a8;
  if (M == 0) return W8A8_OK;
  if (int rc = mx::check_shape("mxfp4_rmsnorm_quant", M, K)) return rc;
  W8A8_REQUIRE(x && weight && data && scales, W8A8_ERR_INVALID_ARG, "mxfp4_rmsnorm_quant: null pointer");
  W8A8_REQUIRE(dtype == mx::kBf16 || dtype == mx::kFp16, W8A8_ERR_INVALID_ARG,
               "mxfp4_rmsnorm_quant: bf16 or fp16 input");
  W8A8_REQUIRE(K <= 32768, W8A8_ERR_UNSUPPORTED, "mxfp4_rmsnorm_quant: K=%lld is above 32768", (long long)K);
  W8A8_REQUIRE(ldx >= K && ldx % 8 == 0 && (!residual || (ldr >= K && ldr % 8 == 0)), W8A8_ERR_INVALID_ARG,
               "mxfp4_rmsnorm_quant: row strides must be multiples of 8, at least K");
  W8A8_REQUIRE(eps >= 0.0f && eps < 1e30f, W8A8_ERR_INVALID_ARG, "mxfp4_rmsnorm_quant: eps must be finite and not negative");
  W8A8_REQUIRE(W8A8_ALIGNED16(x) && W8A8_ALIGNED16(residual) && W8A8_ALIGNED16(weight) && W8A8_ALIGNED16(data) &&
                   W8A8_ALIGNED16(scales),
               W8A8_ERR_ALIGNMENT, "mxfp4_rmsnorm_quant: pointers must be 16-byte aligned");
  if (int rc = mx::check_device("mxfp4_rmsnorm_quant")) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == mx::kBf16)
    return residual ? mx::run_norm<__nv_bfloat16, true>(x, ldx, residual, ldr, weight, eps, data, scales, M, K, s)
                    : mx::run_norm<__nv_bfloat16, false>(x, ldx, residual, ldr, weight, eps, data, scales, M, K, s);
  return residual ? mx::run_norm<__half, true>(x, ldx, residual, ldr, weight, eps, data, scales, M, K, s)
                  : mx::run_norm<__half, false>(x, ldx, residual, ldr, weight, eps, data, scales, M, K, s);
}

}  // extern "C"
