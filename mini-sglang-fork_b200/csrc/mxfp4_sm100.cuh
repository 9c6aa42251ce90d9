// MXFP4 GEMM on the block-scaled tensor-core path (tcgen05.mma kind::mxf4):
// inline PTX of the instructions, and the weight-stationary kernel.
//
// D[m, n] = sum over 32-value blocks c of sA[m, c] sB[n, c] (A_c . B_c): the
// instruction multiplies 64 E2M1 values per row (two blocks), scales the two
// block products by the rows' E8M0 scales and accumulates in fp32 in TMEM.
// Operands come from shared memory in the 128-byte-swizzled K-major layout
// (a row of 256 codes is 128 bytes, one k block of the pipeline); scales come
// from TMEM, where tcgen05.cp puts them: a 512-byte tile of 128 rows x 4
// blocks becomes 4 columns, row r in lane r % 32 of column r / 32, copied to
// all four lane quarters.  The scale tiles in memory have that order already,
// so a stage's scales are plain 1024-byte copies (two tiles per row group).
#pragma once

#include "common.cuh"
#include "mxfp4.cuh"
#include "sm100.cuh"

#include <cuda.h>

namespace w8a8 {
namespace mx {

// Descriptor of a 512-byte scale tile for tcgen05.cp.32x128b: no swizzle, 8
// rows of 16 bytes per core matrix, core matrices 128 bytes apart.
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}

// Instruction descriptor of kind::mxf4 block32: A and B E2M1 (bits 7-9 and
// 10-12 = 1), both K-major, N >> 3 in bits 17-22, E8M0 scales (bit 23), M >> 4
// in bits 24-28, scale ids (the byte of the 4-block word to start from: 0 or
// 2) of B in bits 4-5 and of A in bits 29-30.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24) | (static_cast<uint32_t>(sf) << 29);
}

__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// One lane of a converged warp.  The producer and MMA roles run their loops
// with the whole warp and issue under this predicate, from which the compiler
// knows that one lane is active.  Under a predicate on the lane index, which
// leaves that open, a k block of four MMAs and six scale copies took 606 ns to
// issue; with this 280 ns, which is the MMAs' own time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// mbar_wait by a whole warp: true for all lanes or for none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned int* err, long long tmo) {
  return __all_sync(0xffffffffu, dev::mbar_wait(bar, parity, abort_flag, err, kErrGemmWait, tmo));
}

struct MxGemmArgs {
  const void* bias;  // [N] of the output type, or null
  void* out;         // C [M, N]
  uint8_t* q;        // SiLU: codes [M, I / 2]
  uint8_t* qs;       // SiLU: scale tiles of [M, I]
  unsigned int* err;
  long long timeout_ns;
  int M, N, K;       // N: output columns (I with the SiLU epilogue: B has N gate
                     // rows and N up rows, each half with scale tiles of its own)
  int kblocks;       // 256-value k blocks
  int tiles;         // weight-stationary kernel: 128-column tiles of the output
};

// Copies `bytes` (a multiple of 16) of this CTA's shared memory into another
// CTA's, counted on that CTA's mbarrier (`dst` and `bar` are cluster addresses
// of the same CTA).
__device__ __forceinline__ void dsmem_copy(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "r"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// Makes this thread's writes to its shared memory visible to bulk copies.
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Asks for a tile to be brought into L2; reads nothing, so it may run ahead of
// the kernel that is still writing other memory (or even that tile: L2 is
// where both meet).
__device__ __forceinline__ void tma_prefetch_2d(const void* tmap, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(x), "r"(y)
               : "memory");
}

// Eight output values from column `col` (a multiple of 8) of a row.
template <typename O>
__device__ __forceinline__ void store8_row(const MxGemmArgs& g, int64_t row, int col, const uint4& w) {
  if (row >= g.M || col >= g.N) return;
  O* dst = static_cast<O*>(g.out) + row * g.N + col;
  if ((g.N & 7) == 0) {
    *reinterpret_cast<uint4*>(dst) = w;
  } else {  // rows that are not 16-byte aligned
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col + k < g.N) reinterpret_cast<uint16_t*>(dst)[k] = static_cast<uint16_t>(x[k >> 1] >> (16 * (k & 1)));
  }
}

// Bias of eight columns from `col` (a multiple of 8), zero beyond column N: one
// load where the pointer allows it.
template <typename O>
__device__ __forceinline__ Vec8 bias8(const void* bias, int col, int N) {
  const O* b = static_cast<const O*>(bias) + col;
  if ((reinterpret_cast<uintptr_t>(bias) & 15u) == 0 && col + 8 <= N) return unpack8<O>(__ldg(reinterpret_cast<const uint4*>(b)));
  Vec8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v.p[e] = make_float2(col + 2 * e < N ? to_float(b[2 * e]) : 0.0f, col + 2 * e + 1 < N ? to_float(b[2 * e + 1]) : 0.0f);
  return v;
}

// A block of gated products that fp32 does not settle: its gates and ups in,
// codes and scale out.
struct GatedBlock {
  float g[32], u[32];
  uint32_t w[4];
  int byte;
};

// All of it in 64 bits, by the one lane that has the block, out of line.
static __device__ __noinline__ void gated_block_exact(GatedBlock& b) {
  double m = 0.0;
#pragma unroll 1
  for (int e = 0; e < 32; ++e) {
    const double a = fabs(silu_mul_exact(b.g[e], b.u[e]));
    m = (a > m || isnan(a)) ? a : m;
  }
  b.byte = scale_byte(m);
  b.w[0] = b.w[1] = b.w[2] = b.w[3] = 0;
  if (b.byte == kNanScale) return;
  const double f = ldexp(1.0, 127 - b.byte);
#pragma unroll 1
  for (int e = 0; e < 32; ++e) b.w[e >> 3] |= code_of(silu_mul_exact(b.g[e], b.u[e]) * f) << (4 * (e & 7));
}

// Value `at` of 32 that are in registers, by selections (an index, or a reference
// to one of the words, would put them all in local memory).
__device__ __forceinline__ float pick32(const Vec8 (&v)[4], int at) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = at & 1 ? v[i].p[0].y : v[i].p[0].x, b = at & 1 ? v[i].p[1].y : v[i].p[1].x;
    const float c = at & 1 ? v[i].p[2].y : v[i].p[2].x, d = at & 1 ? v[i].p[3].y : v[i].p[3].x;
    const float ab = at & 2 ? b : a, cd = at & 2 ? d : c;
    x[i] = at & 4 ? cd : ab;
  }
  const float lo = at & 8 ? x[1] : x[0], hi = at & 8 ? x[3] : x[2];
  return at & 16 ? hi : lo;
}

// silu(gate) * up of 32 features (block `j` of 128-feature tile `ft`) of one
// output row, as one MXFP4 block: the quantisation of the exact product of the
// fp32 sums (plus biases), by the border check of the quantisers.  A block in
// 10^4 has a value within the check's 2^-20 of a border; silu_mul_side places it,
// and what that leaves open the block's 64-bit form.  (12288 x 4096: 19.7 us for
// 256 tokens and 290 for 8192, where one conversion without a check took 18.5 and
// 280, gave the neighbouring code once in 4 10^7 and zeros for gates below -87;
// with the second look in 64 bits, beside the running MMAs, 21 to 22 and 300.)
// `bias`: the tile's 128 gate and 128 up biases in shared memory.
__device__ __forceinline__ void silu_block(const MxGemmArgs& g, const float* bias, const float (&gate)[32],
                                           const float (&up)[32], int64_t row, int ft, int j) {
  const int f0 = ft * 128 + 32 * j;
  Vec8 gv[4], uv[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      gv[i].p[e] = make_float2(gate[8 * i + 2 * e], gate[8 * i + 2 * e + 1]);
      uv[i].p[e] = make_float2(up[8 * i + 2 * e], up[8 * i + 2 * e + 1]);
    }
    if (g.bias) {
      const float2* bg = reinterpret_cast<const float2*>(bias + 32 * j + 8 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gv[i].p[e] = __fadd2_rn(gv[i].p[e], bg[e]);
        uv[i].p[e] = __fadd2_rn(uv[i].p[e], bg[64 + e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[i].p[e] = silu_mul_close(gv[i].p[e], uv[i].p[e]);
  }
  if (row >= g.M || f0 >= g.N) return;
  float least_gate = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) least_gate = fminf(least_gate, fminf(gv[i].p[e].x, gv[i].p[e].y));
  const bool far = least_gate < kSiluFar;
  if (far) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (gv[i].p[e].x < kSiluFar) y[i].p[e].x = silu_mul_far(gv[i].p[e].x, uv[i].p[e].x);
        if (gv[i].p[e].y < kSiluFar) y[i].p[e].y = silu_mul_far(gv[i].p[e].y, uv[i].p[e].y);
      }
  }
  const float m = max3_abs(max3_abs(amax8(y[0]), amax8(y[1]), amax8(y[2])), amax8(y[3]), 0.0f);
  const bool tiny = m < 1e-36f;  // results near the end of fp32's range
  const float d = far || tiny ? kSiluDelta : kSiluCloseDelta;
  int byte;
  uint32_t w[4] = {0, 0, 0, 0}, left = 0;  // left: bit e is value e's, to be looked at again
  const auto encode = [&] {
    uint32_t open[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) open[i] = codes_fast(y[i], byte, d, w[i]);
    if (open[0] | open[1] | open[2] | open[3]) {
#pragma unroll
      for (int e = 0; e < 32; ++e) left |= (open[e >> 3] >> (4 * (e & 7)) & 15u) ? 1u << e : 0u;
    }
  };
  bool scale_open = !scale_fast(m, d, byte);
  bool settled = byte < 252 && !tiny;  // (else only the 64-bit form may look again)
  if (!scale_open) {
    settled = true;
    encode();
  } else if (settled) {  // the values that may be the largest, then the codes under the scale found
    const float least = m * (1.0f - 4.0f * d);
#pragma unroll
    for (int e = 0; e < 32; ++e)
      left |= fabsf(e & 1 ? y[e >> 3].p[e >> 1 & 3].y : y[e >> 3].p[e >> 1 & 3].x) >= least ? 1u << e : 0u;
  }
  bool above = false;
#pragma unroll 1
  while (left && settled) {
    const int at = __ffs(left) - 1, nib = 4 * (at & 7);
    left &= left - 1;
    const uint32_t code = at < 8 ? w[0] : at < 16 ? w[1] : at < 24 ? w[2] : w[3];
    const float border = scale_open ? 8.0f : border_above(code >> nib & 7u);
    const int side = silu_mul_side(pick32(gv, at), pick32(uv, at), byte - 127, border);
    settled = side != 0 && !tiny;
    if (scale_open) {
      above |= side > 0;
      if (left == 0) {
        scale_open = false;
        byte += above;
        encode();
      }
    } else if (side > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += at >> 3 == i ? 1u << nib : 0u;
    }
  }
  if (!settled) {
    // a gate or an up that is not finite makes a product that is not either: no
    // need to look at that one in 64 bits
    const float worst = max3_abs(max3_abs(amax8(gv[0]), amax8(gv[1]), amax8(gv[2])), max3_abs(amax8(gv[3]), amax8(uv[0]), amax8(uv[1])),
                                 max3_abs(amax8(uv[2]), amax8(uv[3]), 0.0f));
    if (worst <= 3.402823466e38f) {
      GatedBlock b;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          *reinterpret_cast<float2*>(b.g + 8 * i + 2 * e) = gv[i].p[e];
          *reinterpret_cast<float2*>(b.u + 8 * i + 2 * e) = uv[i].p[e];
        }
      gated_block_exact(b);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = b.w[i];
      byte = b.byte;
    } else {
      w[0] = w[1] = w[2] = w[3] = 0;
      byte = kNanScale;
    }
  }
  const int64_t kt = k_tiles(g.N);
  *reinterpret_cast<uint4*>(g.q + row * (g.N >> 1) + (f0 >> 1)) = make_uint4(w[0], w[1], w[2], w[3]);
  uint8_t* s = g.qs + scale_offset(row, ft, kt);
  s[j] = static_cast<uint8_t>(byte);
  if (f0 + 32 == g.N)  // the last block also writes the padding to 256 features
    for (int b = f0 / 32 + 1; b & 7; ++b) s[(b / 4 - ft) * kTileBytes + (b & 3)] = 0;
}

// ------------------------------------------------- weight-stationary kernel
// For up to T (16 to 128) tokens, all of them in every tile.  One CTA computes 128
// output columns (weight rows, on the MMA's 128-row side); with the SiLU epilogue
// 128 gate rows and the 128 up rows that belong to them, in two accumulators.
// The weights are read once, at the rate of HBM, which is what bounds it; the
// ring (about 200 KB of an SM's shared memory, in one CTA or in several) is
// there to keep enough of them in flight.
//
// Up to 32 tokens, two CTAs share an SM, so that one starts (its weights asked
// for in L2) while the other ends; three with more tiles than SMs (51200 x
// 5120, one token: 23.2 us; one persistent CTA per SM with the same ring:
// 24.5).  With few tiles a cluster of S CTAs splits K (5120 x 25600, one token:
// 14.0 us with six shares, two CTAs per SM; 15.0 with three shares, one per SM;
// 29.6 without): CTA r writes an S-th of the tokens, and every CTA
// sends it its fp32 sums of those by a bulk copy between shared memories, the
// fast way there (gate_up 1536 x 4096, 64 tokens, eight shares: 11.5 us; 22.5
// with loads from the peers' memory, 32.8 with stores to it).  r adds them up
// in the order of the shares, so the result does not depend on timing, and
// nothing is left in memory between calls.
template <int T, bool SILU, bool DEEP>
struct MxRowTraits {
  static constexpr int kTiles = SILU ? 2 : 1;  // weight tiles (gate, up)
  static constexpr int kW = 128 * 128;         // bytes of a weight tile's k block
  static constexpr int kX = T * 128;
  static constexpr int kSf = 1024;             // scale bytes of 128 rows per k block
  static constexpr int kStageBytes = kTiles * (kW + kSf) + kX + kSf;
  static constexpr int kSfCols = 8 * (kTiles + 1);  // TMEM columns of a stage's scales
  static constexpr int kStages = SILU   ? (T == 16 ? 5 : 4)
                                 : DEEP ? (T <= 32 ? 5 : T == 64 ? 8 : 6)
                                        : (T <= 32 ? 3 : 4);
  static constexpr int kChunk = T < 32 ? T : 32;  // columns that the epilogue takes at a time
  static constexpr int kAccCols = kTiles * T;
  // CTAs that take tile after tile have two accumulators where TMEM allows
  static constexpr bool kPersistent = SILU || T == 128;
  static constexpr int kAccs = kPersistent && 2 * kAccCols + kStages * kSfCols <= 512 ? 2 : 1;
  static constexpr int kColsNeeded = kAccs * kAccCols + kStages * kSfCols;
  static constexpr int kTmemCols = kColsNeeded <= 64 ? 64 : kColsNeeded <= 128 ? 128 : kColsNeeded <= 256 ? 256 : 512;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kStagingBytes = SILU ? 4 * 2 * kChunk * 128 : 0;  // per epilogue warp: gate, up
  static constexpr int kBiasBytes = SILU ? 2 * 1024 : 0;                 // per accumulator: gate, up
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBarrierBytes + kStagingBytes + kBiasBytes;
  static_assert(kColsNeeded <= 512, "TMEM");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static constexpr int kPerSm = 228 * 1024 / (kSmemBytes + 1024);  // CTAs on an SM
  // At most three CTAs with at most 128 TMEM columns each share an SM, and one
  // with more leaves no room for another (nor does an int8 GEMM, whose ring
  // alone is 180 KB or more).  So every allocation succeeds at once, and no CTA
  // of a cluster waits for TMEM that a CTA waiting for it holds.
  static_assert(kTmemCols <= 128 ? kSmemBytes >= 60 * 1024 : kSmemBytes >= 170 * 1024, "TMEM share");
  // The ring holds a CTA's own shares for its peers and theirs for it.
  static_assert(!DEEP || 2 * kTiles * (T + 8) * 512 <= kStages * kStageBytes, "the shares reuse the ring");
};

constexpr int kRowThreads = 192;  // producer, MMA, four epilogue warps

template <int CH>
__device__ __forceinline__ void tmem_ld_chunk(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  dev::tmem_ld<CH>(taddr, r);
  dev::tmem_wait_ld(r);
#pragma unroll
  for (int j = 0; j < CH; ++j) v[j] = __uint_as_float(r[j]);
}

template <typename O, int T, bool SILU, bool DEEP>
__global__ void __launch_bounds__(kRowThreads, 1) mx_row_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                                const __grid_constant__ CUtensorMap tm_ws,
                                                                const __grid_constant__ CUtensorMap tm_x,
                                                                const __grid_constant__ CUtensorMap tm_xs,
                                                                const MxGemmArgs args) {
  using P = MxRowTraits<T, SILU, DEEP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // [stage] weight tiles, [stage] tokens, then the scales
  uint8_t* s_w = smem;
  uint8_t* s_x = s_w + P::kStages * P::kTiles * P::kW;
  uint8_t* s_ws = s_x + P::kStages * P::kX;
  uint8_t* s_xs = s_ws + P::kStages * P::kTiles * P::kSf;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_xs + P::kStages * P::kSf);
  uint64_t* full = bars;
  uint64_t* empty = bars + P::kStages;
  uint64_t* acc_full = bars + 2 * P::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;          // [2]
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint64_t* arrived = drain + 1;  // S > 1: the peers' shares
  float* bias_s = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + P::kBarrierBytes + P::kStagingBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = static_cast<int>(cluster_size());
  const int rank = static_cast<int>(dev::cluster_rank());
  const int first = blockIdx.x / S;
  const int step = gridDim.x / S;  // (S > 1: one tile per cluster)
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * args.kblocks / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * args.kblocks / S);
  const int tokens = args.M;  // at most T
  const long long tmo = args.timeout_ns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P::kStages; ++s) {
      dev::mbar_init(dev::smem_u32(full + s), 1);
      dev::mbar_init(dev::smem_u32(empty + s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      dev::mbar_init(dev::smem_u32(acc_full + s), 1);
      dev::mbar_init(dev::smem_u32(acc_empty + s), 4);  // the epilogue warps
    }
    dev::mbar_init(dev::smem_u32(drain), 1);
    dev::mbar_init(dev::smem_u32(arrived), 1);
    *abort_flag = 0;
    dev::fence_mbar_init();
    dev::prefetch_tmap(&tm_w);
    dev::prefetch_tmap(&tm_ws);
    dev::prefetch_tmap(&tm_x);
    dev::prefetch_tmap(&tm_xs);
  }
  if (warp == 1) {
    dev::tmem_alloc(dev::smem_u32(tmem_slot), P::kTmemCols);
    dev::tmem_relinquish();
  }
  dev::griddep_launch();
  if (warp == 0) {
    // the first weights into L2 while the previous kernel ends (five k blocks:
    // 51200 x 5120, one token, 22.0 us against 23.2 without; twenty cost 27)
    if (elect_one()) {
      for (int kb = kb0; kb < min(kb1, kb0 + 5); ++kb)
#pragma unroll
        for (int h = 0; h < P::kTiles; ++h) {
          tma_prefetch_2d(&tm_w, kb * 128, first * 128 + h * args.N);
          tma_prefetch_2d(&tm_ws, kb * 256, first + h * args.tiles);
        }
    }
    __syncwarp();
  }
  dev::tc_fence_before();
  __syncthreads();
  dev::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);  // (the same in every lane, and known to be)
  dev::griddep_wait();  // any operand may be the previous kernel's output

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < args.tiles; tile += step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = warp_wait(dev::smem_u32(empty + stage), phase ^ 1u, abort_flag, args.err, tmo);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t bar = dev::smem_u32(full + stage);
          dev::mbar_expect_tx(bar, P::kStageBytes);
#pragma unroll
          for (int h = 0; h < P::kTiles; ++h) {
            // gate rows, then up rows
            dev::tma_load_2d(dev::smem_u32(s_w + (stage * P::kTiles + h) * P::kW), &tm_w, bar, kb * 128,
                             tile * 128 + h * args.N);
            dev::tma_load_2d(dev::smem_u32(s_ws + (stage * P::kTiles + h) * P::kSf), &tm_ws, bar, kb * 256,
                             tile + h * args.tiles);
          }
          dev::tma_load_2d(dev::smem_u32(s_x + stage * P::kX), &tm_x, bar, kb * 128, 0);
          dev::tma_load_2d(dev::smem_u32(s_xs + stage * P::kSf), &tm_xs, bar, kb * 256, 0);
        }
        __syncwarp();
        issued_mask |= 1u << stage;
        issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == P::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (lane == 0)
      for (int s = 0; s < P::kStages; ++s)  // no copy in flight when the CTA ends
        if (issued_mask & (1u << s))
          if (!dev::mbar_wait_drain(dev::smem_u32(full + s), (issued_phase >> s) & 1u, tmo))
            if (args.err) atomicOr(args.err, kErrGemmDrain);
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    int stage = 0;
    uint32_t phase = 0, i = 0;
    bool ok = true;
    for (int tile = first; ok && tile < args.tiles; tile += step, ++i) {
      const uint32_t acc = i % P::kAccs, use = i / P::kAccs;
      if (!warp_wait(dev::smem_u32(acc_empty + acc), (use & 1u) ^ 1u, abort_flag, args.err, tmo)) break;
      dev::tc_fence_after();
      const uint32_t d = tmem + acc * P::kAccCols;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = warp_wait(dev::smem_u32(full + stage), phase, abort_flag, args.err, tmo);
        if (!ok) break;
        dev::tc_fence_after();
        if (elect_one()) {
          // each stage has its own scale columns: free again once the MMAs that
          // read them have arrived on `empty`
          const uint32_t sf = tmem + P::kAccs * P::kAccCols + stage * P::kSfCols;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            cp_scales(sf + 4 * c, sdesc_scales(dev::smem_u32(s_xs + stage * P::kSf + c * kTileBytes)));
#pragma unroll
            for (int h = 0; h < P::kTiles; ++h)
              cp_scales(sf + 8 * (h + 1) + 4 * c,
                        sdesc_scales(dev::smem_u32(s_ws + (stage * P::kTiles + h) * P::kSf + c * kTileBytes)));
          }
          const uint64_t dx = dev::sdesc_k_sw128(dev::smem_u32(s_x + stage * P::kX));
          const int steps = min(4, (args.K - kb * 256 + 63) / 64);  // beyond K: nothing to add
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= steps) break;
            constexpr uint32_t ids[2] = {idesc_mxf4(128, T, 0), idesc_mxf4(128, T, 2)};
#pragma unroll
            for (int h = 0; h < P::kTiles; ++h) {
              const uint64_t dw = dev::sdesc_k_sw128(dev::smem_u32(s_w + (stage * P::kTiles + h) * P::kW));
              mma_mxf4(d + h * T, dw + 2 * k, dx + 2 * k, ids[k & 1], sf + 8 * (h + 1) + 4 * (k >> 1),
                       sf + 4 * (k >> 1), (kb > kb0 || k > 0) ? 1u : 0u);
            }
          }
          dev::tc_commit(dev::smem_u32(empty + stage));
        }
        __syncwarp();
        if (++stage == P::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (elect_one()) dev::tc_commit(dev::smem_u32(acc_full + acc));
      __syncwarp();
    }
    if (elect_one()) dev::tc_commit(dev::smem_u32(drain));
    if (lane == 0 && !dev::mbar_wait_drain(dev::smem_u32(drain), 0, tmo))
      if (args.err) atomicOr(args.err, kErrGemmDrain);
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lane quarter of this warp: 32 of the tile's columns
    const int n = q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    float* stg = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + P::kBarrierBytes +
                                          q * (P::kStagingBytes / 4));
    uint32_t i = 0;
    for (int tile = first; tile < args.tiles; tile += step, ++i) {
      const uint32_t acc = i % P::kAccs, use = i / P::kAccs;
      // the biases before the wait for the sums
      const int col = tile * 128 + n;
      float* bias = bias_s + (i & 1u) * 256;
      float bias_n = 0.0f;
      if (args.bias) {
        const O* b = static_cast<const O*>(args.bias);
        if constexpr (SILU) {
          bias[n] = col < args.N ? to_float(b[col]) : 0.0f;
          bias[128 + n] = col < args.N ? to_float(b[args.N + col]) : 0.0f;
        } else if (col < args.N) {
          bias_n = to_float(b[col]);
        }
      }
      // (a failed wait leaves the result unspecified; the error word says so)
      const bool ok = warp_wait(dev::smem_u32(acc_full + acc), use & 1u, abort_flag, args.err, tmo);
      if (SILU && args.bias ? dev::named_bar_or(1, 128, !ok) : !ok) break;  // (publishes the biases)
      dev::tc_fence_after();
      const uint32_t t_acc = tmem + lanes + acc * P::kAccCols;
      if (S > 1) break;  // one tile, finished below
      if constexpr (!SILU) {
        const bool in = col < args.N;
        O* out = static_cast<O*>(args.out) + col;
        for (int c = 0; c < tokens; c += P::kChunk) {
          float v[32];
          tmem_ld_chunk<P::kChunk>(t_acc + c, v);
#pragma unroll
          for (int j = 0; j < P::kChunk; ++j)
            if (c + j < tokens && in) {
              const uint32_t p = pack2<O>(v[j] + bias_n, 0.0f);
              *reinterpret_cast<uint16_t*>(out + static_cast<int64_t>(c + j) * args.N) = static_cast<uint16_t>(p);
            }
        }
      } else {
        // a warp's 32 features are one block of the result: 32 tokens at a
        // time are transposed through shared memory, then a lane has a block
        for (int c = 0; c < tokens; c += P::kChunk) {
          float g[32], u[32];
          tmem_ld_chunk<P::kChunk>(t_acc + c, g);
          tmem_ld_chunk<P::kChunk>(t_acc + T + c, u);
#pragma unroll
          for (int j = 0; j < P::kChunk; ++j) {
            const int w = j * 32 + ((((lane >> 2) ^ (j & 7)) << 2) | (lane & 3));
            stg[w] = g[j];
            stg[P::kChunk * 32 + w] = u[j];
          }
          __syncwarp();
          if (lane < P::kChunk && c + lane < tokens) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int w = lane * 32 + ((e ^ (lane & 7)) << 2);
              *reinterpret_cast<float4*>(g + 4 * e) = *reinterpret_cast<const float4*>(stg + w);
              *reinterpret_cast<float4*>(u + 4 * e) = *reinterpret_cast<const float4*>(stg + P::kChunk * 32 + w);
            }
            silu_block(args, bias, g, u, c + lane, tile, q);
          }
          __syncwarp();
        }
      }
      dev::tc_fence_before();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_u32(acc_empty + acc));
    }
    dev::tc_fence_before();
  }
  if (DEEP && S > 1) {
    const auto begin = [&](int s) { return tokens * s / S; };  // tokens [begin(s), begin(s + 1)) are s's
    const int t0 = begin(rank), count = begin(rank + 1) - t0;
    // in the ring: [token][gate / up][128] sums of this CTA, then from each
    // share (in rank order, its own place left empty) the same of its tokens
    constexpr int kTokenWords = P::kTiles * 128;
    float* own = reinterpret_cast<float*>(smem);
    float* in = own + T * kTokenWords;
    if (threadIdx.x == 64 && count > 0) dev::mbar_expect_tx(dev::smem_u32(arrived), (S - 1) * count * kTokenWords * 4);
    dev::cluster_sync();  // every CTA's MMAs are done: its ring may be written
    if (warp >= 2) {
      const int q = warp & 3, n = q * 32 + lane;
      const uint32_t t_acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
      const int et = threadIdx.x - 64;
      dev::tc_fence_after();
      for (int c = 0; c < tokens; c += P::kChunk)
#pragma unroll
        for (int h = 0; h < P::kTiles; ++h) {
          float v[32];
          tmem_ld_chunk<P::kChunk>(t_acc + h * T + c, v);
#pragma unroll
          for (int j = 0; j < P::kChunk; ++j)
            own[(c + j) * kTokenWords + h * 128 + ((((n >> 2) ^ ((c + j) & 7)) << 2) | (n & 3))] = v[j];
        }
      dev::tc_fence_before();
      fence_async_smem();
      dev::named_bar_sync(1, 128);
      if (et < S && et != rank) {
        const int to = begin(et), many = begin(et + 1) - to;
        if (many > 0)
          dsmem_copy(dev::mapa(dev::smem_u32(in) + static_cast<uint32_t>(rank * many * kTokenWords) * 4, et),
                     dev::smem_u32(own + to * kTokenWords), static_cast<uint32_t>(many * kTokenWords) * 4,
                     dev::mapa(dev::smem_u32(arrived), et));
      }
      __syncwarp();
      if (count > 0) warp_wait(dev::smem_u32(arrived), 0, abort_flag, args.err, tmo);
      // 16 bytes of the s-th share of token t (of this CTA's), word w
      const auto piece = [&](int s, int t, int w) {
        const float* p = s == rank ? own + t * kTokenWords : in + (s * count + t - t0) * kTokenWords;
        return *reinterpret_cast<const float4*>(p + (w & ~127) + ((((w & 127) >> 2) ^ (t & 7)) << 2));
      };
      if constexpr (!SILU) {
        // an item: 8 columns of a token
        for (int it = et; it < count * 16; it += 128) {
          const int t = t0 + (it >> 4), n0 = (it & 15) * 8;
          float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          for (int s = 0; s < S; ++s) {
            const float4 x = piece(s, t, n0), y = piece(s, t, n0 + 4);
            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
            v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
          }
          const int col = first * 128 + n0;
          if (args.bias) {
            const Vec8 b = bias8<O>(args.bias, col, args.N);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[2 * j] += b.p[j].x, v[2 * j + 1] += b.p[j].y;
          }
          store8_row<O>(args, t, col,
                        make_uint4(pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3]), pack2<O>(v[4], v[5]), pack2<O>(v[6], v[7])));
        }
      } else {
        // an item: one 32-feature block of a token
        for (int it = et; it < count * 4; it += 128) {
          const int t = t0 + (it >> 2), j = it & 3;
          float g[32], u[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) g[e] = u[e] = 0.0f;
          for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 x = piece(s, t, 32 * j + 4 * e), y = piece(s, t, 128 + 32 * j + 4 * e);
              g[4 * e] += x.x, g[4 * e + 1] += x.y, g[4 * e + 2] += x.z, g[4 * e + 3] += x.w;
              u[4 * e] += y.x, u[4 * e + 1] += y.y, u[4 * e + 2] += y.z, u[4 * e + 3] += y.w;
            }
          }
          silu_block(args, bias_s, g, u, t, first, j);
        }
      }
      __syncwarp();  // (the cluster barrier wants converged warps)
    }
    dev::cluster_sync();  // the copies out of this CTA have been taken
  }
  __syncthreads();
  if (warp == 1) {
    dev::tc_fence_after();
    dev::tmem_dealloc(tmem, P::kTmemCols);
  }
}

}  // namespace mx
}  // namespace w8a8
