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
// with the whole warp and issue under this predicate: the compiler then knows
// that one lane is active and passes the operands of TMA and tcgen05 (which
// the hardware takes from uniform registers) directly.  Under a predicate on
// the lane index it emits a loop over the lanes' values around every such
// instruction; a k block of four MMAs and six scale copies then took 606 ns to
// issue, with this 280 ns, which is the MMAs' own time.
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
  int M, N, K;       // N: output columns (I with the SiLU epilogue)
  int kblocks;       // 256-value k blocks
  int ttiles;        // token tiles of the weight-stationary kernel
};

// 16 columns of fp32 TMEM
__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
}

__device__ __forceinline__ float ld_dsmem(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// ------------------------------------------------- weight-stationary kernel
// One CTA computes 128 output columns (weight rows, on the MMA's 128-row side)
// for T tokens; with the SiLU epilogue 128 gate rows and the 128 up rows that
// belong to them, in two accumulators.  A cluster of S CTAs splits K: each
// leaves its fp32 partial sums in its own shared memory and, after a cluster
// barrier, CTA r adds the S shares of tokens r, r + S, ... in rank order
// through distributed shared memory and writes them, so the sum's order is
// fixed and nothing is left in memory between calls.
template <int T, bool SILU>
struct MxRowTraits {
  static constexpr int kTiles = SILU ? 2 : 1;  // weight tiles (gate, up)
  static constexpr int kW = 128 * 128;         // bytes of a weight tile's k block
  static constexpr int kX = T * 128;
  static constexpr int kSf = 1024;             // scale bytes of 128 rows per k block
  static constexpr int kStageBytes = kTiles * (kW + kSf) + kX + kSf;
  static constexpr int kSfCols = 8 * (kTiles + 1);  // TMEM columns of a stage's scales
  static constexpr int kStages = SILU ? (T <= 32 ? 3 : T == 64 ? 4 : 4) : (T <= 32 ? 3 : T == 64 ? 4 : 3);
  static constexpr int kAccCols = kTiles * T;
  static constexpr int kColsNeeded = kAccCols + kStages * kSfCols;
  static constexpr int kTmemCols = kColsNeeded <= 64 ? 64 : kColsNeeded <= 128 ? 128 : kColsNeeded <= 256 ? 256 : 512;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kUsedBytes = 1024 + kStages * kStageBytes + kBarrierBytes;
  // At least the share of the SM's 228 KB that the kernel takes of its 512 TMEM
  // columns (less the 1 KB that every CTA gets anyway): then whatever mix of
  // this library's CTAs an SM holds, their TMEM allocations fit together, and
  // no CTA of a cluster waits for columns that a CTA waiting for it holds.
  static constexpr int kShare = kTmemCols * 456 - 1024;
  static constexpr int kSmemBytes = kUsedBytes > kShare ? kUsedBytes : kShare;
  static_assert(kColsNeeded <= 512, "TMEM");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(kTiles * T * 128 * 4 <= kStages * kStageBytes, "the partial sums reuse the ring");
};

constexpr int kRowThreads = 192;  // producer, MMA, four epilogue warps

// One output value (or, SiLU, one block of 32 outputs over the warp) for
// output column `col` = this lane's, token `t` (uniform over the warp).
template <typename O, bool SILU>
__device__ __forceinline__ void emit(const MxGemmArgs& a, int t, int col, int lane, float g, float u, float bg,
                                     float bu) {
  if constexpr (!SILU) {
    if (col < a.N) {
      O* c = static_cast<O*>(a.out) + static_cast<int64_t>(t) * a.N + col;
      if constexpr (sizeof(O) == 2) {
        const uint32_t p = pack2<O>(g + bg, 0.0f);
        *reinterpret_cast<uint16_t*>(c) = static_cast<uint16_t>(p);
      }
    }
  } else {
    // the warp's 32 columns are one block of the result (I % 128 == 0)
    const float y = silu_mul_fast(g + bg, u + bu);
    const uint32_t m = __reduce_max_sync(0xffffffffu, abs_bits(y));
    const int byte = scale_byte(m);
    uint32_t w = byte == kNanScale ? 0u : code_of(y * inv_scale(byte)) << (4 * (lane & 7));
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    const int c0 = col - lane;
    if ((lane & 7) == 0)
      *reinterpret_cast<uint32_t*>(a.q + static_cast<int64_t>(t) * (a.N >> 1) + ((c0 + lane) >> 1)) = w;
    if (lane == 0) {
      const int64_t kt = k_tiles(a.N);
      uint8_t* s = a.qs + scale_offset(t, c0 >> 7, kt) + ((c0 >> 5) & 3);
      *s = static_cast<uint8_t>(byte);
      if ((c0 >> 7) + 1 == (a.N >> 7) && ((a.N >> 7) & 1)) s[kTileBytes] = 0;  // the padding tile
    }
  }
}

template <typename O, int T, bool SILU>
__global__ void __launch_bounds__(kRowThreads) mx_row_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                             const __grid_constant__ CUtensorMap tm_ws,
                                                             const __grid_constant__ CUtensorMap tm_x,
                                                             const __grid_constant__ CUtensorMap tm_xs,
                                                             const MxGemmArgs args) {
  using P = MxRowTraits<T, SILU>;
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
  uint64_t* acc_full = bars + 2 * P::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem);  // [tile][token][128], after the ring is done

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = static_cast<int>(cluster_size());
  const int rank = static_cast<int>(dev::cluster_rank());
  const int tile = blockIdx.x / S;
  const int tt = tile % args.ttiles;
  const int wt = tile / args.ttiles;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * args.kblocks / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * args.kblocks / S);
  const long long tmo = args.timeout_ns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P::kStages; ++s) {
      dev::mbar_init(dev::smem_u32(full + s), 1);
      dev::mbar_init(dev::smem_u32(empty + s), 1);
    }
    dev::mbar_init(dev::smem_u32(acc_full), 1);
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
  dev::tc_fence_before();
  __syncthreads();
  dev::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);  // (the same in every lane, and known to be)
  dev::griddep_launch();
  dev::griddep_wait();  // any operand may be the previous kernel's output

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(dev::smem_u32(empty + stage), phase ^ 1u, abort_flag, args.err, tmo)) break;
      if (elect_one()) {
        const uint32_t bar = dev::smem_u32(full + stage);
        dev::mbar_expect_tx(bar, P::kStageBytes);
#pragma unroll
        for (int h = 0; h < P::kTiles; ++h) {
          const int w0 = wt * 128 + h * args.N;  // gate rows, then up rows
          dev::tma_load_2d(dev::smem_u32(s_w + (stage * P::kTiles + h) * P::kW), &tm_w, bar, kb * 128, w0);
          dev::tma_load_2d(dev::smem_u32(s_ws + (stage * P::kTiles + h) * P::kSf), &tm_ws, bar, kb * 256, w0 >> 7);
        }
        dev::tma_load_2d(dev::smem_u32(s_x + stage * P::kX), &tm_x, bar, kb * 128, tt * T);
        dev::tma_load_2d(dev::smem_u32(s_xs + stage * P::kSf), &tm_xs, bar, kb * 256, (tt * T) >> 7);
      }
      __syncwarp();
      issued_mask |= 1u << stage;
      issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
      if (++stage == P::kStages) {
        stage = 0;
        phase ^= 1u;
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
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(dev::smem_u32(full + stage), phase, abort_flag, args.err, tmo)) break;
      dev::tc_fence_after();
      if (elect_one()) {
        // each stage has its own scale columns: free again once the MMAs that
        // read them have arrived on `empty`
        const uint32_t sf = tmem + P::kAccCols + stage * P::kSfCols;
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
            mma_mxf4(tmem + h * T, dw + 2 * k, dx + 2 * k, ids[k & 1], sf + 8 * (h + 1) + 4 * (k >> 1),
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
    if (elect_one()) dev::tc_commit(dev::smem_u32(acc_full));
    if (lane == 0 && !dev::mbar_wait_drain(dev::smem_u32(acc_full), 0, tmo))
      if (args.err) atomicOr(args.err, kErrGemmDrain);
  }
  __syncwarp();
  const int tokens = min(T, args.M - tt * T);
  const int q = warp & 3;  // TMEM lane quarter of this warp
  const int n = q * 32 + lane;
  const int col = wt * 128 + n;
  float bg = 0.0f, bu = 0.0f;
  if (warp >= 2) {
    if (args.bias && col < args.N) {
      bg = to_float(static_cast<const O*>(args.bias)[col]);
      if constexpr (SILU) bu = to_float(static_cast<const O*>(args.bias)[args.N + col]);
    }
    // (a failed wait leaves the result unspecified; the error word says so)
    dev::mbar_wait(dev::smem_u32(acc_full), 0, abort_flag, args.err, kErrGemmWait, tmo);
    dev::tc_fence_after();
    __syncwarp();
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    for (int c = 0; c < tokens; c += 16) {
      float g[16], u[16];
      tmem_ld16f(tmem + lanes + c, g);
      if constexpr (SILU) tmem_ld16f(tmem + lanes + T + c, u);
      if (S == 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < tokens) emit<O, SILU>(args, tt * T + c + j, col, lane, g[j], SILU ? u[j] : 0.0f, bg, bu);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          part[(c + j) * 128 + n] = g[j];
          if constexpr (SILU) part[(T + c + j) * 128 + n] = u[j];
        }
      }
    }
    dev::tc_fence_before();
  }
  if (S > 1) {
    dev::cluster_sync();  // every share is in its CTA's shared memory
    if (warp >= 2) {
      for (int t = rank; t < tokens; t += S) {
        float g = 0.0f, u = 0.0f;
        for (int s = 0; s < S; ++s) {
          const uint32_t base = dev::mapa(dev::smem_u32(part), static_cast<uint32_t>(s));
          g += ld_dsmem(base + static_cast<uint32_t>(t * 128 + n) * 4);
          if constexpr (SILU) u += ld_dsmem(base + static_cast<uint32_t>((T + t) * 128 + n) * 4);
        }
        emit<O, SILU>(args, tt * T + t, col, lane, g, u, bg, bu);
      }
    }
    dev::cluster_sync();  // no CTA leaves while a peer still reads its share
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    dev::tc_fence_after();
    dev::tmem_dealloc(tmem, P::kTmemCols);
  }
}

}  // namespace mx
}  // namespace w8a8
