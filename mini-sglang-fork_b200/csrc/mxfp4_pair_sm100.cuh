// MXFP4 GEMM for prefill: 256 x 256 output blocks on SM pairs.
//
// A cluster of two CTAs shares one tcgen05.mma.cta_group::2 (M = 256, N = 256,
// 64 values of K): CTA h stages rows [128h, 128h + 128) of A and of B and the
// scales of its A rows and of all 256 B rows, 35 KB per 256-value k block; the
// even CTA issues the scale copies and the MMAs, which work on both CTAs'
// shared memory and TMEM.  At the fp4 rate a pair needs 64 operand bytes per
// clock and SM, which is about what the L2 gives; any smaller block would be
// bound by that.
//
// Two 256-column accumulators and the scales do not fit TMEM's 512 columns, so
// the accumulators overlap by 128: accumulator 0 is columns [0, 256),
// accumulator 1 [128, 384), and every stage of the ring has its own 24 scale
// columns from 384 on.  The epilogue reads the 128 shared columns into
// registers first and releases them; the next block's MMAs wait for those
// only, while the rest is still being read.
//
// With few blocks a cluster of two pairs works on one, each on a half of K; each
// pair finishes a half of the columns (S = 2 below; 1 otherwise).
#pragma once

#include "mxfp4_sm100.cuh"

namespace w8a8 {
namespace mx {

struct PairTraits {
  static constexpr int kStages = 5;
  static constexpr int kTile = 128 * 128;  // bytes of 128 rows of a k block
  static constexpr int kSf = 1024;
  static constexpr int kStageBytes = 2 * kTile + 3 * kSf;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int kAccStep = 128;  // columns from accumulator 0 to accumulator 1
  static constexpr int kSfCol = 384;    // a stage's scales: A 8 columns, B 16
  static constexpr int kSfCols = 24;
  static_assert(kSfCol + kStages * kSfCols <= 512, "TMEM");
  static constexpr int kBarrierBytes = 256;
  static constexpr int kStagingBytes = kEpiWarps * 2048;
  static constexpr int kBiasBytes = 2 * 1024;  // of a block's 256 columns, for two blocks
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBarrierBytes + kStagingBytes + kBiasBytes;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(2 * 128 * 128 * 4 <= kStages * kStageBytes, "the shares reuse the ring");
  static_assert(kSmemBytes >= 170 * 1024, "TMEM share");  // as for MxRowTraits
};

__device__ __forceinline__ void cp_scales_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

__device__ __forceinline__ void mma_mxf4_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// Arrive on an mbarrier of either CTA without releasing this thread's memory
// operations.  It announces only that tcgen05.ld has delivered its registers
// (tcgen05.wait::ld and fence::before_thread_sync come first); a releasing
// arrive waits for the warp's output stores of the block before, 1500 clocks
// during which the next block's MMAs stand still.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

struct PairArgs {
  MxGemmArgs g;
  int pairs_m;  // 256-row blocks of the output
  int tiles_n;  // 256-column blocks (SiLU: 128 features)
};

// Block p -> (256-row block, column block): groups of up to 16 row blocks, the
// row block running fastest, so that the pairs at work share a few column
// blocks and a group's A (16 x 256 rows) stays in L2 while B streams past.
__device__ __forceinline__ void pair_block(const PairArgs& a, int p, int& pm, int& tn) {
  constexpr int kGroup = 16;
  const int group = p / (kGroup * a.tiles_n);
  const int first = group * kGroup;
  const int rows = min(kGroup, a.pairs_m - first);
  const int r = p - group * kGroup * a.tiles_n;
  pm = first + r % rows;
  tn = r / rows;
}

// Word offset of column c (a multiple of 4) of a row in a [128][32] fp32 array
// whose 16-byte pieces are XORed with the row (part_word).
__device__ __forceinline__ uint32_t pair_part_word(int r, int c) {
  return static_cast<uint32_t>(r * 32 + (((c >> 2) ^ (r & 7)) << 2));
}

// Plain epilogue of 32 columns (from `col0`, their biases in shared memory at
// `bias`) of a warp's 32 rows: through the
// warp's 2 KB of shared memory (16-byte pieces, the piece index XORed with the
// row pair: no bank conflict either way) to rows of 64 contiguous bytes.
template <typename O>
__device__ __forceinline__ void plain_chunk(const MxGemmArgs& g, const float* bias, uint32_t (&v)[32], uint4* stg,
                                            int lane, int64_t row0, int col0) {
  if (g.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = *reinterpret_cast<const float4*>(bias + 4 * i);
      v[4 * i] = __float_as_uint(__uint_as_float(v[4 * i]) + b.x);
      v[4 * i + 1] = __float_as_uint(__uint_as_float(v[4 * i + 1]) + b.y);
      v[4 * i + 2] = __float_as_uint(__uint_as_float(v[4 * i + 2]) + b.z);
      v[4 * i + 3] = __float_as_uint(__uint_as_float(v[4 * i + 3]) + b.w);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = pack2<O>(__uint_as_float(v[8 * e + 2 * k]), __uint_as_float(v[8 * e + 2 * k + 1]));
    stg[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __syncwarp();
  if ((g.N & 7) == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e * 8 + (lane >> 2), piece = lane & 3;
      store8_row<O>(g, row0 + r, col0 + piece * 8, stg[r * 4 + (piece ^ ((r >> 1) & 3))]);
    }
  } else if (col0 + lane < g.N) {  // rows that are not 16-byte aligned: a row at a time, a value per lane
    O* dst = static_cast<O*>(g.out) + col0 + lane;
    for (int r = 0; r < 32 && row0 + r < g.M; ++r)
      dst[(row0 + r) * g.N] = reinterpret_cast<const O*>(stg + r * 4 + ((lane >> 3) ^ ((r >> 1) & 3)))[lane & 7];
  }
  __syncwarp();
}

template <typename O, bool SILU>
__global__ void __launch_bounds__(PairTraits::kThreads, 1)
    mx_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_as,
                   const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_bs,
                   const PairArgs args) {
  using P = PairTraits;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_a = smem;
  uint8_t* s_b = s_a + P::kStages * P::kTile;
  uint8_t* s_as = s_b + P::kStages * P::kTile;
  uint8_t* s_bs = s_as + P::kStages * P::kSf;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_bs + P::kStages * 2 * P::kSf);
  uint64_t* full = bars;
  uint64_t* empty = bars + P::kStages;
  uint64_t* acc_full = bars + 2 * P::kStages;  // [2]
  uint64_t* acc_free = acc_full + 2;           // the overlap of a block's accumulator has been read
  uint64_t* drain = acc_free + 1;
  uint64_t* arrived = drain + 1;  // S > 1: the other share's sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* staging = reinterpret_cast<uint8_t*>(bars) + P::kBarrierBytes;
  float* bias_s = reinterpret_cast<float*>(staging + P::kStagingBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = dev::cluster_rank();
  const uint32_t half = rank & 1u;  // 0 = leader of its pair
  const uint32_t leader = rank & ~1u;
  const int S = static_cast<int>(cluster_size() >> 1);  // shares of K
  const int share = static_cast<int>(rank >> 1);
  const int first = blockIdx.x / (2 * S);
  const int step = gridDim.x / (2 * S);  // (S > 1: one block per cluster)
  const int blocks = args.pairs_m * args.tiles_n;
  const MxGemmArgs& g = args.g;
  const int kb0 = static_cast<int>(static_cast<int64_t>(share) * g.kblocks / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(share + 1) * g.kblocks / S);
  const long long tmo = g.timeout_ns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P::kStages; ++s) {
      dev::mbar_init(dev::smem_u32(full + s), 1);
      dev::mbar_init(dev::smem_u32(empty + s), 1);
    }
    dev::mbar_init(dev::smem_u32(acc_full), 1);
    dev::mbar_init(dev::smem_u32(acc_full + 1), 1);
    dev::mbar_init(dev::smem_u32(acc_free), 2 * P::kEpiWarps);  // the epilogue warps of both CTAs
    dev::mbar_init(dev::smem_u32(drain), 1);
    dev::mbar_init(dev::smem_u32(arrived), 1);
    *abort_flag = 0;
    dev::fence_mbar_init();
    dev::prefetch_tmap(&tm_a);
    dev::prefetch_tmap(&tm_as);
    dev::prefetch_tmap(&tm_b);
    dev::prefetch_tmap(&tm_bs);
  }
  if (warp == 1) {
    dev::tmem_alloc2(dev::smem_u32(tmem_slot), 512);
    dev::tmem_relinquish2();
  }
  dev::tc_fence_before();
  dev::cluster_sync();  // barriers of both CTAs initialised before any cross-CTA use
  dev::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);  // (the same in every lane, and known to be)
  dev::griddep_launch();
  dev::griddep_wait();  // any operand may be the previous kernel's output

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
    bool ok = true;
    for (int p = first; ok && p < blocks; p += step) {
      int pm, tn;
      pair_block(args, p, pm, tn);
      const int ta = 2 * pm + static_cast<int>(half);  // 128-row tile of A
      // 128-row tiles of B: the block's two, or its gate rows and their up rows
      const int tb0 = SILU ? tn : 2 * tn;
      const int tb1 = SILU ? tn + ((g.N + 127) >> 7) : 2 * tn + 1;
      const int b_row = half == 0 ? tb0 * 128 : SILU ? tn * 128 + g.N : tb1 * 128;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = warp_wait(dev::smem_u32(empty + stage), phase ^ 1u, abort_flag, g.err, tmo);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t bar = dev::mapa(dev::smem_u32(full + stage), leader);
          if (half == 0) dev::mbar_expect_tx(dev::smem_u32(full + stage), 2 * P::kStageBytes);
          dev::tma_load_2d_pair(dev::smem_u32(s_a + stage * P::kTile), &tm_a, bar, kb * 128, ta * 128);
          dev::tma_load_2d_pair(dev::smem_u32(s_b + stage * P::kTile), &tm_b, bar, kb * 128, b_row);
          dev::tma_load_2d_pair(dev::smem_u32(s_as + stage * P::kSf), &tm_as, bar, kb * 256, ta);
          dev::tma_load_2d_pair(dev::smem_u32(s_bs + stage * 2 * P::kSf), &tm_bs, bar, kb * 256, tb0);
          dev::tma_load_2d_pair(dev::smem_u32(s_bs + (stage * 2 + 1) * P::kSf), &tm_bs, bar, kb * 256, tb1);
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
    // The leader's full barriers count both CTAs' bytes: once they have landed,
    // no copy of either CTA is in flight (the pair then meets at the closing
    // cluster barrier).
    if (half == 0 && lane == 0)
      for (int s = 0; s < P::kStages; ++s)
        if (issued_mask & (1u << s))
          if (!dev::mbar_wait_drain(dev::smem_u32(full + s), (issued_phase >> s) & 1u, tmo))
            if (g.err) atomicOr(g.err, kErrGemmDrain);
  } else if (warp == 1) {
    if (half == 0) {
      // --------------------------------------------- MMA issuer (leader only)
      int stage = 0;
      uint32_t phase = 0, blk = 0;
      bool ok = true, ready = false;  // ready: the next stage has been seen full
      for (int p = first; ok && p < blocks; p += step, ++blk) {
        if (blk > 0 && !__all_sync(0xffffffffu, dev::mbar_wait_cluster(dev::smem_u32(acc_free), (blk - 1) & 1u,
                                                                       abort_flag, g.err, kErrGemmWait, tmo)))
          break;
        dev::tc_fence_after();
        const uint32_t d = tmem + (blk & 1u) * P::kAccStep;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ready) {
            ok = warp_wait(dev::smem_u32(full + stage), phase, abort_flag, g.err, tmo);
            if (!ok) break;
          }
          dev::tc_fence_after();
          const int next = stage + 1 == P::kStages ? 0 : stage + 1;
          const uint32_t next_phase = next == 0 ? phase ^ 1u : phase;
          // looked at before this block's MMAs are issued: the issue blocks
          // while earlier MMAs run, and hides the look's latency
          ready = __all_sync(0xffffffffu, dev::mbar_peek(dev::smem_u32(full + next), next_phase));
          if (elect_one()) {
            const uint32_t sfa = tmem + P::kSfCol + stage * P::kSfCols;
            const uint32_t sfb = sfa + 8;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              cp_scales_pair(sfa + 4 * c, sdesc_scales(dev::smem_u32(s_as + stage * P::kSf + c * kTileBytes)));
              cp_scales_pair(sfb + 8 * c, sdesc_scales(dev::smem_u32(s_bs + stage * 2 * P::kSf + c * kTileBytes)));
              cp_scales_pair(sfb + 8 * c + 4,
                             sdesc_scales(dev::smem_u32(s_bs + (stage * 2 + 1) * P::kSf + c * kTileBytes)));
            }
            const uint64_t da = dev::sdesc_k_sw128(dev::smem_u32(s_a + stage * P::kTile));
            const uint64_t db = dev::sdesc_k_sw128(dev::smem_u32(s_b + stage * P::kTile));
            const int steps = min(4, (g.K - kb * 256 + 63) / 64);  // beyond K: nothing to add
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k >= steps) break;
              constexpr uint32_t ids[2] = {idesc_mxf4(256, 256, 0), idesc_mxf4(256, 256, 2)};
              mma_mxf4_pair(d, da + 2 * k, db + 2 * k, ids[k & 1], sfa + 4 * (k >> 1), sfb + 8 * (k >> 1),
                            (kb > kb0 || k > 0) ? 1u : 0u);
            }
            dev::tc_commit_pair(dev::mapa(dev::smem_u32(empty + stage), leader));
            dev::tc_commit_pair(dev::mapa(dev::smem_u32(empty + stage), leader + 1));
          }
          __syncwarp();
          stage = next;
          phase = next_phase;
        }
        if (!ok) break;
        if (elect_one()) {
          dev::tc_commit_pair(dev::mapa(dev::smem_u32(acc_full + (blk & 1u)), leader));
          dev::tc_commit_pair(dev::mapa(dev::smem_u32(acc_full + (blk & 1u)), leader + 1));
        }
        __syncwarp();
      }
      if (elect_one()) dev::tc_commit_pair(dev::mapa(dev::smem_u32(drain), leader));
      if (lane == 0 && !dev::mbar_wait_drain(dev::smem_u32(drain), 0, tmo))
        if (g.err) atomicOr(g.err, kErrGemmDrain);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;      // TMEM lane quarter (warp id mod 4)
    const int hh = (warp - 2) >> 2;    // which of the two warps of that quarter
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint4* stg = reinterpret_cast<uint4*>(staging + (warp - 2) * 2048);
    const uint32_t free_bar = dev::mapa(dev::smem_u32(acc_free), leader);
    uint32_t blk = 0;
    for (int p = first; p < blocks; p += step, ++blk) {
      int pm, tn;
      pair_block(args, p, pm, tn);
      const int row0 = (2 * pm + static_cast<int>(half)) * 128 + quarter * 32;  // this warp's rows
      const uint32_t acc = blk & 1u;
      float* bias = bias_s + acc * 256;  // before the wait for the sums
      if (g.bias) {
        const int et = threadIdx.x - 64;
        const O* b = static_cast<const O*>(g.bias);
        const int c = SILU ? tn * 128 + (et & 127) : tn * 256 + et;
        bias[et] = c < g.N ? to_float(b[SILU ? c + (et >> 7) * g.N : c]) : 0.0f;
      }
      const bool ok = warp_wait(dev::smem_u32(acc_full + acc), (blk >> 1) & 1u, abort_flag, g.err, tmo);
      if (g.bias ? dev::named_bar_or(1, 32 * P::kEpiWarps, !ok) : !ok) break;  // (publishes the biases)
      dev::tc_fence_after();
      const uint32_t t = tmem + lanes + acc * P::kAccStep;
      if (S > 1) break;  // one block, finished below
      // the shared columns: chunks of 32, 4.. 7 of accumulator 0, 0..3 of
      // accumulator 1; this warp's are hh and hh + 2 of the four
      const uint32_t shared_t = t + (acc ? 0 : 128), own_t = t + (acc ? 128 : 0);
      uint32_t s0[32], s1[32], v[32];
      dev::tmem_ld32(shared_t + 32 * hh, s0);
      dev::tmem_ld32(shared_t + 32 * hh + 64, s1);
      dev::tmem_wait_ld(s0);
      dev::tmem_wait_ld(s1);
      dev::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed(free_bar);
      if constexpr (SILU) {
        // columns [0, 128): gate features, [128, 256): their up features
        const auto block = [&](const uint32_t (&sh)[32], const uint32_t (&own)[32], int j) {
          float gate[32], up[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            gate[e] = __uint_as_float(acc ? sh[e] : own[e]);
            up[e] = __uint_as_float(acc ? own[e] : sh[e]);
          }
          silu_block(g, bias, gate, up, row0 + lane, tn, j);
          __syncwarp();  // (tcgen05.ld and the closing barriers want a converged warp)
        };
        dev::tmem_ld32(own_t + 32 * hh, v);
        dev::tmem_wait_ld(v);
        block(s0, v, hh);
        dev::tmem_ld32(own_t + 32 * hh + 64, v);
        dev::tmem_wait_ld(v);
        block(s1, v, hh + 2);
      } else {
        const int cs = tn * 256 + (acc ? 0 : 128) + 32 * hh, co = tn * 256 + (acc ? 128 : 0) + 32 * hh;
        dev::tmem_ld32(own_t + 32 * hh, v);  // lands while the first chunk is written
        const float* bs = bias + (cs - tn * 256);
        const float* bo = bias + (co - tn * 256);
        plain_chunk<O>(g, bs, s0, stg, lane, row0, cs);
        plain_chunk<O>(g, bs + 64, s1, stg, lane, row0, cs + 64);
        dev::tmem_wait_ld(v);
        dev::tmem_ld32(own_t + 32 * hh + 64, s0);
        plain_chunk<O>(g, bo, v, stg, lane, row0, co);
        dev::tmem_wait_ld(s0);
        plain_chunk<O>(g, bo + 64, s0, stg, lane, row0, co + 64);
      }
    }
    dev::tc_fence_before();
  }

  if (S > 1) {
    // Two pairs, each with a half of K.  CTA (share s, half) writes the s-th
    // half of its rows' columns (SiLU: of the features): chunks of 32 columns,
    // [4 chunks][128 rows][32] words.  The other share's four go to its CTA of
    // the same rows, and that CTA's come here.
    constexpr int kChunkWords = 128 * 32;
    constexpr uint32_t kBytes = 4 * kChunkWords * 4;
    float* out = reinterpret_cast<float*>(smem);
    float* in = out + 4 * kChunkWords;
    if (threadIdx.x == 64) dev::mbar_expect_tx(dev::smem_u32(arrived), kBytes);
    dev::cluster_sync();  // every pair's MMAs are done: the rings may be written
    if (warp >= 2) {
      const int quarter = warp & 3, hh = (warp - 2) >> 2;
      const int row = quarter * 32 + lane;
      const uint32_t t = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
      // chunk i (0..3) of share s: columns, or features i & 1 of gate (i < 2) and up
      const auto column = [&](int s, int i) { return SILU ? 128 * (i >> 1) + 64 * s + 32 * (i & 1) : 128 * s + 32 * i; };
      dev::tc_fence_after();
#pragma unroll 1
      for (int i = hh; i < 4; i += 2) {
        uint32_t v[32];
        dev::tmem_ld32(t + column(share ^ 1, i), v);
        dev::tmem_wait_ld(v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(out + i * kChunkWords + pair_part_word(row, 4 * e)) =
              make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
      }
      fence_async_smem();
      dev::named_bar_sync(1, 32 * P::kEpiWarps);
      if (threadIdx.x == 64) {
        const uint32_t peer = rank ^ 2u;
        dsmem_copy(dev::mapa(dev::smem_u32(in), peer), dev::smem_u32(out), kBytes, dev::mapa(dev::smem_u32(arrived), peer));
      }
      __syncwarp();
      // this CTA's own chunk i plus the other share's (share 0's first)
      const auto sum = [&](int i, uint32_t (&v)[32]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4 x = *reinterpret_cast<const float4*>(in + i * kChunkWords + pair_part_word(row, 4 * e));
          const float p[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) v[4 * e + k] = __float_as_uint(__uint_as_float(v[4 * e + k]) + p[k]);
        }
      };
      int pm, tn;
      pair_block(args, first, pm, tn);
      const int row0 = (2 * pm + static_cast<int>(half)) * 128 + quarter * 32;
      uint32_t v[32], w[32];
      if (warp_wait(dev::smem_u32(arrived), 0, abort_flag, g.err, tmo)) {
        if constexpr (SILU) {  // this warp: feature block hh of the share's two
          dev::tmem_ld32(t + column(share, hh), v);
          dev::tmem_ld32(t + column(share, 2 + hh), w);
          dev::tmem_wait_ld(v);
          dev::tmem_wait_ld(w);
          sum(hh, v);
          sum(2 + hh, w);
          float gate[32], up[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            gate[e] = __uint_as_float(v[e]);
            up[e] = __uint_as_float(w[e]);
          }
          silu_block(g, bias_s, gate, up, row0 + lane, tn, 2 * share + hh);
          __syncwarp();
        } else {
#pragma unroll 1
          for (int i = hh; i < 4; i += 2) {
            dev::tmem_ld32(t + column(share, i), v);
            dev::tmem_wait_ld(v);
            sum(i, v);
            plain_chunk<O>(g, bias_s + column(share, i), v, reinterpret_cast<uint4*>(staging + (warp - 2) * 2048), lane,
                           row0, tn * 256 + column(share, i));
          }
        }
      }
      dev::tc_fence_before();
    }
  }

  __syncthreads();
  dev::cluster_sync();  // the cluster is done with every CTA's TMEM and shared memory
  if (warp == 1) {
    dev::tc_fence_after();
    dev::tmem_dealloc2(tmem, 512);
  }
}

}  // namespace mx
}  // namespace w8a8
