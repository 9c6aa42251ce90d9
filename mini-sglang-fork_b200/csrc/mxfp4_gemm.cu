// Host side of the MXFP4 GEMM: which kernel a shape gets, the tensor maps, the
// launches.
#include <algorithm>
#include <cstring>
#include <mutex>

#include "gemm_api.h"
#include "mxfp4_pair_sm100.cuh"

namespace w8a8 {
namespace mx {
namespace {

// Allows a kernel its dynamic shared memory, once per device.
template <auto Kern>
int allow_smem(int bytes) {
  static std::mutex mu;
  static bool done[64] = {false};
  const int dev = current_device();
  W8A8_REQUIRE(dev >= 0 && dev < 64, W8A8_ERR_CUDA, "no current device");
  std::lock_guard<std::mutex> lk(mu);
  if (!done[dev]) {
    W8A8_CUDA_TRY(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return W8A8_OK;
}

// Scale tiles of [gate; up] ([2I, K]) to tiles of each half's own, zero beyond
// row I.  A thread moves 16 bytes: rows r, r + 32, r + 64, r + 96 of a tile (r <
// 32).  I is a multiple of 32, so these stay 32 apart, and begin `shift` groups
// of 32 inside a source tile: they are the last words of that tile's 16 bytes
// for r and the first of the next one's.
__global__ void __launch_bounds__(256) half_scales_kernel(const uint4* __restrict__ src, uint4* __restrict__ dst, int64_t I,
                                                          int64_t ktiles) {
  dev::griddep_launch();
  dev::griddep_wait();
  constexpr int kPieces = kTileBytes / 16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t rtiles = (I + 127) / 128, tile = i / kPieces;
  const int64_t rt = tile / ktiles, kt = tile - rt * ktiles;
  if (rt >= 2 * rtiles) return;
  const int64_t half = rt >= rtiles, t = rt - half * rtiles;  // of the half's tiles
  const int64_t row = half * I + t * 128;                     // of the first of its rows in the source
  const int shift = static_cast<int>(row >> 5) & 3;
  const int64_t at = ((row >> 7) * ktiles + kt) * kPieces + i % kPieces;
  const int groups = static_cast<int>(min(static_cast<int64_t>(4), (I - t * 128) >> 5));  // of 32 rows that exist
  const uint4 a = src[at];
  const uint4 b = shift + groups > 4 ? src[at + ktiles * kPieces] : make_uint4(0, 0, 0, 0);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t o[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t x = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) x = shift == s ? w[g + s] : x;
    o[g] = g < groups ? x : 0u;
  }
  dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
}

struct Operands {
  const uint8_t *a, *as, *b, *bs;
  int64_t b_rows;    // rows of B: N, or 2I
  int64_t bs_tiles;  // row tiles of B's scales: of N rows, or of I rows twice
};

// Clusters of s CTAs of `Kern` that the device holds at once with one CTA per
// SM, which is what the query assumes of kernels that allocate TMEM: fewer than
// SMs / s, since a cluster lives in one group of SMs.
template <auto Kern>
int active_clusters(int s, int threads, int smem, int* out) {
  static std::mutex mu;
  static int known[64][9] = {{0}};
  const int dev = current_device();
  W8A8_REQUIRE(dev >= 0 && dev < 64, W8A8_ERR_CUDA, "no current device");
  std::lock_guard<std::mutex> lk(mu);
  int& n = known[dev][s];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(s));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(s);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    W8A8_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, Kern, &cfg));
    if (n < 1) n = 1;
  }
  *out = n;
  return W8A8_OK;
}

// Launch in clusters of `cluster` CTAs, with programmatic stream serialisation.
template <typename Kernel, typename... Args>
int launch_cluster(Kernel kern, unsigned grid, int threads, int smem, int cluster, cudaStream_t stream,
                   const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  W8A8_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  return W8A8_OK;
}

// Shares of K per output tile, each the work of `ctas` CTAs: as many as leave
// every tile's cluster resident at once (a second wave would cost as much as
// the first), `most` at most, with `least` k blocks each: two, six with the SiLU
// epilogue's two sums, eight for a 256 x 256 block.  Measured (us, B200), by least:
//   plain, least 1, 2, 3, 4:  16 x 2048 x 2048  4.6 4.1 4.6 4.6;  16 x 4096 x 2048
//     5.2 4.7 4.8 4.8;  64 x 2048 x 2048  6.4 5.5 5.9 5.9;  but 16 x 2048 x 1024
//     4.0 3.9 3.3 3.3 and 128 x 4096 x 2048  8.6 8.6 7.8 7.8: two shares of two
//     blocks cost more than they save.  From 4096 x 4096 on there is no difference.
//   SiLU, least 3, 4, 6, 8:  64 x 2816 x 4096  11.7 10.7 10.3 10.3;  64 x 2816 x 8192
//     14.2 14.3 13.4 13.0;  16 x 1536 x 2048  6.6 6.6 5.9 5.9;  but 16 x 1536 x 4096
//     8.1 7.4 8.4 8.5.
//   pairs, least 4, 6, 8, 12:  512 x 4096 x 2048  9.6 7.6 7.5 7.5;  200 x 2048 x 5120
//     10.0 10.0 10.0 10.9;  512 x 4096 x 4096  11.1 11.1 11.1 10.3.
template <auto Kern>
int pick_split(int64_t tiles, int kblocks, int threads, int smem, int per_sm, int ctas, int most, int least, int* out) {
  *out = 1;
  for (int s = 2; s <= std::min(most, kblocks / least) && tiles * s * ctas <= per_sm * sm_count(); ++s) {
    int n = 0;
    if (int rc = active_clusters<Kern>(s * ctas, threads, smem, &n)) return rc;
    if (tiles <= per_sm * n) *out = s;
  }
  return W8A8_OK;
}

// (M <= T)
template <typename O, int T, bool SILU, bool DEEP>
int launch_row(const Operands& o, MxGemmArgs args, cudaStream_t stream) {
  using P = MxRowTraits<T, SILU, DEEP>;
  constexpr auto kern = mx_row_kernel<O, T, SILU, DEEP>;
  if (int rc = allow_smem<kern>(P::kSmemBytes)) return rc;
  const int64_t tiles = (args.N + 127) / 128;
  args.tiles = static_cast<int>(tiles);
  CUtensorMap tw, tws, tx, txs;
  if (int rc = encode_operand(&tw, o.b, o.b_rows, args.K / 2, 128)) return rc;
  if (int rc = encode_words(&tws, o.bs, o.bs_tiles, k_tiles(args.K) * kTileBytes / 4, 256)) return rc;
  if (int rc = encode_operand(&tx, o.a, args.M, args.K / 2, T)) return rc;
  if (int rc = encode_words(&txs, o.as, row_tiles(args.M), k_tiles(args.K) * kTileBytes / 4, 256)) return rc;
  int split = 1;
  if (DEEP)
    if (int rc = pick_split<kern>(tiles, args.kblocks, kRowThreads, P::kSmemBytes, P::kPerSm, 1, 8, SILU ? 6 : 2, &split)) return rc;
  const int64_t grid = split > 1 ? tiles * split : P::kPersistent ? std::min<int64_t>(tiles, std::max(1, sm_count())) : tiles;
  return launch_cluster(kern, static_cast<unsigned>(grid), kRowThreads, P::kSmemBytes, split, stream, tw, tws, tx, txs,
                        args);
}

template <typename O, bool SILU>
int launch_pair(const Operands& o, const MxGemmArgs& g, cudaStream_t stream) {
  constexpr auto kern = mx_pair_kernel<O, SILU>;
  if (int rc = allow_smem<kern>(PairTraits::kSmemBytes)) return rc;
  PairArgs args;
  args.g = g;
  args.pairs_m = (g.M + 255) / 256;
  args.tiles_n = SILU ? (g.N + 127) / 128 : (g.N + 255) / 256;
  const int64_t blocks = static_cast<int64_t>(args.pairs_m) * args.tiles_n;
  // (the block counter runs one grid past the last block)
  W8A8_REQUIRE(blocks <= 0x7fff0000LL, W8A8_ERR_UNSUPPORTED, "mxfp4_gemm: too many output tiles");
  CUtensorMap ta, tas, tb, tbs;
  if (int rc = encode_operand(&ta, o.a, g.M, g.K / 2, 128)) return rc;
  if (int rc = encode_words(&tas, o.as, row_tiles(g.M), k_tiles(g.K) * kTileBytes / 4, 256)) return rc;
  if (int rc = encode_operand(&tb, o.b, o.b_rows, g.K / 2, 128)) return rc;
  if (int rc = encode_words(&tbs, o.bs, o.bs_tiles, k_tiles(g.K) * kTileBytes / 4, 256)) return rc;
  int split = 1;
  if (int rc = pick_split<kern>(blocks, g.kblocks, PairTraits::kThreads, PairTraits::kSmemBytes, 1, 2, 2, 8, &split)) return rc;
  const int64_t pairs = split > 1 ? blocks * split : std::min<int64_t>(blocks, std::max(1, sm_count() / 2));
  return launch_cluster(kern, static_cast<unsigned>(2 * pairs), PairTraits::kThreads, PairTraits::kSmemBytes, 2 * split,
                        stream, ta, tas, tb, tbs, args);
}

// The short ring, several CTAs on an SM, once there are more tiles than SMs; else
// the long one, with K split.  (51200 x 5120, 400 tiles: 22.9 us with the short
// ring for 16 tokens, 26.9 with the long one; 28.7 and 34.6 for 64.)
template <typename O, int T, bool SILU>
int launch_row_any(const Operands& o, const MxGemmArgs& args, cudaStream_t stream) {
  if constexpr (!SILU && T < 128) {
    if ((args.N + 127) / 128 > sm_count()) return launch_row<O, T, false, false>(o, args, stream);
  }
  return launch_row<O, T, SILU, true>(o, args, stream);
}

// The smallest token tile that holds them all; SM pairs above 128 tokens, 64 with
// the SiLU epilogue (us, B200):
//   T = 16, 32, for 16 tokens:  51200 x 5120  22.9 28.1;  5120 x 5120  6.6 6.8;  gate_up
//     12288 x 4096  12.7 13.1
//   T = 64, 128, for 48:  51200 x 5120  28.3 31.6;  5120 x 5120  7.6 8.7;  5120 x 25600
//     16.0 16.3;  for 64:  28.7 26.5, 8.1 8.3, 16.5 16.8
//   T = 128, pairs, for 65:  51200 x 5120  27.0 29.9;  5120 x 25600  17.0 24.3;  for 128:
//     29.1 31.9, 18.9 24.6;  10240 x 5120  12.5 12.7
//   SiLU, T = 64, pairs, for 64:  2816 x 4096  10.3 11.0;  12288 x 4096  14.5 19.1;
//     25600 x 5120  28.8 30.7
template <typename O, bool SILU>
int dispatch(const Operands& o, const MxGemmArgs& args, cudaStream_t stream) {
  if (args.M <= 16) return launch_row_any<O, 16, SILU>(o, args, stream);
  if (args.M <= 32) return launch_row_any<O, 32, SILU>(o, args, stream);
  if (args.M <= 64) return launch_row_any<O, 64, SILU>(o, args, stream);
  if constexpr (!SILU)
    if (args.M <= 128) return launch_row_any<O, 128, false>(o, args, stream);
  return launch_pair<O, SILU>(o, args, stream);
}

int run(const char* what, const Operands& o, const void* bias, void* C, uint8_t* q, uint8_t* qs, int dtype, int64_t M,
        int64_t N, int64_t K, bool silu, cudaStream_t stream) {
  W8A8_REQUIRE(M >= 0 && N >= 0 && K >= 0, W8A8_ERR_INVALID_ARG, "%s: negative shape", what);
  if (M == 0 || N == 0) return W8A8_OK;
  W8A8_REQUIRE(K > 0 && K % kBlock == 0, W8A8_ERR_INVALID_ARG, "%s: K=%lld must be a positive multiple of 32", what,
               (long long)K);
  W8A8_REQUIRE(o.a && o.as && o.b && o.bs && (silu ? q && qs : C != nullptr), W8A8_ERR_INVALID_ARG, "%s: null pointer", what);
  W8A8_REQUIRE(dtype == kBf16 || dtype == kFp16, W8A8_ERR_INVALID_ARG, "%s: bf16 or fp16", what);
  W8A8_REQUIRE(M <= (1LL << 27) && N <= (1LL << 27) && K <= (1LL << 27), W8A8_ERR_UNSUPPORTED, "%s: shape too large",
               what);
  W8A8_REQUIRE(!silu || N % kBlock == 0, W8A8_ERR_INVALID_ARG, "%s: I=%lld must be a multiple of 32", what, (long long)N);
  W8A8_REQUIRE(W8A8_ALIGNED16(o.a) && W8A8_ALIGNED16(o.as) && W8A8_ALIGNED16(o.b) && W8A8_ALIGNED16(o.bs) &&
                   W8A8_ALIGNED16(C) && W8A8_ALIGNED16(q) && W8A8_ALIGNED16(qs) &&
                   (reinterpret_cast<uintptr_t>(bias) & 1u) == 0,
               W8A8_ERR_ALIGNMENT, "%s: operands and result must be 16-byte aligned", what);
  W8A8_REQUIRE(device_cc_major() == 10, W8A8_ERR_UNSUPPORTED,
               "%s: the tcgen05 kernels need an sm_100 (B200) device; found compute capability %d.x", what,
               device_cc_major());
  MxGemmArgs args;
  std::memset(&args, 0, sizeof(args));
  args.bias = bias;
  args.out = C;
  args.q = q;
  args.qs = qs;
  args.err = device_error_word();
  if (!args.err) return W8A8_ERR_CUDA;
  args.timeout_ns = kDefaultGemmTimeoutNs;
  args.M = static_cast<int>(M);
  args.N = static_cast<int>(N);
  args.K = static_cast<int>(K);
  args.kblocks = static_cast<int>((K + 255) / 256);
  if (dtype == kBf16)
    return silu ? dispatch<__nv_bfloat16, true>(o, args, stream) : dispatch<__nv_bfloat16, false>(o, args, stream);
  return silu ? dispatch<__half, true>(o, args, stream) : dispatch<__half, false>(o, args, stream);
}

}  // namespace
}  // namespace mx
}  // namespace w8a8

extern "C" {

int mxfp4_gemm(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data, const uint8_t* b_scales,
               const void* bias, void* C, int dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace w8a8;
  return mx::run("mxfp4_gemm", {a_data, a_scales, b_data, b_scales, N, mx::row_tiles(N)}, bias, C, nullptr, nullptr,
                 dtype, M, N, K, false, static_cast<cudaStream_t>(stream));
}

int mxfp4_gemm_silu_quant(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data,
                          const uint8_t* b_scales, const void* bias, int dtype, uint8_t* y_data, uint8_t* y_scales,
                          int64_t M, int64_t I, int64_t K, void* stream) {
  using namespace w8a8;
  W8A8_REQUIRE(I <= 0 || I % 128 == 0, W8A8_ERR_UNSUPPORTED,
               "mxfp4_gemm_silu_quant: I=%lld must be a multiple of 128 (mxfp4_gemm_silu_quant_halves takes the others)",
               (long long)I);
  return mx::run("mxfp4_gemm_silu_quant", {a_data, a_scales, b_data, b_scales, 2 * I, 2 * mx::row_tiles(I)}, bias,
                 nullptr, y_data, y_scales, dtype, M, I, K, true, static_cast<cudaStream_t>(stream));
}

int mxfp4_gemm_silu_quant_halves(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data,
                                 const uint8_t* b_half_scales, const void* bias, int dtype, uint8_t* y_data,
                                 uint8_t* y_scales, int64_t M, int64_t I, int64_t K, void* stream) {
  using namespace w8a8;
  return mx::run("mxfp4_gemm_silu_quant_halves",
                 {a_data, a_scales, b_data, b_half_scales, 2 * I, 2 * mx::row_tiles(I)}, bias, nullptr, y_data, y_scales,
                 dtype, M, I, K, true, static_cast<cudaStream_t>(stream));
}

int mxfp4_half_scales(const uint8_t* scales, uint8_t* half_scales, int64_t I, int64_t K, void* stream) {
  using namespace w8a8;
  W8A8_REQUIRE(I >= 0 && K >= 0, W8A8_ERR_INVALID_ARG, "mxfp4_half_scales: negative shape");
  if (I == 0) return W8A8_OK;
  W8A8_REQUIRE(I % mx::kBlock == 0 && K > 0 && K % mx::kBlock == 0, W8A8_ERR_INVALID_ARG,
               "mxfp4_half_scales: I=%lld and K=%lld must be positive multiples of 32", (long long)I, (long long)K);
  W8A8_REQUIRE(scales && half_scales, W8A8_ERR_INVALID_ARG, "mxfp4_half_scales: null pointer");
  W8A8_REQUIRE(I <= (1LL << 27) && K <= (1LL << 27), W8A8_ERR_UNSUPPORTED, "mxfp4_half_scales: shape too large");
  W8A8_REQUIRE(W8A8_ALIGNED16(scales) && W8A8_ALIGNED16(half_scales), W8A8_ERR_ALIGNMENT,
               "mxfp4_half_scales: pointers must be 16-byte aligned");
  const int64_t pieces = 2 * mx::row_tiles(I) * mx::k_tiles(K) * (mx::kTileBytes / 16);
  const int64_t ctas = (pieces + 255) / 256;
  W8A8_REQUIRE(ctas < (1LL << 31), W8A8_ERR_UNSUPPORTED, "mxfp4_half_scales: shape too large");
  W8A8_CUDA_TRY(launch_pdl(mx::half_scales_kernel, dim3(static_cast<unsigned>(ctas)), dim3(256), 0,
                           static_cast<cudaStream_t>(stream), reinterpret_cast<const uint4*>(scales),
                           reinterpret_cast<uint4*>(half_scales), I, mx::k_tiles(K)));
  return W8A8_OK;
}

}  // extern "C"
