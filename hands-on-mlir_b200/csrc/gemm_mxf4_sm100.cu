// Product of two microscaled 4-bit matrices (format: mxf4_sm100.cuh) on the block-scaled tensor
// path: D = act(alpha * A.B^T + beta * C), fp32 accumulation, fp16 C and D.
//
// One CTA per 128 x 128 tile of D.  A K step is 256 values: 128 bytes of codes a row, fetched by
// TMA into 128-byte-swizzled tiles like the fp16 kernels' 64 values, and two scale tiles for each
// operand, which tcgen05.cp takes from shared to tensor memory right before the four MMAs that use
// them.  Zeros that TMA fills in beyond the matrix (codes 0, scales 2^-127) add nothing.
//
//   warp 0  TMA producer      warp 1  tensor memory, scale copies, MMA issue
//   warps 2-9  epilogue (gemm_epilogue.cuh), one 32 x 64 block each
#include "gemm_epilogue.cuh"
#include "gemm_sm100.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

using namespace hom::ptx;
using gemm::EpilogueParams;

namespace {

constexpr int BM = 128, BN = 128;
constexpr int kStepBytes = 128;                       // of a row of codes: 256 values
constexpr int kStepBlocks = 2 * kStepBytes / kBlock;  // 8
constexpr int kStepTiles = kStepBlocks / kTileBlocks; // 2 scale tiles
constexpr int kMmasPerStep = 4;
constexpr int kStages = 4;
constexpr int kDrainWarps = 8;
constexpr int kThreads = 32 * (2 + kDrainWarps);
constexpr uint32_t kABytes = BM * kStepBytes, kBBytes = BN * kStepBytes;
constexpr uint32_t kScaleBytes = kStepTiles * kTileBytes;
constexpr uint32_t kStageBytes = kABytes + kBBytes + 2 * kScaleBytes;
static_assert(kStageBytes % 1024 == 0, "swizzled tiles start on 1024 bytes");
constexpr uint32_t kStagingBytes = kDrainWarps * gemm::kEpilogueStageBytes;
constexpr uint32_t kBarrierBytes = 8 * (2 * kStages + 1) + 16;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarrierBytes + 1024;
// tensor memory: the accumulator, then the scales of two steps in turn
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kTmemScales = BN, kTmemScalesB = kStepTiles * 4, kTmemScaleSet = 2 * kStepTiles * 4;

struct Params {
  EpilogueParams ep;
  int steps, n_blocks;
  int *status;
};

__global__ void __launch_bounds__(kThreads, 1)
gemm_mxf4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                 const __grid_constant__ CUtensorMap tmD, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t staging_base = smem_base + kStages * kStageBytes;
  const uint32_t bar_base = staging_base + kStagingBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  const uint32_t acc_bar = bar_base + 8u * (2 * kStages);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kStages * kStageBytes + kStagingBytes +
                                                                       8 * (2 * kStages + 1));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = static_cast<int>(blockIdx.x) / p.n_blocks * BM, n0 = static_cast<int>(blockIdx.x) % p.n_blocks * BN;

  if (threadIdx.x == 64) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmSA);
    prefetch_tensormap(&tmSB);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 0) {
    if (elect_one()) {
      pdl_wait();
      bool ok = true;
      int armed = 0;
      for (int i = 0; i < p.steps; ++i) {
        const int s = i % kStages;
        const uint32_t ph = (i / kStages) & 1;
        ok = mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
        if (!ok) break;
        const uint32_t dst = smem_base + s * kStageBytes;
        mbar_arrive_expect_tx(full_bar(s), kStageBytes);
        tma_load_2d(dst, &tmA, full_bar(s), i * (kStepBytes / 2), m0);
        tma_load_2d(dst + kABytes, &tmB, full_bar(s), i * (kStepBytes / 2), n0);
        tma_load_3d(dst + kABytes + kBBytes, &tmSA, full_bar(s), 0, i * kStepTiles, m0 / kTileRows);
        tma_load_3d(dst + kABytes + kBBytes + kScaleBytes, &tmSB, full_bar(s), 0, i * kStepTiles, n0 / kTileRows);
        ++armed;
      }
      if (!ok) {
        // Let every copy this thread started land before the CTA gives its shared memory back.
        const long long t0 = clock64();
        for (int st = 0; st < kStages; ++st) {
          const int n_st = armed / kStages + (st < armed % kStages ? 1 : 0);
          if (n_st > 0)
            while (!mbar_try_wait(full_bar(st), (n_st - 1) & 1) && clock64() - t0 < 400000000LL) {
            }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      bool ok = true;
      for (int i = 0; i < p.steps; ++i) {
        const int s = i % kStages;
        ok = mbar_wait(full_bar(s), (i / kStages) & 1, abort_flag, p.status, kDevWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t src = smem_base + s * kStageBytes;
        const uint32_t scales = tmem_base + kTmemScales + (i & 1) * kTmemScaleSet;
#pragma unroll
        for (int t = 0; t < 2 * kStepTiles; ++t)
          tc_copy_scales(scales + t * 4, make_smem_desc_scales(src + kABytes + kBBytes + t * kTileBytes));
        const uint64_t da = make_smem_desc_sw128(src, 16, 1024), db = make_smem_desc_sw128(src + kABytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < kMmasPerStep; ++k)
          tc_mma_mxf4_ss(tmem_base, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32),
                         k & 1 ? make_idesc_mxf4(BM, BN, 1) : make_idesc_mxf4(BM, BN, 0), scales + (k >> 1) * 4,
                         scales + kTmemScalesB + (k >> 1) * 4, i != 0 || k != 0 ? 1u : 0u);
        tc_commit(empty_bar(s));
      }
      if (ok) tc_commit(acc_bar);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const int col_begin = ((warp - 2) >> 2) * 64;
    uint4 cval[8];
    pdl_wait();  // C may be produced, and D still read, by the previous kernel
    gemm::epilogue_load_c(p.ep, m0 + quarter * 32 + lane, n0 + col_begin, cval);
    bool ok = mbar_wait(acc_bar, 0, abort_flag, p.status, kDevWaitTimeoutEpilogue);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after_sync();
      gemm::epilogue_warp_block(p.ep, &tmD, tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col_begin,
                                m0 + quarter * 32, n0 + col_begin, true, staging_base + (warp - 2) * gemm::kEpilogueStageBytes,
                                lane, cval, [] {});
      if (lane == 0) bulk_wait_group_read_0();
      __syncwarp();
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace

bool run_product(const Problem &pb, cudaStream_t stream) {
  if (pb.N % 8 == 0 && (pb.M + 255) / 256 * ((pb.N + 255) / 256) >= 16) return run_product_pair(pb, stream);
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (!attr_set[dev]) {
    if (!check_cuda(cudaFuncSetAttribute(gemm_mxf4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes),
                    "cudaFuncSetAttribute(4-bit product)"))
      return false;
    attr_set[dev] = true;
  }
  const int64_t pitch = pb.blocks * 8;  // in two-byte elements, what the tensor maps count in
  const int64_t tile_cols = tile_cols_of(pb.blocks);
  const bool unaligned_n = pb.N % 8 != 0;
  CUtensorMap tmA, tmB, tmSA, tmSB, tmD;
  if (!gemm::make_tensor_map_2d(pb.A, pitch, pb.M, kStepBytes / 2, BM, &tmA) ||
      !gemm::make_tensor_map_2d(pb.B, pitch, pb.N, kStepBytes / 2, BN, &tmB) ||
      !gemm::make_tensor_map_scales(pb.scales_a, tile_cols, tile_rows_of(pb.M), kStepTiles, BM / kTileRows, &tmSA) ||
      !gemm::make_tensor_map_scales(pb.scales_b, tile_cols, tile_rows_of(pb.N), kStepTiles, BN / kTileRows, &tmSB))
    return false;
  if (unaligned_n) tmD = tmA;  // never dereferenced: the epilogue stores without TMA
  else if (!gemm::make_tensor_map_2d(pb.D, pb.N, pb.M, 64, 32, &tmD)) return false;
  Params p = {};
  p.ep.C = pb.C;
  p.ep.ldc = pb.N;
  p.ep.c_mode = pb.c_mode;
  p.ep.D = pb.D;
  p.ep.ldd = pb.N;
  p.ep.alpha = pb.alpha;
  p.ep.beta = pb.beta;
  p.ep.act = pb.act;
  p.ep.M = static_cast<int>(pb.M);
  p.ep.N = static_cast<int>(pb.N);
  p.ep.unaligned_n = unaligned_n ? 1 : 0;
  p.steps = static_cast<int>((pb.blocks + kStepBlocks - 1) / kStepBlocks);
  p.n_blocks = static_cast<int>((pb.N + BN - 1) / BN);
  p.status = device_status_word();
  const int64_t tiles = (pb.M + BM - 1) / BM * p.n_blocks;
  if (tiles > INT32_MAX) {
    set_error(HOM_ERR_UNSUPPORTED, "4-bit product: more than 2^31 - 1 output tiles");
    return false;
  }
  LaunchScope scope(kOpGemm, product_flops(pb), product_bytes(pb));
  return check_cuda(launch_pdl(gemm_mxf4_kernel, dim3(static_cast<unsigned>(tiles)), dim3(kThreads), kSmemBytes, stream,
                               1, tmA, tmB, tmSA, tmSB, tmD, p),
                    "4-bit product launch");
}

}  // namespace mxf4
}  // namespace hom
