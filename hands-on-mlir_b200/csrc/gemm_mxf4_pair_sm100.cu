// Product of two microscaled 4-bit matrices on CTA pairs: D = act(alpha * A.B^T + beta * C) for
// problems with many tiles (format: mxf4_sm100.cuh).
//
// A 256 x 256 tile belongs to a cluster of two CTAs on neighbouring SMs; each holds 128 rows of A,
// 128 rows of B and the accumulator of its 128 output rows.  The grid is persistent.  Per step of
// 256 values along K a CTA receives 32 KB of codes and 3 KB of scales (its own 128 rows of A's, all
// 256 columns of B's); four 256 x 256 x 64 MMAs consume that in 512 tensor-pipe cycles, 70 bytes
// a cycle and SM out of L2.  A 128 x 256 tile per CTA would need 103.
//
// Tensor memory is the tight resource: two accumulators fill its 512 columns, and the scales need
// 24 columns per step.  The accumulators therefore share 64 columns: the first lies in [0, 256),
// the second in [192, 448), two sets of scales behind it.  The warps that drain the shared columns
// take all 64 of them into registers at once, so the next tile's MMAs start some 300 cycles after
// the last one of this tile while the other three quarters are drained beside them.
//
// A set of scales is written for step i + 2 only when the MMAs of step i have completed: copies are
// ordered before later MMAs of the thread, but not behind earlier ones.
//
//   warp 0   TMA producer
//   warp 1   tensor memory, scale copies and MMA issue (even CTA)
//   warps 2-17  epilogue: four warps per tensor-memory lane quarter, one 64-column group each
#include "gemm_epilogue.cuh"
#include "gemm_sm100.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

using namespace hom::ptx;
using gemm::EpilogueParams;
using gemm::kEpiAddC;
using gemm::kEpiGelu;
using gemm::kEpiGeneric;
using gemm::kEpiPlain;

namespace {

constexpr int BM = 256, BN = 256, kHalf = 128;         // tile; rows of A and of B per CTA
constexpr int kStepBytes = 128;                        // of a row of codes: 256 values
constexpr int kStepBlocks = 2 * kStepBytes / kBlock;   // 8
constexpr int kStepTiles = kStepBlocks / kTileBlocks;  // 2 scale tiles along K
constexpr int kStages = 4;
constexpr int kDrainWarps = 16;
constexpr int kThreads = 32 * (2 + kDrainWarps);
constexpr uint32_t kCodeBytes = kHalf * kStepBytes;    // of one operand, per CTA and stage
constexpr uint32_t kScaleABytes = kStepTiles * kTileBytes, kScaleBBytes = 2 * kScaleABytes;
constexpr uint32_t kStageBytes = 2 * kCodeBytes + kScaleABytes + kScaleBBytes;
static_assert(kStageBytes % 1024 == 0, "swizzled tiles start on 1024 bytes");
constexpr uint32_t kStagingBytes = kDrainWarps * gemm::kEpilogueStageBytes;
constexpr int kBarriers = 2 * kStages + 5;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + kStagingBytes + 8 * kBarriers + 16 + 1024;
// tensor memory columns
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSecondAcc = 192;                   // the accumulators share [192, 256)
constexpr uint32_t kScales = kSecondAcc + BN, kScaleSet = 4 * kStepTiles * 3, kScalesB = 4 * kStepTiles;
static_assert(kScales + 2 * kScaleSet <= kTmemCols, "accumulators and scales exceed tensor memory");

struct Params {
  EpilogueParams ep;
  int steps, n_blocks, tiles;
  int b_early;  // B is a declared constant: request its first tiles before griddepcontrol.wait
  int *status;
};

// Reads 32 accumulator values of this lane's row, applies the epilogue and leaves fp16 results in
// the staging tile.
template <int EPI>
__device__ __forceinline__ void finish_half(const EpilogueParams &ep, uint32_t (&acc)[32], const uint4 *cval, int half,
                                            uint32_t my_row, int lane) {
  const float2 alpha2 = make_float2(ep.alpha, ep.alpha), beta2 = make_float2(ep.beta, ep.beta);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const __half2 *c2 = reinterpret_cast<const __half2 *>(&cval[half * 4 + g]);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * 8 + 2 * j;
      float2 v = make_float2(__uint_as_float(acc[i]), __uint_as_float(acc[i + 1]));
      if (EPI == kEpiGeneric) {
        v = __fmul2_rn(alpha2, v);
        if (ep.c_mode != 0) v = __ffma2_rn(beta2, __half22float2(c2[j]), v);
      }
      if (EPI == kEpiAddC) v = __fadd2_rn(__half22float2(c2[j]), v);
      if (EPI == kEpiGelu || (EPI == kEpiGeneric && ep.act == 1)) v = gemm::gelu_erf_fast2(v);
      const __half2 h = __floats2half2_rn(v.x, v.y);
      w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
    const uint32_t addr = my_row + ((static_cast<uint32_t>(half * 4 + g) ^ (lane & 7u)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                 : "memory");
  }
}

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1)
gemm_mxf4_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                      const __grid_constant__ CUtensorMap tmD, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t staging_base = smem_base + kStages * kStageBytes;
  const uint32_t bar_base = staging_base + kStagingBytes;
  // full (even CTA, both CTAs' bytes) and empty (both) per stage; accumulator full (both) and empty
  // (even); shared columns drained (even)
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (2 * kStages + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (2 * kStages + 2 + a); };
  const uint32_t shared_bar = bar_base + 8u * (2 * kStages + 4);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kStages * kStageBytes + kStagingBytes +
                                                                       8 * kBarriers);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0: even CTA (issues the MMAs), 1: odd CTA
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 64) {
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmSB);
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmSA);
    prefetch_tensormap(&tmD);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 2 * kDrainWarps);
    }
    mbar_init(shared_bar, 2 * 4);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();  // barriers of both CTAs are initialised before anyone signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 0) {
    // -------------------------------------------------------------- TMA producer
    if (elect_one()) {
      const uint32_t full_even = map_to_cta(full_bar(0), 0);
      auto load_b = [&](uint32_t dst, uint32_t bar, int step, int n0) {
        tma_load_2d_pair(dst + kCodeBytes, &tmB, bar, step * (kStepBytes / 2), n0 + static_cast<int>(rank) * kHalf);
        tma_load_3d_pair(dst + 2 * kCodeBytes + kScaleABytes, &tmSB, bar, 0, step * kStepTiles, n0 / kTileRows);
      };
      auto load_a = [&](uint32_t dst, uint32_t bar, int step, int m0) {
        tma_load_2d_pair(dst, &tmA, bar, step * (kStepBytes / 2), m0);
        tma_load_3d_pair(dst + 2 * kCodeBytes, &tmSA, bar, 0, step * kStepTiles, m0 / kTileRows);
      };
      // The first ring: a declared B does not depend on the previous kernel.
      int early = 0;
      if (pair < p.tiles) {
        early = min(kStages, p.steps);
        for (int i = 0; i < early; ++i) {
          if (rank == 0) mbar_arrive_expect_tx(full_bar(i), 2 * kStageBytes);
          if (p.b_early) load_b(smem_base + i * kStageBytes, full_even + 8 * i, i, pair % p.n_blocks * BN);
        }
      }
      pdl_wait();
      uint32_t slot = 0, ph = 0;
      bool ok = true;
      for (int tile = pair; tile < p.tiles && ok; tile += num_pairs) {
        const int m0 = tile / p.n_blocks * BM + static_cast<int>(rank) * kHalf, n0 = tile % p.n_blocks * BN;
        for (int i = 0; i < p.steps; ++i) {
          const uint32_t dst = smem_base + slot * kStageBytes, bar = full_even + 8 * slot;
          if (early > 0) {
            --early;
            if (!p.b_early) load_b(dst, bar, i, n0);
          } else {
            ok = mbar_wait(empty_bar(slot), ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
            if (!ok) break;
            if (rank == 0) mbar_arrive_expect_tx(full_bar(slot), 2 * kStageBytes);
            load_b(dst, bar, i, n0);
          }
          load_a(dst, bar, i, m0);
          if (++slot == kStages) {
            slot = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok) {
        // gives copies already in flight time to land (about 2 ms)
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (even CTA only)
    if (rank == 0 && elect_one()) {
      uint32_t slot = 0, ph = 0;
      bool ok = true;
      uint32_t step = 0;  // over all tiles
      int it = 0;
      for (int tile = pair; tile < p.tiles && ok; tile += num_pairs, ++it) {
        const int acc = it & 1;
        ok = mbar_wait(acc_empty_bar(acc), ((it >> 1) & 1) ^ 1, abort_flag, p.status, kDevWaitTimeoutMma);
        if (ok && it > 0) ok = mbar_wait(shared_bar, (it - 1) & 1, abort_flag, p.status, kDevWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + (acc ? kSecondAcc : 0);
        for (int i = 0; i < p.steps; ++i, ++step) {
          // the MMAs that read this set of scales two steps ago have completed
          if (step >= 2)
            ok = mbar_wait(empty_bar((step - 2) % kStages), ((step - 2) / kStages) & 1, abort_flag, p.status,
                           kDevWaitTimeoutMma);
          if (ok) ok = mbar_wait(full_bar(slot), ph, abort_flag, p.status, kDevWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t src = smem_base + slot * kStageBytes, src_scales = src + 2 * kCodeBytes;
          const uint32_t scales = tmem_base + kScales + (step & 1) * kScaleSet;
#pragma unroll
          for (int k = 0; k < kStepTiles; ++k) {
            tc_copy_scales_pair(scales + 4 * k, make_smem_desc_scales(src_scales + k * kTileBytes));
#pragma unroll
            for (int n = 0; n < BN / kTileRows; ++n)
              tc_copy_scales_pair(scales + kScalesB + 4 * (k * (BN / kTileRows) + n),
                                  make_smem_desc_scales(src_scales + kScaleABytes + (n * kStepTiles + k) * kTileBytes));
          }
          const uint64_t da = make_smem_desc_sw128(src, 16, 1024);
          const uint64_t db = make_smem_desc_sw128(src + kCodeBytes, 16, 1024);
#pragma unroll
          for (int k = 0; k < 2 * kStepTiles; ++k)
            tc_mma_mxf4_ss_pair(d_tmem, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32),
                                k & 1 ? make_idesc_mxf4(BM, BN, 1) : make_idesc_mxf4(BM, BN, 0), scales + 4 * (k >> 1),
                                scales + kScalesB + 4 * (k >> 1) * (BN / kTileRows), i != 0 || k != 0 ? 1u : 0u);
          tc_commit_pair(empty_bar(slot), 0x3);  // frees the stage in both CTAs
          if (++slot == kStages) {
            slot = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit_pair(acc_full_bar(acc), 0x3);
      }
    }
    __syncwarp();
  } else {
    // --------------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    const int group = (warp - 2) >> 2;
    const uint32_t stage_smem = staging_base + (warp - 2) * gemm::kEpilogueStageBytes;
    const uint32_t my_row = stage_smem + lane * 128;
    auto arrive_even = [&](uint32_t bar) {
      if (lane == 0) {
        if (rank == 0) mbar_arrive(bar);
        else mbar_arrive_cluster(map_to_cta(bar, 0));
      }
    };
    pdl_wait();  // C may be produced, and D still read, by the previous kernel
    int it = 0;
    for (int tile = pair; tile < p.tiles; tile += num_pairs, ++it) {
      const int acc = it & 1;
      const int row0 = tile / p.n_blocks * BM + static_cast<int>(rank) * kHalf + quarter * 32;
      const int c0 = tile % p.n_blocks * BN + group * 64;
      // the columns that the other accumulator shares: the first one's last group, the second one's first
      const bool shares = group == (acc ? 0 : 3);
      constexpr bool kReadsC = EPI == kEpiAddC || EPI == kEpiGeneric;
      uint4 cval[8];
      if (kReadsC) {
        if (shares) gemm::epilogue_load_c<0, 4, true>(p.ep, row0 + lane, c0, cval);
        else gemm::epilogue_load_c<0, 8, true>(p.ep, row0 + lane, c0, cval);
      }
      bool ok = mbar_wait(acc_full_bar(acc), (it >> 1) & 1, abort_flag, p.status, kDevWaitTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (acc ? kSecondAcc : 0) + group * 64;
      // The staging tile was handed to TMA by this warp's previous block: that read must be over.
      auto staging_free = [&]() {
        if (lane == 0) bulk_wait_group_read_0();
        __syncwarp();
      };
      auto drained = [&]() {
        tc_fence_before_sync();
        __syncwarp();
      };
      // two copies of the arithmetic: only the shared columns' warps hold 64 accumulators at once,
      // and they ask for the second half of C when the first half's registers are free
      if (shares) {
        uint32_t lo[32], hi[32];
        tmem_ld_32x32(t_row, lo);
        tmem_ld_32x32(t_row + 32, hi);
        tmem_ld_wait();
        drained();
        arrive_even(shared_bar);
        arrive_even(acc_empty_bar(acc));
        staging_free();
        finish_half<EPI>(p.ep, lo, cval, 0, my_row, lane);
        if (kReadsC) gemm::epilogue_load_c<4, 8, true>(p.ep, row0 + lane, c0, cval);
        finish_half<EPI>(p.ep, hi, cval, 1, my_row, lane);
      } else {
        uint32_t v[32];
        tmem_ld_32x32(t_row, v);
        tmem_ld_wait();
        staging_free();
        finish_half<EPI>(p.ep, v, cval, 0, my_row, lane);
        tmem_ld_32x32(t_row + 32, v);
        tmem_ld_wait();
        drained();
        arrive_even(acc_empty_bar(acc));
        finish_half<EPI>(p.ep, v, cval, 1, my_row, lane);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (c0 < p.ep.N && row0 < p.ep.M) tma_store_2d(&tmD, stage_smem, c0, row0);
        bulk_commit_group();
      }
    }
    if (lane == 0) bulk_wait_group_read_0();
    __syncwarp();
  }

  // Nobody leaves while the other CTA may still read this CTA's shared memory or signal its barriers.
  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace

bool run_product_pair(const Problem &pb, cudaStream_t stream) {
  auto kernel = gemm_mxf4_pair_kernel<kEpiGeneric>;
  if (pb.alpha == 1.f) {
    if (pb.c_mode == 0) kernel = pb.act ? gemm_mxf4_pair_kernel<kEpiGelu> : gemm_mxf4_pair_kernel<kEpiPlain>;
    else if (pb.beta == 1.f && !pb.act) kernel = gemm_mxf4_pair_kernel<kEpiAddC>;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  static int max_pairs[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (max_pairs[dev] == 0) {
    for (auto k : {gemm_mxf4_pair_kernel<kEpiGeneric>, gemm_mxf4_pair_kernel<kEpiPlain>, gemm_mxf4_pair_kernel<kEpiGelu>,
                   gemm_mxf4_pair_kernel<kEpiAddC>})
      if (!check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes),
                      "cudaFuncSetAttribute(4-bit product on pairs)"))
        return false;
    // How many CTA pairs the device can hold at once (pairs need neighbouring SMs).
    cfg.gridDim = dim3(2 * (sm_count() / 2));
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sm_count() / 2;
    }
    max_pairs[dev] = n;
  }
  const int64_t pitch = pb.blocks * 8;  // in two-byte elements, what the tensor maps count in
  const int64_t tile_cols = tile_cols_of(pb.blocks);
  CUtensorMap tmA, tmB, tmSA, tmSB, tmD;
  if (!gemm::make_tensor_map_2d(pb.A, pitch, pb.M, kStepBytes / 2, kHalf, &tmA) ||
      !gemm::make_tensor_map_2d(pb.B, pitch, pb.N, kStepBytes / 2, kHalf, &tmB) ||
      !gemm::make_tensor_map_scales(pb.scales_a, tile_cols, tile_rows_of(pb.M), kStepTiles, 1, &tmSA) ||
      !gemm::make_tensor_map_scales(pb.scales_b, tile_cols, tile_rows_of(pb.N), kStepTiles, BN / kTileRows, &tmSB) ||
      !gemm::make_tensor_map_2d(pb.D, pb.N, pb.M, 64, 32, &tmD))
    return false;
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
  p.steps = static_cast<int>((pb.blocks + kStepBlocks - 1) / kStepBlocks);
  p.n_blocks = static_cast<int>((pb.N + BN - 1) / BN);
  p.b_early = pb.b_const ? 1 : 0;
  p.status = device_status_word();
  const int64_t tiles = (pb.M + BM - 1) / BM * p.n_blocks;
  if (tiles > INT32_MAX) {
    set_error(HOM_ERR_UNSUPPORTED, "4-bit product: more than 2^31 - 1 output tiles");
    return false;
  }
  p.tiles = static_cast<int>(tiles);
  cfg.gridDim = dim3(2 * (p.tiles < max_pairs[dev] ? p.tiles : max_pairs[dev]));
  LaunchScope scope(kOpGemm, product_flops(pb), product_bytes(pb));
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmSA, tmSB, tmD, p), "4-bit product launch (CTA pairs)");
}

}  // namespace mxf4
}  // namespace hom
