// fp16 GEMM family for sm_100a: D = epilogue(alpha * A.B + beta * C), fp32 accumulate in
// tensor memory, Row,Row,Row operands (B as [K,N]) or the "transb" form (B as [N,K]).
//
// One persistent CTA per SM walks a static list of work units: a 128 x BN output tile, or one
// of the `split_k` K ranges of a tile.  Inside a CTA (608 threads):
//   warps 0, 2  TMA producers: 128x64 A box / BN x 64 B boxes per K block into a ring of
//               128-byte-swizzled shared-memory stages (mbarrier full/empty hand-off);
//   warp 1      issues tcgen05.mma (M=128, N=BN, K=16) into one of two TMEM accumulators and
//               releases stages / publishes accumulators with tcgen05.commit;
//   warps 3-18  epilogue (four warps per tensor-memory lane quarter, one 64-column group of
//               the tile each): tcgen05.ld the finished accumulator (one output row per
//               thread, 32 columns at a time), fp32 alpha/beta/bias/erf-GELU, one fp16
//               rounding, results staged in swizzled shared memory and written out by TMA
//               stores, while warp 1 already fills the other accumulator.  The units of a split
//               tile are reduced serially through an fp32 workspace (SplitK, gemm_epilogue.cuh).
//
// This replaces the reference's CUTLASS 2.x mma.sync kernels and its compile-time autotuner
// (include/NVGPUKernels/GemmRunner.h:119-310, lib/NVGPUKernels/GemmProfiler.cu:143-236) with six
// tile shapes, an estimate of their times that picks one, and a tuner whose choices come first.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstdio>
#include <tuple>
#include <map>
#include <cstring>
#include <mutex>
#include <unordered_map>

#include "gemm_epilogue.cuh"
#include "gemm_sm100.cuh"
#include "hom_diag.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace gemm {

using namespace hom::ptx;

namespace {

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int kThreads = 32 * (kControlWarps + kEpilogueWarps);
constexpr uint32_t kABytes = BM * BK * 2;

template <int BN>
struct TileCfg {
  static constexpr uint32_t kBBytes = BN * BK * 2;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  // As many stages as fit beside the epilogue staging of the tile's BN / 64 column groups.
  static constexpr int kStages = BN == 256 ? 3 : BN == 192 ? 4 : BN == 128 ? 6 : 8;
  static constexpr uint32_t kTmemCols = BN == 64 ? 128 : BN == 128 ? 256 : 512;
  static constexpr uint32_t kStagingBytes = BN / 64 * 4 * kEpilogueStageBytes;
  static constexpr uint32_t kBarrierBytes = 8 * (2 * kStages + 4) + 16;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarrierBytes + 1024;
};

struct Params {
  EpilogueParams ep;
  int K;
  int n_blocks, num_tiles, num_kb;
  int b_grouped;  // B [K,N] is fetched through the grouped 3-D tensor map (N % 64 == 0)
  int b_early;    // B is a declared constant: request its first tiles before griddepcontrol.wait
  // Split-K: every tile is cut into `split_k` work units (K-block ranges); num_units = num_tiles
  // * split_k.  Workspace: per (tile, epilogue warp) `split_k` fp32 slots and a pair of counters
  // (see SplitK in gemm_epilogue.cuh).
  int split_k, num_units;
  float *ws_slots;
  int *ws_counters;
  int *status;
  HOM_DIAG(long long *prof;)  // optional per-role cycle counters of CTA 0, else null
  HOM_DIAG(long long *tl;)    // optional launch-timeline slot, else null
  // fused LayerNorm over the output rows (LN kernels only): grid = tiles, one cluster per 128 rows
  float ln_eps, ln_inv_n;
  int ln_cluster;
};

// After an expired wait: gives copies already in flight time to land (about 2 ms) before the
// CTA's shared memory is released.
__device__ __forceinline__ void drain_copies() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000LL) {
  }
}

template <int BN, bool B_NK, bool LN = false, bool SPLIT = false, int FORMS = 0, int EPI = 0>
__global__ void __launch_bounds__(kThreads, 1)
gemm_f16_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmD, const Params p) {
  using Cfg = TileCfg<BN>;
  constexpr int STAGES = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);

  const uint32_t staging_base = smem_base + STAGES * Cfg::kStageBytes;
  const uint32_t bar_base = staging_base + Cfg::kStagingBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
  volatile uint32_t *tmem_slot =
      reinterpret_cast<volatile uint32_t *>(smem_gen + STAGES * Cfg::kStageBytes + Cfg::kStagingBytes +
                                            8 * (2 * STAGES + 4));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  HOM_DIAG(const long long t_entry = p.prof ? clock64() : 0; unsigned long long g_entry = 0;
           if (p.prof) asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(g_entry));
           if (p.tl && threadIdx.x == 0) timeline_stamp(p.tl, 0);)
  // The first TMA instruction stalls until its descriptor has been fetched: start those
  // fetches before anything else so that they overlap the barrier and tensor-memory set-up.
  if (threadIdx.x == 64) {
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmD);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kEpilogueWarps);  // one arrival per epilogue warp
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // Dependents may be scheduled from here on: every CTA of this grid that reaches this point
  // already holds its tensor-memory columns, so a dependent CTA that becomes co-resident and
  // allocates its own columns can never starve one of ours.
  pdl_launch_dependents();
  HOM_DIAG(if (p.prof && blockIdx.x == 0 && threadIdx.x == 0) p.prof[10] = clock64() - t_entry;)

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer, A
    // One elected lane runs the whole loop (see the MMA issuer).  A and B come from two warps: one
    // thread that waits, arms and issues both copies needs about 280 clk per K block, more than
    // the tensor pipe takes for a tile up to 128 columns wide.
    if (elect_one()) {
      // A chain of dependent instructions of one thread: addresses advance by additions.
      uint32_t dst = smem_base, bar = full_bar(0), ph = 0;
      bool ok = true;
      HOM_DIAG(long long t_wait = 0; const long long t_begin = clock64();)
      auto advance = [&]() {
        dst += Cfg::kStageBytes;
        bar += 8;
        if (bar == full_bar(STAGES)) {
          dst = smem_base;
          bar = full_bar(0);
          ph ^= 1u;
        }
      };
      // The first ring is armed (for the bytes of both copies) before the wait for the previous
      // kernel, so that only the copies themselves are left to do after it.
      int ready = 0;
      if (blockIdx.x < p.num_units) {
        const int part0 = blockIdx.x % p.split_k;
        ready = min(STAGES, (part0 + 1) * p.num_kb / p.split_k - part0 * p.num_kb / p.split_k);
        for (int i = 0; i < ready; ++i) mbar_arrive_expect_tx(full_bar(i), Cfg::kStageBytes);
      }
      pdl_wait();
      HOM_DIAG(if (p.tl) timeline_stamp(p.tl, 2);)
      for (int unit = blockIdx.x; unit < p.num_units && ok; unit += gridDim.x) {
        const int tile = unit / p.split_k, part = unit % p.split_k;
        const int m0 = (tile / p.n_blocks) * BM;
        const int k_end = (part + 1) * p.num_kb / p.split_k * BK;
        int k = part * p.num_kb / p.split_k * BK;
        for (; ready > 0; --ready, k += BK) {
          tma_load_2d(dst, &tmA, bar, k, m0);
          advance();
        }
        for (; k < k_end; k += BK) {
          HOM_DIAG(const long long tw = p.prof ? clock64() : 0;)
          ok = mbar_wait(bar + 8u * STAGES, ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
          if (!ok) break;
          HOM_DIAG(if (p.prof) t_wait += clock64() - tw;)
          mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
          tma_load_2d(dst, &tmA, bar, k, m0);
          advance();
        }
      }
      HOM_DIAG(if (p.prof && blockIdx.x == 0) {
        p.prof[0] = clock64() - t_begin;
        p.prof[1] = t_wait;
      })
      if (!ok) drain_copies();
    }
    __syncwarp();
    if constexpr (LN) cluster_sync_all();  // the epilogue's statistics exchange counts every thread
  } else if (warp == 2) {
    // ------------------------------------------------------------ TMA producer, B
    if (elect_one()) {
      uint32_t dst = smem_base + kABytes, bar = full_bar(0), ph = 0;
      bool ok = true;
      const bool b_grouped = p.b_grouped != 0;
      // A declared constant (weights, which no kernel of the stream writes) is requested without
      // waiting for the previous kernel: the first ring of B tiles then arrives while that one
      // finishes.  A B of unknown origin only after.  (Its bytes may land before the A warp has
      // armed the barrier: the phase cannot complete without that arrival.)  The ring's stages are
      // free the first time round, so that no limited wait comes before the one for that kernel.
      bool early = p.b_early != 0;
      if (!early) pdl_wait();
      for (int unit = blockIdx.x; unit < p.num_units && ok; unit += gridDim.x) {
        const int tile = unit / p.split_k, part = unit % p.split_k;
        const int n0 = (tile % p.n_blocks) * BN;
        const int k_end = (part + 1) * p.num_kb / p.split_k * BK;
        for (int k = part * p.num_kb / p.split_k * BK; k < k_end; k += BK) {
          ok = mbar_wait(bar + 8u * STAGES, ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
          if (!ok) break;
          if (B_NK) {
            tma_load_2d(dst, &tmB, bar, k, n0);
          } else if (b_grouped) {
            tma_load_3d(dst, &tmB, bar, 0, k, n0 / 64);
          } else {
#pragma unroll
            for (int g = 0; g < BN / 64; ++g) tma_load_2d(dst + g * (BK * 128), &tmB, bar, n0 + g * 64, k);
          }
          dst += Cfg::kStageBytes;
          bar += 8;
          if (bar == full_bar(STAGES)) {
            dst = smem_base + kABytes;
            bar = full_bar(0);
            ph ^= 1u;
            if (early) {
              pdl_wait();
              early = false;
            }
          }
        }
      }
      if (!ok) drain_copies();
    }
    __syncwarp();
    if constexpr (LN) cluster_sync_all();
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issuer
    // One lane, elected once by elect.sync around the whole loop: the compiler then knows that a
    // single thread runs it, and a K block costs the tensor pipe's time.  A loop of the whole warp
    // with only the issue under the election spends 415-435 clk per 64-deep K block on votes,
    // reconvergence and re-election, whatever the tile's width; this form 267 / 296 / 401 clk at
    // N = 64 / 128 / 192, where the pipe itself needs 192 / 256 / 384.
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_f16(BM, BN, false, !B_NK);
      // A: K-major rows of 128 B; 8-row groups 1024 B apart; 16 K elements = 32 B.
      // B as [N,K]: same as A.  B as [K,N] (N contiguous): 64-column groups are separate
      // sub-tiles BK*128 B apart, 8-row K groups 1024 B apart, and 16 K rows = 2048 B.
      const uint64_t da0 = make_smem_desc_sw128(smem_base, 16, 1024);
      const uint64_t db0 = make_smem_desc_sw128(smem_base + kABytes, B_NK ? 16 : BK * 128, 1024);
      uint64_t da = da0, db = db0;
      uint32_t bar = full_bar(0), ph = 0;
      bool ok = true;
      int it = 0;
      HOM_DIAG(long long t_full = 0, t_acc = 0; const long long t_begin = clock64();)
      for (int unit = blockIdx.x; unit < p.num_units && ok; unit += gridDim.x, ++it) {
        const int part = unit % p.split_k;
        const int num_kb = (part + 1) * p.num_kb / p.split_k - part * p.num_kb / p.split_k;
        const int acc = it & 1;
        const uint32_t acc_ph = (it >> 1) & 1;
        HOM_DIAG(const long long ta = p.prof ? clock64() : 0;)
        ok = mbar_wait(tempty_bar(acc), acc_ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutMma);
        if (!ok) break;
        HOM_DIAG(if (p.prof) t_acc += clock64() - ta;)
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          HOM_DIAG(const long long tw = p.prof ? clock64() : 0;)
          ok = mbar_wait<true>(bar, ph, abort_flag, p.status, kDevWaitTimeoutMma);
          if (!ok) break;
          HOM_DIAG(if (p.prof) t_full += clock64() - tw;)
          tc_fence_after_sync();
          tc_mma_f16_ss(d_tmem, da, db, idesc, kb != 0 ? 1u : 0u);
#pragma unroll
          for (int k = 1; k < BK / 16; ++k)
            tc_mma_f16_ss(d_tmem, smem_desc_advance(da, k * 32), smem_desc_advance(db, B_NK ? k * 32 : k * 2048),
                          idesc, 1u);
          tc_commit(bar + 8u * STAGES);  // frees the stage
          da = smem_desc_advance(da, Cfg::kStageBytes);
          db = smem_desc_advance(db, Cfg::kStageBytes);
          bar += 8;
          if (bar == full_bar(STAGES)) {
            da = da0;
            db = db0;
            bar = full_bar(0);
            ph ^= 1u;
          }
        }
        if (ok) tc_commit(tfull_bar(acc));
      }
      HOM_DIAG(if (p.prof && blockIdx.x == 0) {
        p.prof[2] = clock64() - t_begin;
        p.prof[3] = t_full;
        p.prof[4] = t_acc;
      })
    }
    __syncwarp();
    if constexpr (LN) cluster_sync_all();  // the epilogue's statistics exchange counts every thread
  } else {
    // --------------------------------------------------------------- epilogue
    const int quarter = warp & 3;       // TMEM lanes [32*quarter, 32*quarter + 32)
    const int group = (warp - kControlWarps) >> 2;  // which 64-column group of the tile
    const int col_begin = group * 64;
    const bool active = col_begin < BN;
    const uint32_t stage_smem = staging_base + (warp - kControlWarps) * kEpilogueStageBytes;
    int it = 0;
    bool ln_done = false;
    HOM_DIAG(long long t_wait = 0; const long long t_begin = clock64();)
    pdl_wait();  // C may be produced, and D still read, by the previous kernel
    float2 next_col_sums = make_float2(0.f, 0.f);
    if constexpr ((FORMS & kFormLnA) != 0) {
      if (active && static_cast<int>(blockIdx.x) < p.num_units)
        next_col_sums = epilogue_load_col_sums(p.ep, (static_cast<int>(blockIdx.x) % p.n_blocks) * BN + col_begin, lane);
    }
    for (int unit = blockIdx.x; unit < p.num_units; unit += gridDim.x, ++it) {
      const int tile = unit / p.split_k;
      const int acc = it & 1;
      const uint32_t acc_ph = (it >> 1) & 1;
      const int m0 = (tile / p.n_blocks) * BM;
      const int n0 = (tile % p.n_blocks) * BN;
      uint4 cval[8];
      SplitK sk;
      if constexpr (SPLIT) {
        // this warp's block of the tile: (tile, epilogue warp)
        const size_t block = static_cast<size_t>(tile) * kEpilogueWarps + (warp - kControlWarps);
        sk.parts = p.split_k;
        sk.part = unit % p.split_k;
        sk.slot = p.ws_slots + block * kSplitSlotFloats;
        sk.counter = p.ws_counters + block;
      } else {
        if constexpr (EPI == kEpiGeneric || EPI == kEpiAddC) {
          if (active) epilogue_load_c<0, 8, EPI != kEpiGeneric || FORMS != 0>(p.ep, m0 + quarter * 32 + lane, n0 + col_begin, cval);
        }
      }
      RowAffine ra;
      float2 col_sums = make_float2(0.f, 0.f);
      if constexpr ((FORMS & (kFormLnA | kFormLnR)) != 0) {
        if (active) ra = epilogue_row_affine(p.ep, m0 + quarter * 32 + lane);
      }
      if constexpr ((FORMS & kFormLnA) != 0) {
        col_sums = next_col_sums;
        const int next = unit + gridDim.x;
        if (active && next < p.num_units)
          next_col_sums = epilogue_load_col_sums(p.ep, (next % p.n_blocks) * BN + col_begin, lane);
      }
      HOM_DIAG(const long long tw = p.prof ? clock64() : 0;)
      bool ok = mbar_wait(tfull_bar(acc), acc_ph, abort_flag, p.status, kDevWaitTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      HOM_DIAG(if (p.prof) t_wait += clock64() - tw;)
      tc_fence_after_sync();
      const uint32_t t_row =
          tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * BN + col_begin;
      if constexpr (LN) {
        // one tile per CTA; the pipeline stages are idle by now and stage 0 holds the statistics
        LayernormFusion ln;
        ln.stats_smem = smem_base;
        ln.cluster_n = p.ln_cluster;
        ln.row_in_tile = quarter * 32 + lane;
        ln.group = group;
        ln.eps = p.ln_eps;
        ln.inv_n = p.ln_inv_n;
        epilogue_warp_block_ln(p.ep, &tmD, t_row, m0 + quarter * 32, n0 + col_begin, active, stage_smem,
                               lane, cval, ln);
        ln_done = true;
      } else {
        if (!epilogue_warp_block<SPLIT, FORMS, EPI>(p.ep, &tmD, t_row, m0 + quarter * 32, n0 + col_begin, active,
                                               stage_smem, lane, cval, [&]() {
                                                 if (lane == 0) mbar_arrive(tempty_bar(acc));
                                               }, sk, abort_flag, p.status, ra, col_sums))
          break;
      }
    }
    if constexpr (LN) {
      if (!ln_done) {  // error path: keep the named barrier's and the cluster barrier's counts whole
        asm volatile("bar.sync 1, 512;" ::: "memory");
        cluster_sync_all();
      }
    }
    // A store still in flight reads this warp's staging tile: let it finish reading.
    if (lane == 0) bulk_wait_group_read_0();
    __syncwarp();
    HOM_DIAG(if (p.prof && blockIdx.x == 0 && threadIdx.x == 32 * kControlWarps) {
      p.prof[5] = clock64() - t_begin;
      p.prof[6] = t_wait;
    })
  }

  tc_fence_before_sync();
  if constexpr (LN) cluster_sync_all();  // peers may still be reading this CTA's statistics
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
  HOM_DIAG(if (p.tl && threadIdx.x == 0) timeline_stamp(p.tl, 4);
           if (p.prof && blockIdx.x == 0 && threadIdx.x == 32) {
             unsigned long long g_exit;
             asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(g_exit));
             p.prof[11] = clock64() - t_entry;
             p.prof[12] = static_cast<long long>(g_entry);
             p.prof[13] = static_cast<long long>(g_exit);
             // ring of (entry, exit) wall-clock stamps of the last launches
             const long long slot = p.prof[15] & 15;
             p.prof[16 + 2 * slot] = static_cast<long long>(g_entry);
             p.prof[17 + 2 * slot] = static_cast<long long>(g_exit);
             p.prof[15] += 1;
           })
}

// ------------------------------------------------------------------ host side

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                              const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn get_encode_fn() {
  static EncodeFn fn = []() -> EncodeFn {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &sym, 12000, cudaEnableDefault,
                                         &qres) != cudaSuccess ||
        qres != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeFn>(sym);
  }();
  return fn;
}

struct MapKey {
  const void *ptr;
  uint64_t inner, outer;
  uint32_t box_inner, box_outer;  // box_outer | groups << 16 for the grouped 3-D form
  uint64_t pitch;                 // row pitch in elements (== inner unless the rows are padded)
  bool operator==(const MapKey &o) const {
    return ptr == o.ptr && inner == o.inner && outer == o.outer && box_inner == o.box_inner &&
           box_outer == o.box_outer && pitch == o.pitch;
  }
};
struct MapKeyHash {
  size_t operator()(const MapKey &k) const {
    size_t h = reinterpret_cast<size_t>(k.ptr);
    h = h * 1000003u ^ k.inner;
    h = h * 1000003u ^ k.outer;
    h = h * 1000003u ^ (static_cast<size_t>(k.box_inner) << 16 | k.box_outer);
    h = h * 1000003u ^ k.pitch;
    return h;
  }
};

std::mutex g_map_mutex;
std::unordered_map<MapKey, CUtensorMap, MapKeyHash> g_map_cache;

}  // namespace

#if HOM_DIAG_ENABLED
// Diagnostics (HOM_GEMM_PROFILE=1): a small device buffer the kernels fill with per-role
// cycle counters of CTA 0, printed after a stream synchronisation.  Never on by default.
static long long *g_profile_buf = nullptr;

long long *profile_buffer() {
  static bool checked = false;
  if (!checked) {
    checked = true;
    if (std::getenv("HOM_GEMM_PROFILE") || std::getenv("HOM_ATTN_PROFILE")) {
      if (cudaMalloc(&g_profile_buf, 4096 * sizeof(long long)) != cudaSuccess) g_profile_buf = nullptr;
      else {
        cudaMemset(g_profile_buf, 0, 4096 * sizeof(long long));
        // slots [32, 64): {first entry, last entry, first exit, last exit} of eight launches
        long long init[32];
        for (int i = 0; i < 32; ++i) init[i] = (i & 1) == 0 ? 0x7fffffffffffffffLL : 0;
        cudaMemcpy(g_profile_buf + 32, init, sizeof(init), cudaMemcpyHostToDevice);
        // slots [3000, 3480): {first, last} x {entry, dependency resolved, exit, first MMA issued,
        // last accumulator complete} of 48 GEMM launches
        long long init2[480];
        for (int i = 0; i < 480; ++i) init2[i] = (i & 1) == 0 ? 0x7fffffffffffffffLL : 0;
        cudaMemcpy(g_profile_buf + 3000, init2, sizeof(init2), cudaMemcpyHostToDevice);
      }
    }
  }
  // The role counters are only collected while one of the variables is (still) set, so that a
  // program can switch them off before it captures a graph.
  if (!g_profile_buf || !(std::getenv("HOM_GEMM_PROFILE") || std::getenv("HOM_ATTN_PROFILE"))) return nullptr;
  if (!std::getenv("HOM_GEMM_TIMELINE")) cudaMemset(g_profile_buf, 0, 15 * sizeof(long long));
  return g_profile_buf;
}

long long *profile_buffer_raw() { return g_profile_buf; }

// Launch timeline (HOM_GEMM_LAUNCH_TIMELINE set while the calls are made, e.g. during graph
// capture): the slot this launch stamps, or null.
long long *launch_timeline_slot() {
  static int calls = 0;
  if (!g_profile_buf || !std::getenv("HOM_GEMM_LAUNCH_TIMELINE")) return nullptr;
  return g_profile_buf + 3000 + 10 * (calls++ % 48);
}

void profile_report(const char *what, int tiles, int grid, int num_kb, cudaStream_t stream) {
  if (std::getenv("HOM_GEMM_TIMELINE")) return;  // stamps are read back by the caller
  long long h[16];
  cudaStreamSynchronize(stream);
  cudaMemcpy(h, g_profile_buf, sizeof(h), cudaMemcpyDeviceToHost);
  fprintf(stderr,
          "[hom] %s tiles %d grid %d kblocks %d | producer total %lld wait-empty %lld | mma total %lld "
          "wait-full %lld wait-acc %lld | epilogue total %lld wait-full %lld | odd-CTA producer total "
          "%lld wait-empty %lld | setup %lld kernel %lld cycles, entry %lld ns, exit-entry %lld ns\n",
          what, tiles, grid, num_kb, h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[8], h[9], h[10], h[11],
          h[12], h[13] - h[12]);
}
#endif  // HOM_DIAG_ENABLED

// 2-D fp16 tensor [outer, inner] (inner contiguous, rows `pitch` elements apart; 0 = inner),
// 128-byte swizzle, zero fill.
bool make_tensor_map_2d(const void *ptr, uint64_t inner, uint64_t outer, uint32_t box_inner,
                        uint32_t box_outer, CUtensorMap *out, uint64_t pitch) {
  if (pitch == 0) pitch = inner;
  MapKey key{ptr, inner, outer, box_inner, box_outer, pitch};
  {
    std::lock_guard<std::mutex> lock(g_map_mutex);
    auto it = g_map_cache.find(key);
    if (it != g_map_cache.end()) {
      *out = it->second;
      return true;
    }
  }
  EncodeFn encode = get_encode_fn();
  if (!encode) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return false;
  }
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {pitch * 2};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t elem_strides[2] = {1, 1};
  CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(ptr), dims,
                      strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for [%llu x %llu] box [%u x %u]",
              static_cast<int>(r), static_cast<unsigned long long>(outer),
              static_cast<unsigned long long>(inner), box_outer, box_inner);
    return false;
  }
  std::lock_guard<std::mutex> lock(g_map_mutex);
  if (g_map_cache.size() > 8192) g_map_cache.clear();
  g_map_cache.emplace(key, *out);
  return true;
}

bool make_tensor_map_scales(const void *ptr, uint64_t tile_cols, uint64_t tile_rows, uint32_t box_cols,
                            uint32_t box_rows, CUtensorMap *out) {
  MapKey key{ptr, tile_cols, tile_rows, box_cols | 0x40000000u, box_rows, 0};
  {
    std::lock_guard<std::mutex> lock(g_map_mutex);
    auto it = g_map_cache.find(key);
    if (it != g_map_cache.end()) {
      *out = it->second;
      return true;
    }
  }
  EncodeFn encode = get_encode_fn();
  if (!encode) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return false;
  }
  cuuint64_t dims[3] = {256, tile_cols, tile_rows};  // in two-byte elements
  cuuint64_t strides[2] = {512, tile_cols * 512};
  cuuint32_t box[3] = {256, box_cols, box_rows};
  cuuint32_t elem_strides[3] = {1, 1, 1};
  CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(ptr), dims, strides, box,
                      elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed (%d) for [%llu x %llu] tiles",
              static_cast<int>(r), static_cast<unsigned long long>(tile_rows),
              static_cast<unsigned long long>(tile_cols));
    return false;
  }
  std::lock_guard<std::mutex> lock(g_map_mutex);
  if (g_map_cache.size() > 8192) g_map_cache.clear();
  g_map_cache.emplace(key, *out);
  return true;
}

// Row-major fp16 matrix [rows, cols] with cols % 64 == 0, seen as a 3-D tensor
// (64 columns, rows, cols / 64 column groups): one box of (64, box_rows, groups) lands in
// shared memory as `groups` consecutive 128-byte-swizzled [box_rows x 64] sub-tiles, so one
// TMA instruction fetches what would otherwise take one 2-D load per 64-column group.
bool make_tensor_map_grouped(const void *ptr, uint64_t cols, uint64_t rows, uint32_t box_rows,
                             uint32_t groups, CUtensorMap *out) {
  MapKey key{ptr, cols, rows, 64u | 0x80000000u, box_rows | (groups << 16), cols};
  {
    std::lock_guard<std::mutex> lock(g_map_mutex);
    auto it = g_map_cache.find(key);
    if (it != g_map_cache.end()) {
      *out = it->second;
      return true;
    }
  }
  EncodeFn encode = get_encode_fn();
  if (!encode) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return false;
  }
  cuuint64_t dims[3] = {64, rows, cols / 64};
  cuuint64_t strides[2] = {cols * 2, 128};
  cuuint32_t box[3] = {64, box_rows, groups};
  cuuint32_t elem_strides[3] = {1, 1, 1};
  CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(ptr), dims,
                      strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled (grouped) failed (%d) for [%llu x %llu]",
              static_cast<int>(r), static_cast<unsigned long long>(rows),
              static_cast<unsigned long long>(cols));
    return false;
  }
  std::lock_guard<std::mutex> lock(g_map_mutex);
  if (g_map_cache.size() > 8192) g_map_cache.clear();
  g_map_cache.emplace(key, *out);
  return true;
}

namespace {

// Splits a tile's K blocks into at most `want` parts of at least one block each.
int clamp_split(int want, int num_kb) {
  int s = want < 1 ? 1 : want;
  if (s > 16) s = 16;
  if (s > num_kb) s = num_kb;
  return s;
}

template <int BN, bool B_NK>
bool launch_variant(const Problem &pb, int split_k, cudaStream_t stream) {
  using Cfg = TileCfg<BN>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  // the whole-K kernel without LayerNorm forms: generic, or one of the three specialised epilogues
  const int epi = epilogue_kind(pb);
  auto kernel = epi == kEpiPlain  ? gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiPlain>
                : epi == kEpiGelu ? gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiGelu>
                : epi == kEpiAddC ? gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiAddC>
                                  : gemm_f16_kernel<BN, B_NK>;
  auto kernel_split = gemm_f16_kernel<BN, B_NK, false, true>;
  // the LayerNorm forms of the epilogue: on A only / on the residual + statistics / any mix
  const int forms = layernorm_forms(pb);
  auto kernel_forms = forms == kFormLnA ? gemm_f16_kernel<BN, B_NK, false, false, kFormLnA>
                      : (forms & kFormLnA) == 0 ? gemm_f16_kernel<BN, B_NK, false, false, kFormLnR | kFormStats>
                                                : gemm_f16_kernel<BN, B_NK, false, false, kFormLnA | kFormLnR | kFormStats>;
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    if (!check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiPlain>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, plain)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiGelu>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, GELU)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, 0, kEpiAddC>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, + C)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, kFormLnA>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, LayerNorm on A)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, kFormLnR | kFormStats>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, LayerNorm on the residual)") ||
        !check_cuda(cudaFuncSetAttribute(gemm_f16_kernel<BN, B_NK, false, false, kFormLnA | kFormLnR | kFormStats>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, LayerNorm forms)") ||
        !check_cuda(cudaFuncSetAttribute(kernel_split, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm, split-K)"))
      return false;
    attr_set[dev] = true;
  }
  CUtensorMap tmA, tmB, tmD;
  if (!make_tensor_map_2d(pb.A, pb.K, pb.M, BK, BM, &tmA)) return false;
  if (pb.N % 8 == 0) {
    if (!make_tensor_map_2d(pb.D, pb.N, pb.M, 64, 32, &tmD)) return false;
  } else {
    tmD = tmA;  // never dereferenced: the epilogue stores without TMA when N % 8 != 0
  }
  const bool grouped = !B_NK && pb.N % 64 == 0;
  if (B_NK) {
    if (!make_tensor_map_2d(pb.B, pb.K, pb.N, BK, BN, &tmB)) return false;
  } else if (grouped) {
    if (!make_tensor_map_grouped(pb.B, pb.N, pb.K, BK, BN / 64, &tmB)) return false;
  } else {
    if (!make_tensor_map_2d(pb.B, pb.N, pb.K, 64, BK, &tmB, pb.ldb)) return false;
  }
  Params p;
  p.b_grouped = grouped ? 1 : 0;
  p.b_early = pb.b_const ? 1 : 0;
  p.ep.M = static_cast<int>(pb.M);
  p.ep.N = static_cast<int>(pb.N);
  p.K = static_cast<int>(pb.K);
  p.ep.C = pb.C;
  p.ep.ldc = pb.N;
  p.ep.c_mode = pb.c_mode;
  p.ep.D = pb.D;
  p.ep.ldd = pb.N;
  p.ep.alpha = pb.alpha;
  p.ep.beta = pb.beta;
  p.ep.act = pb.act;
  p.ep.row_scale = pb.row_scale;
  p.ep.row_shift = pb.row_shift;
  p.ep.col_sum = pb.col_sum;
  p.ep.a_partials = pb.a_partials;
  p.ep.r_partials = pb.r_partials;
  p.ep.a_groups = pb.a_groups;
  p.ep.r_groups = pb.r_groups;
  p.ep.a_inv_n = pb.K > 0 ? 1.f / static_cast<float>(pb.K) : 0.f;
  p.ep.r_inv_n = pb.N > 0 ? 1.f / static_cast<float>(pb.N) : 0.f;
  p.ep.ln_eps = pb.ln_eps;
  p.ep.unaligned_n = pb.N % 8 != 0 ? 1 : 0;
  p.ep.row_partials = pb.row_partials;
  const int m_blocks = static_cast<int>((pb.M + BM - 1) / BM);
  p.n_blocks = static_cast<int>((pb.N + BN - 1) / BN);
  p.num_tiles = m_blocks * p.n_blocks;
  p.num_kb = static_cast<int>((pb.K + BK - 1) / BK);
  p.status = device_status_word();
  HOM_DIAG(p.prof = profile_buffer(); p.tl = launch_timeline_slot();)
  p.split_k = has_layernorm_form(pb) ? 1 : clamp_split(split_k, p.num_kb);
  p.num_units = p.num_tiles * p.split_k;
  p.ws_slots = nullptr;
  p.ws_counters = nullptr;
  if (p.split_k > 1) {
    const size_t blocks = static_cast<size_t>(p.num_tiles) * kEpilogueWarps;
    SplitWorkspace ws;
    if (!split_workspace(blocks * kSplitSlotFloats, blocks, stream, &ws)) return false;
    p.ws_slots = ws.slots;
    p.ws_counters = ws.counters;
  }
  const int grid = p.num_units < sm_count() ? p.num_units : sm_count();
  const double flops = 2.0 * pb.M * pb.N * pb.K;
  const double bytes = 2.0 * (static_cast<double>(pb.M) * pb.K + static_cast<double>(pb.K) * pb.N +
                              static_cast<double>(pb.M) * pb.N) +
                       (pb.c_mode == 1 ? 2.0 * pb.M * pb.N : pb.c_mode == 2 ? 2.0 * pb.N : 0.0);
  LaunchScope scope(kOpGemm, flops, bytes);
  if (!check_cuda(launch_pdl(forms != 0 ? kernel_forms : p.split_k > 1 ? kernel_split : kernel,
                             dim3(grid), dim3(kThreads), Cfg::kSmemBytes, stream, 1, tmA, tmB, tmD, p),
                  "gemm kernel launch"))
    return false;
  HOM_DIAG(if (p.prof) profile_report("gemm 1-CTA", p.num_tiles, grid, p.num_kb, stream);)
  return check_cuda(cudaGetLastError(), "gemm kernel launch");
}

// D = LayerNorm(fp16(A.B + R)) over the last dimension: one cluster of pb.N / BN CTAs per 128
// rows (grid = tiles); R in pb.C (c_mode 1) or absent.
template <int BN, bool B_NK>
bool launch_ln_variant(const Problem &pb, float eps, cudaStream_t stream) {
  using Cfg = TileCfg<BN>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  auto kernel = gemm_f16_kernel<BN, B_NK, true>;
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    if (!check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Cfg::kSmemBytes),
                    "cudaFuncSetAttribute(gemm + layernorm)"))
      return false;
    attr_set[dev] = true;
  }
  CUtensorMap tmA, tmB, tmD;
  if (!make_tensor_map_2d(pb.A, pb.K, pb.M, BK, BM, &tmA)) return false;
  if (!make_tensor_map_2d(pb.D, pb.N, pb.M, 64, 32, &tmD)) return false;
  if (B_NK) {
    if (!make_tensor_map_2d(pb.B, pb.K, pb.N, BK, BN, &tmB)) return false;
  } else {
    if (!make_tensor_map_grouped(pb.B, pb.N, pb.K, BK, BN / 64, &tmB)) return false;
  }
  Params p;
  p.b_grouped = B_NK ? 0 : 1;
  p.b_early = pb.b_const ? 1 : 0;
  p.ep.M = static_cast<int>(pb.M);
  p.ep.N = static_cast<int>(pb.N);
  p.K = static_cast<int>(pb.K);
  p.ep.C = pb.C;
  p.ep.ldc = pb.N;
  p.ep.c_mode = pb.c_mode;
  p.ep.D = pb.D;
  p.ep.ldd = pb.N;
  p.ep.alpha = 1.f;
  p.ep.beta = 1.f;
  p.ep.act = 0;
  p.ep.row_scale = nullptr;
  p.ep.row_shift = nullptr;
  p.ep.col_sum = nullptr;
  p.ep.a_partials = nullptr;
  p.ep.r_partials = nullptr;
  p.ep.a_groups = p.ep.r_groups = 0;
  p.ep.a_inv_n = p.ep.r_inv_n = p.ep.ln_eps = 0.f;
  p.ep.unaligned_n = 0;
  p.ep.row_partials = nullptr;
  const int m_blocks = static_cast<int>((pb.M + BM - 1) / BM);
  p.n_blocks = static_cast<int>(pb.N / BN);
  p.num_tiles = m_blocks * p.n_blocks;
  p.num_kb = static_cast<int>((pb.K + BK - 1) / BK);
  p.status = device_status_word();
  HOM_DIAG(p.prof = nullptr; p.tl = nullptr;)
  p.split_k = 1;
  p.num_units = p.num_tiles;
  p.ws_slots = nullptr;
  p.ws_counters = nullptr;
  p.ln_eps = eps;
  p.ln_inv_n = 1.f / static_cast<float>(pb.N);
  p.ln_cluster = p.n_blocks;
  const double flops = 2.0 * pb.M * pb.N * pb.K;
  const double bytes = 2.0 * (static_cast<double>(pb.M) * pb.K + static_cast<double>(pb.K) * pb.N +
                              static_cast<double>(pb.M) * pb.N) +
                       (pb.c_mode == 1 ? 2.0 * pb.M * pb.N : 0.0);
  LaunchScope scope(kOpGemm, flops, bytes);
  return check_cuda(launch_pdl(kernel, dim3(p.num_tiles), dim3(kThreads), Cfg::kSmemBytes, stream,
                               static_cast<unsigned>(p.n_blocks), tmA, tmB, tmD, p),
                    "gemm + layernorm kernel launch");
}

// Tile-table rows: 1-4 = one CTA per 128 x {64,128,192,256} tile; 5, 6 = one CTA pair per
// 256 x {128,256} tile.
struct TileRow {
  int tile_m, tile_n, stages;
  bool pair;
};
const TileRow kTileRows[7] = {
    {0, 0, 0, false},      {128, 64, 8, false},  {128, 128, 6, false}, {128, 192, 4, false},
    {128, 256, 3, false},  {256, 128, 8, true},  {256, 256, 5, true},
};
constexpr int kNumTileRows = 6;

}  // namespace

namespace {

// cuTensorMapEncodeTiled without the cache (no host allocation either).
bool encode_map_uncached(const void *ptr, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
                         const cuuint32_t *box, CUtensorMap *out) {
  EncodeFn encode = get_encode_fn();
  if (!encode) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return false;
  }
  cuuint32_t elem_strides[3] = {1, 1, 1};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank),
                            const_cast<void *>(ptr), dims, strides, box, elem_strides,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(HOM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return false;
  }
  return true;
}

}  // namespace

// Launches the 128 x 128 single-CTA kernel for `pb` (B as [K, N]) without allocating anything:
// tensor maps are encoded on the stack instead of being cached, the device status word is used
// only if an earlier call already created it, and the SM count comes straight from the
// device attribute.
bool run_fixed_no_alloc(const Problem &pb, cudaStream_t stream) {
  constexpr int BN = 128;
  using Cfg = TileCfg<BN>;
  if (pb.M == 0 || pb.N == 0) return true;
  // the instantiation with the LayerNorm forms of the epilogue: this path is the LayerNorm-on-A form
  auto kernel = gemm_f16_kernel<BN, false, false, false, kFormLnA>;
  if (!check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg::kSmemBytes),
                  "cudaFuncSetAttribute(gemm)"))
    return false;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    sms = 148;
  CUtensorMap tmA, tmB, tmD;
  const bool grouped = pb.N % 64 == 0;
  {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(pb.K), static_cast<cuuint64_t>(pb.M)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pb.K) * 2};
    const cuuint32_t box[2] = {BK, BM};
    if (!encode_map_uncached(pb.A, 2, dims, strides, box, &tmA)) return false;
  }
  if (grouped) {
    const cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(pb.K), static_cast<cuuint64_t>(pb.N / 64)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pb.N) * 2, 128};
    const cuuint32_t box[3] = {64, BK, BN / 64};
    if (!encode_map_uncached(pb.B, 3, dims, strides, box, &tmB)) return false;
  } else {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(pb.N), static_cast<cuuint64_t>(pb.K)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pb.N) * 2};
    const cuuint32_t box[2] = {64, BK};
    if (!encode_map_uncached(pb.B, 2, dims, strides, box, &tmB)) return false;
  }
  {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(pb.N), static_cast<cuuint64_t>(pb.M)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pb.N) * 2};
    const cuuint32_t box[2] = {64, 32};
    if (!encode_map_uncached(pb.D, 2, dims, strides, box, &tmD)) return false;
  }
  Params p;
  p.ep.M = static_cast<int>(pb.M);
  p.ep.N = static_cast<int>(pb.N);
  p.K = static_cast<int>(pb.K);
  p.ep.C = pb.C;
  p.ep.ldc = pb.N;
  p.ep.c_mode = pb.c_mode;
  p.ep.D = pb.D;
  p.ep.ldd = pb.N;
  p.ep.alpha = pb.alpha;
  p.ep.beta = pb.beta;
  p.ep.act = pb.act;
  p.ep.row_scale = pb.row_scale;
  p.ep.row_shift = pb.row_shift;
  p.ep.col_sum = pb.col_sum;
  p.ep.a_partials = pb.a_partials;
  p.ep.r_partials = pb.r_partials;
  p.ep.a_groups = pb.a_groups;
  p.ep.r_groups = pb.r_groups;
  p.ep.a_inv_n = pb.K > 0 ? 1.f / static_cast<float>(pb.K) : 0.f;
  p.ep.r_inv_n = pb.N > 0 ? 1.f / static_cast<float>(pb.N) : 0.f;
  p.ep.ln_eps = pb.ln_eps;
  p.ep.unaligned_n = pb.N % 8 != 0 ? 1 : 0;
  p.ep.row_partials = pb.row_partials;
  p.b_grouped = grouped ? 1 : 0;
  p.b_early = pb.b_const ? 1 : 0;
  const int m_blocks = static_cast<int>((pb.M + BM - 1) / BM);
  p.n_blocks = static_cast<int>((pb.N + BN - 1) / BN);
  p.num_tiles = m_blocks * p.n_blocks;
  p.num_kb = static_cast<int>((pb.K + BK - 1) / BK);
  p.status = device_status_word_if_ready();
  HOM_DIAG(p.prof = nullptr; p.tl = nullptr;)
  p.split_k = 1;
  p.num_units = p.num_tiles;
  p.ws_slots = nullptr;
  p.ws_counters = nullptr;
  const int grid = p.num_tiles < sms ? p.num_tiles : sms;
  const double flops = 2.0 * pb.M * pb.N * pb.K;
  const double bytes = 2.0 * (static_cast<double>(pb.M) * pb.K + static_cast<double>(pb.K) * pb.N +
                              static_cast<double>(pb.M) * pb.N);
  LaunchScope scope(kOpGemm, flops, bytes, /*may_allocate=*/false);
  return check_cuda(launch_pdl(kernel, dim3(grid), dim3(kThreads), Cfg::kSmemBytes, stream, 1, tmA, tmB,
                               tmD, p),
                    "gemm kernel launch");
}

// ---- tuned shapes: (M, N, K, activation) -> (tile-table row, K split), filled by tune() or a
// cache file.  Takes the place of the reference's GemmProfiler timing cache
// (include/NVGPUKernels/GemmProfiler.h:39-41), whose entries are (kernel number, split-K factor).
namespace {
using TuneKey = std::tuple<int64_t, int64_t, int64_t, int>;
struct TuneChoice {
  int row, split;
};
std::map<TuneKey, TuneChoice> g_tuned;
std::mutex g_tuned_mutex;
std::atomic<uint32_t> g_tuned_epoch{1};  // bumped after every change of g_tuned

void load_env_cache_once() {
  static std::once_flag once;
  std::call_once(once, [] {
    if (const char *path = std::getenv("HOM_TUNE_CACHE")) tune_cache_load(path);
  });
}

__global__ void fill_pattern_kernel(__half *p, size_t n, uint32_t seed, float scale) {
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<size_t>(gridDim.x) * blockDim.x) {
    uint32_t h = static_cast<uint32_t>(i) * 2654435761u + seed;
    h ^= h >> 15;
    h *= 2246822519u;
    h ^= h >> 13;
    p[i] = __float2half((static_cast<float>(h & 0xffff) / 32768.f - 1.f) * scale);
  }
}

// Candidate K splits for a tile with `num_kb` K blocks: 1..min(16, K / 128) like the
// reference's sweep (lib/NVGPUKernels/GemmProfiler.cu:71-79), thinned to the useful ones.
int split_candidates(int64_t k, int *out) {
  const int num_kb = static_cast<int>((k + BK - 1) / BK);
  const int limit = static_cast<int>(k / 128 < 16 ? k / 128 : 16);
  int n = 0;
  for (int sp : {1, 2, 3, 4, 6, 8, 12, 16})
    if (sp == 1 || (sp <= limit && sp <= num_kb)) out[n++] = sp;
  return n;
}
}  // namespace

bool tuned_choice(int64_t m, int64_t n, int64_t k, int act, int *row, int *split) {
  load_env_cache_once();
  std::lock_guard<std::mutex> lock(g_tuned_mutex);
  auto it = g_tuned.find(TuneKey{m, n, k, act});
  if (it == g_tuned.end()) return false;
  if (row) *row = it->second.row;
  if (split) *split = it->second.split;
  return true;
}

// Text lines "M N K activation row [split]" (split defaults to 1).
int tune_cache_load(const char *path) {
  FILE *f = path ? std::fopen(path, "r") : nullptr;
  if (!f) return -1;
  char line[256];
  int count = 0;
  std::lock_guard<std::mutex> lock(g_tuned_mutex);
  while (std::fgets(line, sizeof(line), f)) {
    long long m, n, k;
    int act, row, split = 1;
    const int got = std::sscanf(line, "%lld %lld %lld %d %d %d", &m, &n, &k, &act, &row, &split);
    if (got >= 5 && row >= 1 && row <= kNumTileRows) {
      if (got < 6 || split < 1) split = 1;
      g_tuned[TuneKey{m, n, k, act}] = TuneChoice{row, split};
      ++count;
    }
  }
  std::fclose(f);
  g_tuned_epoch.fetch_add(1);
  return count;
}

int tune_cache_save(const char *path) {
  FILE *f = path ? std::fopen(path, "w") : nullptr;
  if (!f) return -1;
  std::lock_guard<std::mutex> lock(g_tuned_mutex);
  for (const auto &kv : g_tuned)
    std::fprintf(f, "%lld %lld %lld %d %d %d\n", static_cast<long long>(std::get<0>(kv.first)),
                 static_cast<long long>(std::get<1>(kv.first)),
                 static_cast<long long>(std::get<2>(kv.first)), std::get<3>(kv.first), kv.second.row,
                 kv.second.split);
  std::fclose(f);
  return static_cast<int>(g_tuned.size());
}

// Times every row of the tile table, each with every candidate K split, on scratch buffers of
// the given shape (the contract of GemmProfiler::profile, lib/NVGPUKernels/GemmProfiler.cu:
// 143-236: warm up, then batches of launches between two events on one stream; a candidate that
// is 1.2 x slower than the best so far after its warm-up batch is dropped early; beta != 0 reads
// C = D like the reference does).  row_us[r - 1] is the best time of row r over its splits.
bool tune(int64_t m, int64_t n, int64_t k, int act, float alpha, float beta, bool b_is_nk, int iters,
          int *best_row, int *best_split, float *best_us, float *row_us, cudaStream_t stream) {
  if (m <= 0 || n <= 0 || k <= 0 || k % 8 != 0 || (!b_is_nk && n % 8 != 0)) {
    set_error(HOM_ERR_UNSUPPORTED, "homGemmTune: shape %lld x %lld x %lld is not supported",
              static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k));
    return false;
  }
  if (iters < 1) iters = 20;
  __half *a = nullptr, *b = nullptr, *d = nullptr;
  cudaEvent_t e0 = nullptr, e1 = nullptr;
  auto cleanup = [&]() {
    cudaFree(a);
    cudaFree(b);
    cudaFree(d);
    if (e0) cudaEventDestroy(e0);
    if (e1) cudaEventDestroy(e1);
  };
  if (cudaMalloc(&a, sizeof(__half) * m * k) != cudaSuccess || cudaMalloc(&b, sizeof(__half) * k * n) != cudaSuccess ||
      cudaMalloc(&d, sizeof(__half) * m * n) != cudaSuccess || cudaEventCreate(&e0) != cudaSuccess ||
      cudaEventCreate(&e1) != cudaSuccess) {
    cleanup();
    check_cuda(cudaGetLastError(), "homGemmTune allocation");
    set_error(HOM_ERR_CUDA, "homGemmTune: could not allocate the scratch operands");
    return false;
  }
  fill_pattern_kernel<<<592, 256, 0, stream>>>(a, static_cast<size_t>(m) * k, 1u, 1.f);
  fill_pattern_kernel<<<592, 256, 0, stream>>>(b, static_cast<size_t>(k) * n, 2u, 0.03f);
  fill_pattern_kernel<<<592, 256, 0, stream>>>(d, static_cast<size_t>(m) * n, 3u, 0.5f);
  declare_constant_range(b, sizeof(__half) * k * n);  // weights in the model: prefetched early
  Problem pb;
  pb.M = m;
  pb.N = n;
  pb.K = k;
  pb.A = a;
  pb.B = b;
  pb.b_is_nk = b_is_nk;
  pb.b_const = true;
  pb.C = beta != 0.f ? d : nullptr;
  pb.c_mode = beta != 0.f ? 1 : 0;
  pb.D = d;
  pb.alpha = alpha;
  pb.beta = beta;
  pb.act = act;
  int best = 0, best_sp = 1;
  float best_ms = 1e30f;
  bool ok = true;
  int splits[8];
  const int n_splits = split_candidates(k, splits);
  for (int row = 1; row <= kNumTileRows && ok; ++row) {
    float row_best = 1e30f;
    for (int si = 0; si < n_splits && ok; ++si) {
      pb.split_k = splits[si];
      auto timed = [&](int count, float *ms) {
        cudaEventRecord(e0, stream);
        for (int i = 0; i < count && ok; ++i) ok = run(pb, row, stream);
        cudaEventRecord(e1, stream);
        if (cudaEventSynchronize(e1) != cudaSuccess) ok = false;
        *ms = 0.f;
        if (ok) cudaEventElapsedTime(ms, e0, e1);
      };
      float warm_ms = 0.f, ms = 0.f;
      timed(5, &warm_ms);
      if (!ok) break;
      if (warm_ms / 5 > 1.2f * best_ms) continue;  // early-out like the reference's profiler
      timed(iters, &ms);
      if (!ok) break;
      ms /= iters;
      if (ms < row_best) row_best = ms;
      if (ms < best_ms) {
        best_ms = ms;
        best = row;
        best_sp = splits[si];
      }
    }
    if (row_us) row_us[row - 1] = row_best < 1e29f ? 1e3f * row_best : -1.f;
  }
  forget_constant_range(b);
  cleanup();
  if (!ok || best == 0) return false;
  {
    std::lock_guard<std::mutex> lock(g_tuned_mutex);
    g_tuned[TuneKey{m, n, k, act}] = TuneChoice{best, best_sp};
    g_tuned_epoch.fetch_add(1);
  }
  if (best_row) *best_row = best;
  if (best_split) *best_split = best_sp;
  if (best_us) *best_us = 1e3f * best_ms;
  return true;
}

namespace {
// Estimated duration (microseconds, inside a chain of dependent launches) of a launch with
// tile-table row `row` and K split `sp`.  The constants are a fit to 1,500 launches measured on
// the GEMMs of both BERT sizes at M = 64 .. 16384 (rms 6-8 % per row; over those shapes the row
// the estimate picks is on average 0.4 %, at worst 8 %, slower than the fastest one measured):
//   whole-K tiles     fixed + rounds * K blocks * time per K block, which grows with the share of
//                     the chip in use (the CTAs share the L2 -> SM path and the power budget),
//                     plus what an epilogue outlasts the next tile's main loop by;
//   clusters (rows 1 and 2 with a split of 2..8)   fixed + K blocks per CTA * time per block +
//                     exchange, which grows with the parts and with the CTAs that exchange.
struct RowCost {
  double fixed, per_kb, epilogue, busy_kb, busy;
};
constexpr RowCost kRowCost[7] = {
    {0, 0, 0, 0, 0},
    {3.16, 0.181, 2.65, 0.087, 0.77},  // 128 x 64
    {3.98, 0.182, 3.42, 0.383, 0.08},  // 128 x 128
    {3.97, 0.273, 4.56, 0.249, 0.27},  // 128 x 192
    {4.02, 0.396, 5.86, 0.168, 0.55},  // 128 x 256
    {4.15, 0.193, 3.13, 0.217, 1.32},  // pair 256 x 128
    {5.21, 0.286, 4.73, 0.268, 0.90},  // pair 256 x 256
};

double estimate_us(int row, int sp, int64_t m, int64_t n, int64_t k) {
  const TileRow &t = kTileRows[row];
  const double tiles = static_cast<double>(((m + t.tile_m - 1) / t.tile_m) * ((n + t.tile_n - 1) / t.tile_n));
  const double num_kb = static_cast<double>((k + BK - 1) / BK);
  if (sp > 1 && row <= 2 && sp <= kMaxClusterParts) {
    const double kb = std::ceil(num_kb / sp);
    return row == 1 ? 3.9 + 0.16 * kb + 0.13 * (sp - 2) + 0.006 * tiles * sp
                    : 5.9 + 0.22 * kb + 0.10 * (sp - 2) + 0.005 * tiles * sp;
  }
  const RowCost &c = kRowCost[row];
  const double slots = t.pair ? sm_count() / 2 : sm_count();
  const double rounds = std::ceil(tiles * sp / slots);
  const double share = std::min(tiles * sp, slots) / slots;
  const double unit = std::ceil(num_kb / sp) * c.per_kb * (1.0 + c.busy_kb * share * share);
  double us = c.fixed + rounds * unit + (rounds - 1) * std::max(0.0, c.epilogue - unit) + c.busy * share;
  // The serial split (any other row or factor): every part moves its fp32 block through L2 once
  // more and the parts' epilogues form a chain, 6-8 us per extra part at 256-wide tiles.
  if (sp > 1) us += (sp - 1) * (1.6 + 0.02 * t.tile_n);
  return us;
}
}  // namespace

namespace {
int choose_tile_row(int64_t m, int64_t n, int64_t k, int act, int *split_k, bool may_split) {
  if (split_k) *split_k = 1;
  const bool whole_n = may_split && n % 8 == 0;  // what the cluster form asks for
  HOM_DIAG(if (const char *env = std::getenv("HOM_GEMM_TILE")) {  // experiment knob
    const int v = std::atoi(env);
    if (v >= 1 && v <= kNumTileRows) {
      if (split_k) *split_k = std::getenv("HOM_GEMM_SPLIT") ? std::atoi(std::getenv("HOM_GEMM_SPLIT")) : 1;
      return v;
    }
  })
  int row = 0, sp = 1;
  if (tuned_choice(m, n, k, act, &row, &sp)) {
    if (split_k) *split_k = sp;
    return row;
  }
  int best = 1, best_sp = 1;
  double best_cost = 1e300;
  int splits[8];
  const int n_splits = split_candidates(k, splits);
  for (int r = 1; r <= kNumTileRows; ++r) {
    const TileRow &t = kTileRows[r];
    const int64_t tiles = ((m + t.tile_m - 1) / t.tile_m) * ((n + t.tile_n - 1) / t.tile_n);
    for (int i = 0; i < n_splits; ++i) {
      const int parts = splits[i];
      // Only the cluster form splits by itself, and only while all clusters run at once: a second
      // wave of them costs 5 us, more than any split gains (36 clusters of 4, of which 33 fit:
      // 8.3 us against 4.3 us for 36 clusters of 2).
      if (parts > 1 && (!whole_n || r > 2 || parts > kMaxClusterParts || tiles > cluster_capacity(t.tile_n, parts)))
        continue;
      const double c = estimate_us(r, parts, m, n, k);
      if (c < best_cost - 1e-9) {
        best_cost = c;
        best = r;
        best_sp = parts;
      }
    }
  }
  if (split_k) *split_k = best_sp;
  return best;
}

}  // namespace

// A program calls with a handful of shapes over and over, and weighing 20 candidates takes longer
// than the rest of a call: each thread keeps its latest choices, one per hash slot, valid for one
// device until the table of tuned shapes changes.
int select_tile_row(int64_t m, int64_t n, int64_t k, int act, int *split_k, bool may_split) {
#if HOM_DIAG_ENABLED
  return choose_tile_row(m, n, k, act, split_k, may_split);  // the experiment knobs may change between calls
#else
  struct Choice {
    int64_t m = -1, n = 0, k = 0;
    int act = 0, device = -1;
    bool may_split = false;
    uint32_t epoch = 0;
    int row = 0, split = 1;
  };
  thread_local Choice recent[64];
  load_env_cache_once();
  const uint32_t epoch = g_tuned_epoch.load();
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t h = (static_cast<uint64_t>(m) * 0x9E3779B97F4A7C15ull) ^ (static_cast<uint64_t>(n) * 0xC2B2AE3D27D4EB4Full) ^
                     (static_cast<uint64_t>(k) * 0x165667B19E3779F9ull) ^ static_cast<uint64_t>(2 * act + may_split);
  Choice &c = recent[(h ^ (h >> 32)) >> 7 & 63];
  if (c.m != m || c.n != n || c.k != k || c.act != act || c.may_split != may_split || c.device != device ||
      c.epoch != epoch) {
    c.row = choose_tile_row(m, n, k, act, &c.split, may_split);
    c.m = m;
    c.n = n;
    c.k = k;
    c.act = act;
    c.may_split = may_split;
    c.device = device;
    c.epoch = epoch;
  }
  if (split_k) *split_k = c.split;
  return c.row;
#endif
}

int query_tile(int64_t m, int64_t n, int64_t k, int act, int *bn, int *stages, int *split_k) {
  int sp = 1;
  const int row = select_tile_row(m, n, k, act, &sp);
  if (bn) *bn = kTileRows[row].tile_n;
  if (stages) *stages = kTileRows[row].stages;
  if (split_k) *split_k = sp;
  return row;
}

bool layernorm_fusion_shape(int64_t n, int *cluster_n, int *bn) {
  for (int c : {1, 2, 4, 8}) {
    if (n % c != 0) continue;
    const int64_t w = n / c;
    if (w == 64 || w == 128 || w == 192 || w == 256) {
      if (cluster_n) *cluster_n = c;
      if (bn) *bn = static_cast<int>(w);
      return true;
    }
  }
  return false;
}

bool run_layernorm_fused(const Problem &pb, float eps, cudaStream_t stream) {
  if (pb.M == 0 || pb.N == 0) return true;
  int cluster_n = 0, bn = 0;
  if (!layernorm_fusion_shape(pb.N, &cluster_n, &bn)) {
    set_error(HOM_ERR_UNSUPPORTED,
              "fused GEMM + LayerNorm needs N = c x {64,128,192,256} with c in {1,2,4,8} (got N = %lld)",
              static_cast<long long>(pb.N));
    return false;
  }
  if (pb.b_is_nk) {
    switch (bn) {
      case 64: return launch_ln_variant<64, true>(pb, eps, stream);
      case 128: return launch_ln_variant<128, true>(pb, eps, stream);
      case 192: return launch_ln_variant<192, true>(pb, eps, stream);
      default: return launch_ln_variant<256, true>(pb, eps, stream);
    }
  }
  switch (bn) {
    case 64: return launch_ln_variant<64, false>(pb, eps, stream);
    case 128: return launch_ln_variant<128, false>(pb, eps, stream);
    case 192: return launch_ln_variant<192, false>(pb, eps, stream);
    default: return launch_ln_variant<256, false>(pb, eps, stream);
  }
}

bool run(const Problem &pb, int tile_row, cudaStream_t stream) {
  if (pb.M == 0 || pb.N == 0) return true;
  int split = 1;
  if (tile_row < 1 || tile_row > kNumTileRows) {
    tile_row = select_tile_row(pb.M, pb.N, pb.K, pb.act, &split, !has_layernorm_form(pb));
    if (pb.split_k >= 2) split = pb.split_k;
  } else {
    split = pb.split_k >= 2 ? pb.split_k : 1;
  }
  if (has_layernorm_form(pb)) {
    split = 1;  // those epilogue forms exist for whole-K tiles only
    if (pb.N % 8 != 0) {
      set_error(HOM_ERR_UNSUPPORTED, "the LayerNorm forms of the GEMM epilogue need N %% 8 == 0 (got N = %lld)",
                static_cast<long long>(pb.N));
      return false;
    }
  }
  split = clamp_split(split, static_cast<int>((pb.K + BK - 1) / BK));
  const TileRow &t = kTileRows[tile_row];
  if (t.pair) return run_pair(pb, t.tile_n, split, stream);
  // 128 x {64,128} tiles with a short K split: one cluster per tile, parts reduced SM to SM.
  if (tile_row <= 2 && cluster_supported(pb, split) && cluster_pays(pb, t.tile_n, split))
    return run_cluster(pb, t.tile_n, split, stream);
  if (pb.b_is_nk) {
    switch (t.tile_n) {
      case 64: return launch_variant<64, true>(pb, split, stream);
      case 128: return launch_variant<128, true>(pb, split, stream);
      case 192: return launch_variant<192, true>(pb, split, stream);
      default: return launch_variant<256, true>(pb, split, stream);
    }
  }
  switch (t.tile_n) {
    case 64: return launch_variant<64, false>(pb, split, stream);
    case 128: return launch_variant<128, false>(pb, split, stream);
    case 192: return launch_variant<192, false>(pb, split, stream);
    default: return launch_variant<256, false>(pb, split, stream);
  }
}

}  // namespace gemm
}  // namespace hom
