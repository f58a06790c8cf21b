// Product of two microscaled 4-bit matrices on CTA pairs: D = act(alpha * A.B^T + beta * C) for
// problems with many tiles (format: mxf4_sm100.cuh).
//
// A 256 x 256 tile belongs to a cluster of two CTAs on neighbouring SMs; each holds 128 rows of A,
// 128 rows of B and the accumulator of its 128 output rows.  The grid is persistent.  A step is 256
// values along K; its four 256 x 256 x 64 MMAs take 512 tensor-pipe cycles.
//
// The times in this file are those of a few calls in a burst.  In a loop that the power limit has
// slowed down the long ones take more: 131072 x 4096 x 1024 with GELU 392 us instead of 324, 16384 x
// 4096 x 4096 125 instead of 109, 131072 x 4096 x 256 with GELU 305 instead of 274.
//
// What bounds it: a step brings 35 KB to each SM, and with four stages in flight L2 delivers some
// 16 TB/s.  Timed by leaving parts out, 16384 x 4096 x 4096 (107 us) takes 77 us with a quarter of
// the MMAs and no stores, 74 with neither loads nor stores: the two overlap, but not wholly.  The
// scale copies cost 5 %.  With up to four steps (K <= 1024) A's rows can stay in shared memory while
// the pair works through the column tiles of a row block ("resident"), and only B streams.
//
// Tensor memory: every stage of the ring has its own 24 columns of scales, so that the issuing
// thread waits for nothing but the stage: that it was filled again says that the MMAs of its last
// use, and their reads of the scales, are over.  Two whole accumulators do not fit beside 96 columns
// of scales: the first lies in [0, 256), the second in [160, 416), and the warps that drain the 96
// columns they share take them into registers at once, so that the next tile's MMAs can start while
// the rest is drained beside them.  (192-column tiles need not share, but pull 1.18 times the bytes
// through L2 for the same work, 31 KB a step instead of 35 for three quarters of the columns: 16384 x
// 4096 x 4096 120 us instead of 107, 32768 x 4096 x 1024 73 instead of 69.)
//
// With GELU the epilogue's instructions are the bound where K is small: 131072 x 4096 x 256 takes
// 277 us, 209 without GELU, the rate at which D can be written; 3400 of the 5300 cycles that a tile
// takes are arithmetic.  What lies between two tiles' arithmetic counts as well: with a division for
// the tile's place, and the row of C laid out before the accumulator was asked for, 293 us.
//
//   warps 0, 2, 3  TMA producers of A's codes, of B's and of the scales
//   warp 1         tensor memory, scale copies and MMA issue (even CTA)
//   warps 4 and up epilogue: four warps per tensor-memory lane quarter, one 64-column group each
#include <atomic>

#include "gemm_epilogue.cuh"
#include "gemm_sm100.cuh"
#include "mxf4_epilogue.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

using namespace hom::ptx;

namespace {

constexpr int BM = 256, BN = 256, kHalf = 128;         // tile; rows of A and of B per CTA
constexpr int kStepBytes = 128;                        // of a row of codes: 256 values
constexpr int kStepBlocks = 2 * kStepBytes / kBlock;   // 8
constexpr int kStepTiles = kStepBlocks / kTileBlocks;  // 2 scale tiles along K
constexpr int kStages = 4;                             // and the steps that A may have to stay resident
constexpr int kControlWarps = 4;
constexpr int kMaxPairs = 512;                         // of any device, generously
constexpr uint32_t kCodeBytes = kHalf * kStepBytes;    // of one operand, per CTA and stage
constexpr uint32_t kScaleABytes = kStepTiles * kTileBytes, kScaleBBytes = 2 * kScaleABytes;
constexpr uint32_t kAStageBytes = kCodeBytes + kScaleABytes;
constexpr uint32_t kBStageBytes = kCodeBytes + kScaleBBytes;
constexpr int kDrainWarps = 16;
constexpr int kThreads = 32 * (kControlWarps + kDrainWarps);
// shared-memory offsets: stages of A, of B, staging tiles and rows of C per epilogue warp, barriers
constexpr uint32_t kB = kStages * kAStageBytes;
constexpr uint32_t kStaging = kB + kStages * kBStageBytes;
constexpr uint32_t kBias = kStaging + kDrainWarps * gemm::kEpilogueStageBytes;
constexpr uint32_t kBars = kBias + kDrainWarps * 256;
constexpr int kBarriers = 4 * kStages + 5 + kDrainWarps;
constexpr uint32_t kSmemBytes = kBars + 8 * kBarriers + 16 + 1024;
// tensor-memory columns
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSecondAcc = 160, kScales = kSecondAcc + BN;
constexpr int kSharingGroups = 2;  // 64-column groups with shared columns: the first accumulator's last, the second's first
constexpr uint32_t kScaleSet = 4 * kStepTiles * 3, kScalesB = 4 * kStepTiles;
static_assert(kAStageBytes % 1024 == 0 && kBStageBytes % 1024 == 0, "swizzled tiles start on 1024 bytes");
static_assert(kScales + kStages * kScaleSet <= kTmemCols, "accumulators and scales exceed tensor memory");
static_assert(kSmemBytes <= 227 * 1024, "exceeds a CTA's shared memory");

struct Params {
  const __half *C;  // read where TMA does not: a row of N; a matrix of the ragged forms
  __half *D;        // written by the ragged forms
  float alpha, beta;
  int c_mode, act;
  int M, N;
  int steps, n_blocks, tiles;
  int resident;  // steps <= kStages: A's rows stay in shared memory for the tiles of a row block
  int b_early;   // B is a declared constant: request its first tiles before griddepcontrol.wait
  int *status;
  int fill[6];
};
static_assert(quick_to_launch<Params>, "see launch_pdl");  // (the tensor maps before it are whole 64 bytes)

// Which C and activation an instantiation handles, with alpha = beta = 1; kAny handles all of it,
// kRagged also N that is not a multiple of 8: rows of C and D then start at any element, and the
// warp moves them between memory and its staging tile itself, a row at a time; kWords where N is even
// and C and D start on 4 bytes (4096 x 30522 x 768 93 us, value by value 125).
enum Form { kNone = 0, kRow = 1, kFull = 2, kGelu = 4, kAny = 8, kRagged = 16, kWords = 32 };
__host__ __device__ constexpr bool general(int form) { return form >= kAny; }

// The staging tile of 32 rows x 64 columns: 128-byte rows whose 16-byte chunks are XOR-swizzled by
// the row; this lane's two neighbouring columns are the 32-bit word at this place.
__device__ __forceinline__ uint32_t staging_word(uint32_t stage_smem, int row, int lane) {
  return stage_smem + row * 128 + ((static_cast<uint32_t>(lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4;
}

// Ragged forms: C's block to the staging tile, zeros beyond the matrix; eight rows in flight.  WORDS: two
// neighbouring values are one word of memory.
template <bool WORDS>
__device__ __forceinline__ void ragged_load(const __half *c, int m, int n, int row0, int c0, uint32_t stage_smem, int lane) {
  const unsigned short *from = reinterpret_cast<const unsigned short *>(c);
  const int col = c0 + 2 * lane;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {
    uint32_t v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = row0 + r0 + r;
      const unsigned short *at = from + static_cast<long long>(row) * n + col;
      if constexpr (WORDS) {
        v[r] = row < m && col < n ? *reinterpret_cast<const uint32_t *>(at) : 0u;
      } else {
        const uint32_t lo = row < m && col < n ? at[0] : 0u, hi = row < m && col + 1 < n ? at[1] : 0u;
        v[r] = lo | hi << 16;
      }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(staging_word(stage_smem, r0 + r, lane)), "r"(v[r]) : "memory");
  }
}

// And D's block from the staging tile.
template <bool WORDS>
__device__ __forceinline__ void ragged_store(__half *d, int m, int n, int row0, int c0, uint32_t stage_smem, int lane) {
  unsigned short *to = reinterpret_cast<unsigned short *>(d);
  const int col = c0 + 2 * lane;
  if constexpr (WORDS) {
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 8) {
      uint32_t v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[r]) : "r"(staging_word(stage_smem, r0 + r, lane)) : "memory");
      unsigned short *at = to + static_cast<long long>(row0 + r0) * n + col;
#pragma unroll
      for (int r = 0; r < 8; ++r, at += n)
        if (row0 + r0 + r < m && col < n) *reinterpret_cast<uint32_t *>(at) = v[r];
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      const int row = row0 + r;
      uint32_t v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(staging_word(stage_smem, r, lane)) : "memory");
      unsigned short *at = to + static_cast<long long>(row) * n + col;
      if (row < m && col < n) at[0] = static_cast<unsigned short>(v);
      if (row < m && col + 1 < n) at[1] = static_cast<unsigned short>(v >> 16);
    }
  }
}

// Applies the epilogue to 32 accumulators of this lane's row and leaves the fp16 results in the
// staging tile, whose row holds C's values where C is a matrix; `bias` is
// the row of C otherwise, in fp32 (in the general forms, which are short of registers, in fp16).
template <int FORM>
__device__ __forceinline__ void finish_half(const Params &p, const uint32_t (&acc)[32], int half, uint32_t my_row,
                                            uint32_t bias, int lane) {
  const float2 alpha2 = make_float2(p.alpha, p.alpha), beta2 = make_float2(p.beta, p.beta);
  const bool full = general(FORM) ? p.c_mode == 1 : (FORM & kFull) != 0;
  const bool row = general(FORM) ? p.c_mode == 2 : (FORM & kRow) != 0;
  constexpr int kChunks = 2;  // 16-byte pieces of the staging row at a time
#pragma unroll
  for (int g = 0; g < 4; g += kChunks) {
    float2 v[4 * kChunks];
    uint32_t addr[kChunks];
#pragma unroll
    for (int h = 0; h < kChunks; ++h) {
      addr[h] = my_row + ((static_cast<uint32_t>(half * 4 + g + h) ^ (lane & 7u)) << 4);
      float2 c[4];
      if (full || (row && general(FORM))) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(full ? addr[h] : bias + (half * 4 + g + h) * 16)
                     : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      } else if (row) {
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(c[j].x), "=f"(c[j].y), "=f"(c[j + 1].x), "=f"(c[j + 1].y)
                       : "r"(bias + (half * 32 + (g + h) * 8 + j * 2) * 4)
                       : "memory");
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (g + h) * 8 + 2 * j;
        float2 x = make_float2(__uint_as_float(acc[i]), __uint_as_float(acc[i + 1]));
        if (general(FORM)) x = __fmul2_rn(alpha2, x);
        if (full || row) x = general(FORM) ? __ffma2_rn(beta2, c[j], x) : __fadd2_rn(c[j], x);
        v[4 * h + j] = x;
      }
    }
    if (general(FORM) ? p.act == 1 : (FORM & kGelu) != 0) gelu2(v);
#pragma unroll
    for (int h = 0; h < kChunks; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2 r = __floats2half2_rn(v[4 * h + j].x, v[4 * h + j].y);
        w[j] = *reinterpret_cast<const uint32_t *>(&r);
      }
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr[h]), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                   : "memory");
    }
  }
}

template <int FORM>
__global__ void __launch_bounds__(kThreads, 1)
gemm_mxf4_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                      const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmD,
                      const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t bar_base = smem_base + kBars;
  // full (even CTA, both CTAs' bytes) and empty (both) per stage of the ring, the same for a
  // resident A; accumulator full (both) and empty (even); shared columns drained (even); C landed
  // (per epilogue warp)
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto a_full_bar = [&](int s) { return bar_base + 8u * (2 * kStages + s); };
  auto a_empty_bar = [&](int s) { return bar_base + 8u * (3 * kStages + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (4 * kStages + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (4 * kStages + 2 + a); };
  const uint32_t shared_bar = bar_base + 8u * (4 * kStages + 4);
  auto c_bar = [&](int w) { return bar_base + 8u * (4 * kStages + 5 + w); };
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kBars + 8 * kBarriers);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0: even CTA (issues the MMAs), 1: odd CTA
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  // A resident A wants the tiles of a row block one after the other; otherwise the pairs work side
  // by side on neighbouring tiles, which share their operands in L2.
  const bool resident = p.resident != 0;
  const int first = resident ? static_cast<int>(static_cast<long long>(p.tiles) * pair / num_pairs) : pair;
  const int last = resident ? static_cast<int>(static_cast<long long>(p.tiles) * (pair + 1) / num_pairs) : p.tiles;
  const int stride = resident ? 1 : num_pairs;

  if (threadIdx.x == 64) {
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmSB);
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmSA);
    prefetch_tensormap(&tmD);
  }
  if (warp == 0) {
    for (int i = lane; i < kBarriers; i += 32) {
      const uint32_t bar = bar_base + 8 * i;
      const bool acc_empty = bar == acc_empty_bar(0) || bar == acc_empty_bar(1);
      mbar_init(bar, bar == shared_bar ? 2 * 4 * kSharingGroups : acc_empty ? 2 * kDrainWarps : 1);
    }
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
    __syncwarp();
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

  if (warp == 0 || warp == 2 || warp == 3) {
    // ------------------------------------------------------------- TMA producers
    if (elect_one()) {
      const uint32_t full_even = map_to_cta(full_bar(0), 0), a_full_even = map_to_cta(a_full_bar(0), 0);
      // Each phase is armed by the even CTA for the bytes of both (copies may land first: the phase
      // needs the arrival): the ring's by the producer of B, a resident A's by the producer of A.
      const bool arms = rank == 0 && (warp == 2 || (warp == 0 && resident));
      const uint32_t armed_bytes = 2 * (warp == 0 ? kAStageBytes : kBStageBytes + (resident ? 0 : kAStageBytes));
      const uint32_t armed_bar = warp == 0 ? a_full_bar(0) : full_bar(0);
      auto load_a = [&](uint32_t slot, int step, int m0) {
        const uint32_t bar = (resident ? a_full_even : full_even) + 8 * slot, dst = smem_base + slot * kAStageBytes;
        if (warp == 0) tma_load_2d_pair(dst, &tmA, bar, step * (kStepBytes / 2), m0);
        else tma_load_3d_pair(dst + kCodeBytes, &tmSA, bar, 0, step * kStepTiles, m0 / kTileRows);
      };
      auto load_b = [&](uint32_t slot, int step, int n0) {
        const uint32_t bar = full_even + 8 * slot, dst = smem_base + kB + slot * kBStageBytes;
        if (warp == 2) tma_load_2d_pair(dst, &tmB, bar, step * (kStepBytes / 2), n0 + static_cast<int>(rank) * kHalf);
        else tma_load_3d_pair(dst + kCodeBytes, &tmSB, bar, 0, step * kStepTiles, n0 / kTileRows);
      };
      // The first round of stages is armed, and a declared B requested, before the previous kernel
      // has finished.  The stages are free the first time round: the producer of B waits for that
      // kernel after it, before its first limited wait.
      int early = first < last ? min(kStages, p.steps) : 0, a_early = early;
      if (arms)
        for (int i = 0; i < early; ++i) mbar_arrive_expect_tx(armed_bar + 8 * i, armed_bytes);
      bool waits = warp == 2 && p.b_early;
      if (!waits) pdl_wait();
      uint32_t slot = 0, ph = 0, a_ph = 0;
      bool ok = true;
      for (int tile = first; tile < last && ok; tile += stride) {
        const int m0 = tile / p.n_blocks * BM + static_cast<int>(rank) * kHalf, n0 = tile % p.n_blocks * BN;
        const bool new_a = !resident || tile == first || tile % p.n_blocks == 0;
        for (int i = 0; i < p.steps; ++i) {
          if (warp != 2 && resident && new_a) {
            if (a_early > 0) {
              --a_early;
            } else {
              ok = mbar_wait(a_empty_bar(i), a_ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
              if (!ok) break;
              if (arms) mbar_arrive_expect_tx(armed_bar + 8 * i, armed_bytes);
            }
            load_a(i, i, m0);
          }
          if (warp == 0 && resident) continue;
          if (early > 0) {
            --early;
          } else {
            ok = mbar_wait(empty_bar(slot), ph ^ 1u, abort_flag, p.status, kDevWaitTimeoutProducer);
            if (!ok) break;
            if (arms) mbar_arrive_expect_tx(armed_bar + 8 * slot, armed_bytes);
          }
          if (warp != 0) load_b(slot, i, n0);
          if (warp != 2 && !resident) load_a(slot, i, m0);
          if (++slot == kStages) {
            slot = 0;
            ph ^= 1u;
            if (waits) {
              pdl_wait();
              waits = false;
            }
          }
        }
        if (new_a) a_ph ^= 1u;
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
      uint32_t slot = 0, ph = 0, a_ph = 0;
      bool ok = true;
      int it = 0, n_block = first % p.n_blocks;  // (where A is resident)
      for (int tile = first; tile < last && ok; tile += stride, ++it) {
        const int acc = it & 1;
        const uint32_t d_tmem = tmem_base + (acc ? kSecondAcc : 0);
        const bool new_a = resident && (tile == first || n_block == 0);
        if (++n_block == p.n_blocks) n_block = 0;
        const bool ends_a = resident && (tile + 1 == last || n_block == 0);
        for (int i = 0; i < p.steps; ++i) {
          ok = mbar_wait<true>(full_bar(slot), ph, abort_flag, p.status, kDevWaitTimeoutMma);
          if (ok && new_a) ok = mbar_wait<true>(a_full_bar(i), a_ph, abort_flag, p.status, kDevWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t src_a = smem_base + (resident ? i : slot) * kAStageBytes;
          const uint32_t src_b = smem_base + kB + slot * kBStageBytes;
          const uint32_t scales = tmem_base + kScales + slot * kScaleSet;
#pragma unroll
          for (int k = 0; k < kStepTiles; ++k) {
            tc_copy_scales_pair(scales + 4 * k, make_smem_desc_scales(src_a + kCodeBytes + k * kTileBytes));
#pragma unroll
            for (int n = 0; n < 2; ++n)
              tc_copy_scales_pair(scales + kScalesB + 4 * (2 * k + n),
                                  make_smem_desc_scales(src_b + kCodeBytes + (n * kStepTiles + k) * kTileBytes));
          }
          if (i == 0) {
            // everything else of the tile's first step is in place when its accumulator becomes free
            ok = mbar_wait(acc_empty_bar(acc), ((it >> 1) & 1) ^ 1, abort_flag, p.status, kDevWaitTimeoutMma);
            if (ok && it > 0)
              ok = mbar_wait(shared_bar, (it - 1) & 1, abort_flag, p.status, kDevWaitTimeoutMma);
            if (!ok) break;
            tc_fence_after_sync();
          }
          const uint64_t da = make_smem_desc_sw128(src_a, 16, 1024), db = make_smem_desc_sw128(src_b, 16, 1024);
#pragma unroll
          for (int k = 0; k < 2 * kStepTiles; ++k)
            tc_mma_mxf4_ss_pair(d_tmem, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32),
                                k & 1 ? make_idesc_mxf4(BM, BN, 1) : make_idesc_mxf4(BM, BN, 0), scales + 4 * (k >> 1),
                                scales + kScalesB + 8 * (k >> 1), i != 0 || k != 0 ? 1u : 0u);
          tc_commit_pair(empty_bar(slot), 0x3);  // frees the stage in both CTAs
          if (ends_a) tc_commit_pair(a_empty_bar(i), 0x3);
          if (++slot == kStages) {
            slot = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit_pair(acc_full_bar(acc), 0x3);
        if (new_a) a_ph ^= 1u;
      }
    }
    __syncwarp();
  } else {
    // --------------------------------------------------------------- epilogue
    const int drain = warp - kControlWarps;
    const int quarter = warp & 3;
    const int group = drain >> 2;
    const uint32_t stage_smem = smem_base + kStaging + drain * gemm::kEpilogueStageBytes;
    const uint32_t my_row = stage_smem + lane * 128;
    const uint32_t bias = smem_base + kBias + drain * 256;
    const bool full = general(FORM) ? p.c_mode == 1 : (FORM & kFull) != 0;
    const bool row = general(FORM) ? p.c_mode == 2 : (FORM & kRow) != 0;
    constexpr bool ragged = FORM >= kRagged;
    auto arrive_even = [&](uint32_t bar) {
      if (lane == 0) {
        if (rank == 0) mbar_arrive(bar);
        else mbar_arrive_remote(map_to_cta(bar, 0));
      }
    };
    // two neighbouring values of the row of C, requested one tile ahead
    auto load_row = [&](int n_block) {
      const int col = n_block * BN + group * 64 + 2 * lane;
      if (ragged) {
        const unsigned short *at = reinterpret_cast<const unsigned short *>(p.C) + col;
        const uint32_t lo = col < p.N ? at[0] : 0u, hi = col + 1 < p.N ? at[1] : 0u;
        return lo | hi << 16;
      }
      return p.C != nullptr && col < p.N ? *reinterpret_cast<const uint32_t *>(p.C + col) : 0u;
    };
    pdl_wait();  // C may be produced, and D still read, by the previous kernel
    // the tile's place, carried along: a division per tile stood in the way of its first steps
    int m_block = first / p.n_blocks, n_block = first - m_block * p.n_blocks;
    const int m_stride = stride / p.n_blocks, n_stride = stride - m_stride * p.n_blocks;
    uint32_t next_row = row && first < last ? load_row(n_block) : 0u;
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < last; tile += stride, ++it) {
      const int acc = it & 1;
      const int row0 = m_block * BM + static_cast<int>(rank) * kHalf + quarter * 32;
      const int c0 = n_block * BN + group * 64;
      // Is the block part of the matrix?  (kRagged tests every place by itself; this test around it made
      // 8000 x 1001 x 1000 with a matrix C 24.5 us instead of 21.7.)
      const bool live = FORM == kRagged || (c0 < p.N && row0 < p.M);
      m_block += m_stride;
      n_block += n_stride;
      if (n_block >= p.n_blocks) {
        n_block -= p.n_blocks;
        ++m_block;
      }
      // The staging tile was handed to TMA by this warp's previous block: that read must be over
      // before the tile is written again.
      if (ragged) {
        __syncwarp();
        if (full && live) ragged_load<FORM == kWords>(p.C, p.M, p.N, row0, c0, stage_smem, lane);
        __syncwarp();
      } else if (full && lane == 0) {
        bulk_wait_group_read_0();
        mbar_arrive_expect_tx(c_bar(drain), gemm::kEpilogueTileBytes);
        tma_load_2d(stage_smem, &tmC, c_bar(drain), c0, row0);
      }
      ok = mbar_wait(acc_full_bar(acc), (it >> 1) & 1, abort_flag, p.status, kDevWaitTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (acc ? kSecondAcc : 0) + group * 64;
      // (not before the wait for the accumulator, where the way to the shared columns would be longer)
      auto prepare = [&]() {
        if (row) {
          if (general(FORM)) {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(bias + 4 * lane), "r"(next_row) : "memory");
          } else {
            const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&next_row));
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(bias + 8 * lane), "f"(two.x), "f"(two.y) : "memory");
          }
          if (tile + stride < last) next_row = load_row(n_block);
        }
        if (!full && !ragged && lane == 0) bulk_wait_group_read_0();
        __syncwarp();
      };
      auto drained = [&]() {
        tc_fence_before_sync();
        __syncwarp();
      };
      auto staging_ready = [&]() {
        if (full && !ragged)
          ok = __all_sync(0xffffffffu, mbar_wait(c_bar(drain), it & 1, abort_flag, p.status, kDevWaitTimeoutEpilogue));
      };
      if (acc ? group < kSharingGroups : group >= 4 - kSharingGroups) {
        uint32_t lo[32], hi[32];
        tmem_ld_32x32(t_row, lo);
        tmem_ld_32x32(t_row + 32, hi);
        tmem_ld_wait();
        drained();
        arrive_even(shared_bar);
        arrive_even(acc_empty_bar(acc));
        prepare();
        staging_ready();
        finish_half<FORM>(p, lo, 0, my_row, bias, lane);
        finish_half<FORM>(p, hi, 1, my_row, bias, lane);
      } else {
        uint32_t v[32];
        tmem_ld_32x32(t_row, v);
        prepare();
        tmem_ld_wait();
        staging_ready();
        finish_half<FORM>(p, v, 0, my_row, bias, lane);
        tmem_ld_32x32(t_row + 32, v);
        tmem_ld_wait();
        drained();
        arrive_even(acc_empty_bar(acc));
        finish_half<FORM>(p, v, 1, my_row, bias, lane);
      }
      if (!ok) break;
      if (ragged) {
        __syncwarp();
        if (live) ragged_store<FORM == kWords>(p.D, p.M, p.N, row0, c0, stage_smem, lane);
        continue;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (live) tma_store_2d(&tmD, stage_smem, c0, row0);
        bulk_commit_group();
      }
    }
    if (lane == 0) {
      if (full && !ragged && !ok) {  // C's block may still be on its way into the staging tile
        const long long t0 = clock64();
        while (!mbar_try_wait(c_bar(drain), it & 1) && clock64() - t0 < 400000000LL) {
        }
      }
      bulk_wait_group_read_0();
    }
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

using Kernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Params);

}  // namespace

bool run_product_pair(const Problem &pb, cudaStream_t stream) {
  static const Kernel kernels[] = {gemm_mxf4_pair_kernel<kNone>,        gemm_mxf4_pair_kernel<kRow>,
                                   gemm_mxf4_pair_kernel<kFull>,        gemm_mxf4_pair_kernel<kRow | kGelu>,
                                   gemm_mxf4_pair_kernel<kFull | kGelu>, gemm_mxf4_pair_kernel<kAny>,
                                   gemm_mxf4_pair_kernel<kRagged>,       gemm_mxf4_pair_kernel<kWords>};
  const bool units = pb.alpha == 1.f && (pb.c_mode == 0 || pb.beta == 1.f);
  const bool ragged = pb.N % 8 != 0;
  const bool words = pb.N % 2 == 0 && (reinterpret_cast<uintptr_t>(pb.C) | reinterpret_cast<uintptr_t>(pb.D)) % 4 == 0;
  // GELU without C runs as with a row of zeros: without the reads between them, its steps were taken up
  // before the shared columns were given back (32768 x 4096 x 1024 111 us, with the zeros 96).
  const Kernel kernel = kernels[ragged ? (words ? 7 : 6) : !units ? 5 : pb.act ? (pb.c_mode == 1 ? 4 : 3) : pb.c_mode == 0 ? 0 : pb.c_mode == 2 ? 1 : 2];
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
  static std::atomic<int> max_pairs[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  int pairs = max_pairs[dev].load(std::memory_order_acquire);
  if (pairs == 0) {
    for (const Kernel k : kernels)
      if (!check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes),
                      "cudaFuncSetAttribute(4-bit product on pairs)"))
        return false;
    // How many CTA pairs the device can hold at once (pairs need neighbouring SMs).
    cfg.gridDim = dim3(2 * (sm_count() / 2));
    if (cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg) != cudaSuccess || pairs <= 0) {
      cudaGetLastError();
      pairs = sm_count() / 2;
    }
    max_pairs[dev].store(pairs, std::memory_order_release);
  }
  const int64_t pitch = pb.blocks * 8;  // in two-byte elements, what the tensor maps count in
  const int64_t tile_cols = tile_cols_of(pb.blocks);
  CUtensorMap tmA, tmB, tmSA, tmSB, tmC, tmD;
  if (!gemm::make_tensor_map_2d(pb.A, pitch, pb.M, kStepBytes / 2, kHalf, &tmA) ||
      !gemm::make_tensor_map_2d(pb.B, pitch, pb.N, kStepBytes / 2, kHalf, &tmB) ||
      !gemm::make_tensor_map_scales(pb.scales_a, tile_cols, tile_rows_of(pb.M), kStepTiles, 1, &tmSA) ||
      !gemm::make_tensor_map_scales(pb.scales_b, tile_cols, tile_rows_of(pb.N), kStepTiles, 2, &tmSB))
    return false;
  tmD = tmA;  // not used when the rows are ragged
  if (!ragged && !gemm::make_tensor_map_2d(pb.D, pb.N, pb.M, 64, 32, &tmD)) return false;
  tmC = tmD;
  if (!ragged && pb.c_mode == 1 && pb.C != pb.D && !gemm::make_tensor_map_2d(pb.C, pb.N, pb.M, 64, 32, &tmC)) return false;
  Params p = {};
  p.C = pb.C;
  p.D = pb.D;
  p.alpha = pb.alpha;
  p.beta = pb.beta;
  p.c_mode = pb.c_mode;
  p.act = pb.act;
  p.M = static_cast<int>(pb.M);
  p.N = static_cast<int>(pb.N);
  p.steps = static_cast<int>((pb.blocks + kStepBlocks - 1) / kStepBlocks);
  p.n_blocks = static_cast<int>((pb.N + BN - 1) / BN);
  p.b_early = pb.b_const ? 1 : 0;
  p.status = device_status_word();
  const int64_t tiles = (pb.M + BM - 1) / BM * p.n_blocks;
  if (tiles > INT32_MAX - kMaxPairs) {
    set_error(HOM_ERR_UNSUPPORTED, "4-bit product: more than 2^31 output tiles");
    return false;
  }
  p.tiles = static_cast<int>(tiles);
  if (p.tiles < pairs) pairs = p.tiles;
  // Keeping A saves half of what is pulled through L2, but lets the pairs drift apart; measured with
  // and without, in us: 32768 x 4096 x 1024 68 / 76, 131072 x 4096 x 1024 with GELU and a row of C
  // 338 / 359, 32768 x 2304 x 768 41.0 / 43.2; with a matrix C, whose tiles are read as well,
  // 16384 x 4096 x 1024 55.3 / 54.2, 32768 x 1024 x 1024 32.4 / 31.4, 32768 x 768 x 768 26.3 / 25.9.
  p.resident = p.steps <= kStages && p.tiles >= 2 * pairs && pb.c_mode != 1 ? 1 : 0;

  cfg.gridDim = dim3(2 * pairs);
  LaunchScope scope(kOpGemm, product_flops(pb), product_bytes(pb));
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmSA, tmSB, tmC, tmD, p),
                    "4-bit product launch (CTA pairs)");
}

}  // namespace mxf4
}  // namespace hom
