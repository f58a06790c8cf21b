// Product of two microscaled 4-bit matrices (format: mxf4_sm100.cuh) on the block-scaled tensor
// path, for problems with few output tiles: D = act(alpha * A.B^T + beta * C), fp32 accumulation,
// fp16 C and D.  And the choice between this form and the others.
//
// A 128 x 64 tile of D belongs to a cluster of one, two or four CTAs that share its K range.  A K
// step is 256 values: 128 bytes of codes a row, fetched by TMA into 128-byte-swizzled tiles like the
// fp16 kernels' 64 values, and two scale tiles for each operand, which tcgen05.cp takes from shared
// to tensor memory right before the four MMAs that use them.  Zeros that TMA fills
// in beyond the matrix (codes 0, scales 2^-127) add nothing.  A stage of the ring has scales of its
// own in tensor memory: that the stage was filled again says that the MMAs of its last use, and
// their reads of the scales, are over.
//
// The partial tiles are exchanged SM to SM as in the fp16 cluster kernel (gemm_cluster_sm100.cu):
// CTA r owns rows [r, r + 1) * ceil(rows / parts) of the tile, every CTA stores its part of them
// into the owner's shared memory, and after a cluster barrier the owner adds the parts in part order
// (bit-identical from run to run), applies the epilogue and writes full rows.  A CTA that has its tile
// to itself passes it through its shared memory the same way, to write full rows.
//
// What bounds it is latency: launch, first loads, exchange and store one after the other.  128 x 768
// x 768 takes 5900 cycles from entry to exit: 1500 until the previous kernel is waited for, 2400 for
// the first loads and three steps, 800 to take the accumulator to shared memory, 1200 for sums,
// epilogue and stores.  (With a branch, a loop and a copy of the GELU for every piece of eight values
// the last were 3400.)  A further step takes 0.2 us, the rate at which L2 feeds one SM.
//
//   warp 0  TMA producer      warp 1  tensor memory, scale copies, MMA issue
//   warps 2-9  accumulator exchange and epilogue
#include <atomic>
#include <type_traits>

#include "gemm_sm100.cuh"
#include "mxf4_epilogue.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

using namespace hom::ptx;

namespace {

constexpr int BM = 128, BN = 64;
constexpr int kStepBytes = 128;                        // of a row of codes: 256 values
constexpr int kStepBlocks = 2 * kStepBytes / kBlock;   // 8
constexpr int kStepTiles = kStepBlocks / kTileBlocks;  // 2 scale tiles
constexpr int kStages = 4;
constexpr int kExchangeThreads = 256;
constexpr int kThreads = 64 + kExchangeThreads;
constexpr uint32_t kABytes = BM * kStepBytes, kBBytes = BN * kStepBytes;
constexpr uint32_t kScaleBytes = kStepTiles * kTileBytes;
constexpr uint32_t kStageBytes = kABytes + kBBytes + 2 * kScaleBytes;
constexpr uint32_t kRecv = kStages * kStageBytes;
constexpr uint32_t kBars = kRecv + BM * BN * 4;  // parts * ceil(rows / parts) <= 128 for 1, 2 and 4 parts
constexpr uint32_t kScaleCols = 4 * kStepTiles;  // tensor-memory columns of one operand's scales
constexpr uint32_t kTmemCols = 128;
// All that a CTA can have: no CTA of another kernel may sit beside one of this (gemm_cluster_sm100.cu).
constexpr uint32_t kSmemBytes = 227 * 1024;
static_assert(kStageBytes % 1024 == 0, "swizzled tiles start on 1024 bytes");
static_assert(kBars + 8 * (2 * kStages + 1) + 16 + 1024 <= kSmemBytes, "exceeds a CTA's shared memory");
static_assert(BN + kStages * 2 * kScaleCols <= kTmemCols, "accumulator and scales exceed the allocation");

struct Params {
  const __half *C;
  __half *D;
  float alpha, beta;
  int c_mode, act;
  int M, N, steps, n_blocks;
  int b_early;  // B is a declared constant: request its tiles before griddepcontrol.wait
  int *status;
  int fill[8];
};
static_assert(quick_to_launch<Params>, "see launch_pdl");  // (the tensor maps before it are whole 64 bytes)

__device__ __forceinline__ uint32_t cluster_nctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Where a row of the exchanged tile has its 16-byte chunk: neither the stores (a chunk of 32 rows) nor
// the loads (every other chunk of a row, first the even, then the odd ones) meet in a bank.
__device__ __forceinline__ uint32_t place_of(int chunk, int row) {
  return static_cast<uint32_t>(chunk ^ (row & 7) ^ (chunk >> 3));
}

// Of PAIRS pairs of sums and of C's values.  All of them take each step together: one test of `act`
// with one copy of its code behind it, and the rest in a straight line.
template <int PAIRS>
__device__ __forceinline__ void epilogue2(const Params &p, float2 (&v)[PAIRS], const float2 (&c)[PAIRS]) {
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    v[i] = __fmul2_rn(make_float2(p.alpha, p.alpha), v[i]);
    if (p.c_mode != 0) v[i] = __ffma2_rn(make_float2(p.beta, p.beta), c[i], v[i]);
  }
  if (p.act == 1) gelu2(v);
}

// ALIGNED: N % 8 == 0, rows of C and D travel in 16-byte pieces; otherwise element by element,
// neighbouring threads at neighbouring columns.  (Two columns a lane, as one where the row's address
// allows it: the choice between two kinds of load keeps them from being under way together, 385 x
// 1001 x 808 7.1 us.)
template <bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 1)
gemm_mxf4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  auto full_bar = [&](int s) { return smem_base + kBars + 8u * s; };
  auto empty_bar = [&](int s) { return smem_base + kBars + 8u * (kStages + s); };
  const uint32_t acc_bar = smem_base + kBars + 8u * (2 * kStages);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kBars + 8 * (2 * kStages + 1));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = static_cast<int>(cluster_nctas()), part = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / parts;
  const int m0 = tile / p.n_blocks * BM, n0 = tile % p.n_blocks * BN;
  const int first = part * p.steps / parts;
  const int steps = (part + 1) * p.steps / parts - first;  // >= 1: the launcher keeps parts <= steps

  if (threadIdx.x == 64) {
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmSB);
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmSA);
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
  // Cluster barrier, phase 1: "this CTA runs"; its shared memory may be written by its peers.
  // Every thread of every CTA arrives and waits exactly once per phase, on error paths too.  (A CTA
  // that has the tile to itself does without: its parts go from warp to warp.)
  const bool alone = parts == 1;
  if (!alone) cluster_arrive();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      auto load_b = [&](uint32_t dst, uint32_t bar, int i) {
        tma_load_2d(dst + kABytes, &tmB, bar, (first + i) * (kStepBytes / 2), n0);
        tma_load_3d(dst + kABytes + kBBytes + kScaleBytes, &tmSB, bar, 0, (first + i) * kStepTiles, n0 / kTileRows);
      };
      const int early = min(steps, kStages);
      for (int i = 0; i < early; ++i) {
        mbar_arrive_expect_tx(full_bar(i), kStageBytes);
        if (p.b_early) load_b(smem_base + i * kStageBytes, full_bar(i), i);
      }
      pdl_wait();
      bool ok = true;
      int armed = early;
      for (int i = 0; i < steps; ++i) {
        const int s = i % kStages;
        const uint32_t dst = smem_base + s * kStageBytes;
        if (i >= early) {
          ok = mbar_wait(empty_bar(s), ((i / kStages) & 1) ^ 1, abort_flag, p.status, kDevWaitTimeoutProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(full_bar(s), kStageBytes);
          ++armed;
        }
        if (i >= early || !p.b_early) load_b(dst, full_bar(s), i);
        tma_load_2d(dst, &tmA, full_bar(s), (first + i) * (kStepBytes / 2), m0);
        tma_load_3d(dst + kABytes + kBBytes, &tmSA, full_bar(s), 0, (first + i) * kStepTiles, m0 / kTileRows);
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
    if (!alone) {
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      // the tile may start in the middle of a scale tile
      const uint32_t shift = n0 % kTileRows / 32;
      bool ok = true;
      for (int i = 0; i < steps; ++i) {
        const int s = i % kStages;
        ok = mbar_wait<true>(full_bar(s), (i / kStages) & 1, abort_flag, p.status, kDevWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t src = smem_base + s * kStageBytes;
        const uint32_t scales = tmem_base + BN + s * 2 * kScaleCols;
#pragma unroll
        for (int t = 0; t < 2 * kStepTiles; ++t)
          tc_copy_scales(scales + t * 4, make_smem_desc_scales(src + kABytes + kBBytes + t * kTileBytes));
        const uint64_t da = make_smem_desc_sw128(src, 16, 1024), db = make_smem_desc_sw128(src + kABytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < 2 * kStepTiles; ++k)
          tc_mma_mxf4_ss(tmem_base, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32),
                         k & 1 ? make_idesc_mxf4(BM, BN, 1) : make_idesc_mxf4(BM, BN, 0), scales + (k >> 1) * 4,
                         scales + kScaleCols + (k >> 1) * 4 + shift, i != 0 || k != 0 ? 1u : 0u);
        tc_commit(empty_bar(s));
      }
      if (ok) tc_commit(acc_bar);
    }
    __syncwarp();
    if (!alone) {
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    // ------------------------------------------- accumulator exchange and epilogue
    const int rows = min(BM, p.M - m0);               // rows of the tile inside the matrix
    const int rows_per = (rows + parts - 1) / parts;  // rows each CTA of the cluster finishes
    const int row_first = part * rows_per;
    const int my_rows = max(0, min(rows_per, rows - row_first));
    const int t = threadIdx.x - 64;
    constexpr int kPieces = BN / 8;  // 8-column pieces of an output row
    constexpr int kPieceRows = kExchangeThreads / kPieces;  // 32 rows of pieces at a time
    constexpr int kTasks = ALIGNED ? BM / kPieceRows : 1;
    static_assert(kPieceRows == 32 && kPieceRows / (kExchangeThreads / 32) == 4, "four rows to a warp, four times");
    // not aligned: one column per thread and every fourth row
    constexpr int kRowStep = kExchangeThreads / BN, kRows = BM / kRowStep;
    const int column = t % BN, first_local = t / BN;
    unsigned short c_bits[ALIGNED ? 1 : kRows];

    pdl_wait();  // C may be produced, and D still read, by the previous kernel
    uint4 cval[kTasks];
    if constexpr (ALIGNED) {
#pragma unroll
      for (int i = 0; i < kTasks; ++i) {
        cval[i] = make_uint4(0, 0, 0, 0);
        const int row = (t + i * kExchangeThreads) / kPieces, col = n0 + (t + i * kExchangeThreads) % kPieces * 8;
        if (p.c_mode != 0 && row < my_rows && col < p.N)
          cval[i] = *reinterpret_cast<const uint4 *>(
              p.C + (p.c_mode == 1 ? static_cast<long long>(m0 + row_first + row) * p.N : 0) + col);
      }
    } else {
      const int col = n0 + column;
      const unsigned short *c = reinterpret_cast<const unsigned short *>(p.C) + col +
                                (p.c_mode == 1 ? static_cast<long long>(m0 + row_first + first_local) * p.N : 0);
      const long long step = p.c_mode == 1 ? static_cast<long long>(kRowStep) * p.N : 0;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        c_bits[i] = p.c_mode != 0 && first_local + i * kRowStep < my_rows && col < p.N ? *c : 0;
        c += step;
      }
    }
    bool ok = mbar_wait(acc_bar, 0, abort_flag, p.status, kDevWaitTimeoutEpilogue);
    ok = __all_sync(0xffffffffu, ok);
    if (!alone) cluster_wait();  // phase 1: every CTA of the cluster runs
    if (ok) {
      tc_fence_after_sync();
      const int quarter = warp & 3;
      const int row = quarter * 32 + lane;
      const int col_begin = ((warp - 2) >> 2) * (BN / 2);
      if (quarter * 32 < rows) {  // warp-uniform: the accumulator read is warp-collective
        const int owner = min(row / rows_per, parts - 1), local = row - owner * rows_per;
        const uint32_t dst =
            map_to_cta(smem_base + kRecv + static_cast<uint32_t>(part * rows_per + (row < rows ? local : 0)) * (BN * 4),
                       static_cast<uint32_t>(owner));
#pragma unroll
        for (int h = 0; h < BN / 64; ++h) {
          uint32_t acc[32];
          tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col_begin + h * 32, acc);
          tmem_ld_wait();
          if (row < rows) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t chunk = place_of((col_begin + h * 32) / 4 + j, local);
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + chunk * 16), "r"(acc[4 * j]),
                           "r"(acc[4 * j + 1]), "r"(acc[4 * j + 2]), "r"(acc[4 * j + 3])
                           : "memory");
            }
          }
        }
        tc_fence_before_sync();
      }
    }
    if (alone) {
      asm volatile("bar.sync 1, %0;" ::"n"(kExchangeThreads) : "memory");
    } else {
      cluster_arrive();  // phase 2: the parts are delivered
      cluster_wait();
    }
    if (ok) {
      // the sums of the parts, in part order
      if constexpr (ALIGNED) {
        const int piece = t % kPieces, col = n0 + piece * 8;
        auto finish = [&](auto count) {  // of the pieces that this thread may have
          constexpr int kCount = decltype(count)::value;
          float2 v[kCount * 4], c[kCount * 4];
#pragma unroll
          for (int i = 0; i < kCount * 4; ++i) {
            v[i] = make_float2(0.f, 0.f);
            c[i] = __half22float2(reinterpret_cast<const __half2 *>(&cval[i / 4])[i % 4]);
          }
          for (int q = 0; q < parts; ++q) {
            float f[kCount * 8];
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
              const int local = min(t / kPieces + i * kPieceRows, rows_per - 1);
#pragma unroll
              for (int h = 0; h < 2; ++h)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(f[8 * i + 4 * h]), "=f"(f[8 * i + 4 * h + 1]), "=f"(f[8 * i + 4 * h + 2]),
                               "=f"(f[8 * i + 4 * h + 3])
                             : "r"(smem_base + kRecv + static_cast<uint32_t>(q * rows_per + local) * (BN * 4) +
                                   place_of(2 * piece + h, local) * 16)
                             : "memory");
            }
#pragma unroll
            for (int i = 0; i < kCount * 4; ++i) v[i] = __fadd2_rn(v[i], make_float2(f[2 * i], f[2 * i + 1]));
          }
          epilogue2(p, v, c);
#pragma unroll
          for (int i = 0; i < kCount; ++i) {
            const int local = t / kPieces + i * kPieceRows;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __half2 h = __floats2half2_rn(v[4 * i + j].x, v[4 * i + j].y);
              w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
            if (local < my_rows && col < p.N)
              *reinterpret_cast<uint4 *>(p.D + static_cast<long long>(m0 + row_first + local) * p.N + col) =
                  make_uint4(w[0], w[1], w[2], w[3]);
          }
        };
        if (rows_per > 2 * kPieceRows) finish(std::integral_constant<int, 4>());
        else if (rows_per > kPieceRows) finish(std::integral_constant<int, 2>());
        else if (warp - 2 < (my_rows + 3) / 4) finish(std::integral_constant<int, 1>());
      } else {
        auto finish = [&](auto count) {
          constexpr int kCount = decltype(count)::value;
          float2 v[kCount / 2], c[kCount / 2];  // of two of the thread's rows
#pragma unroll
          for (int i = 0; i < kCount / 2; ++i) {
            v[i] = make_float2(0.f, 0.f);
            c[i] = make_float2(__half2float(__ushort_as_half(c_bits[2 * i])), __half2float(__ushort_as_half(c_bits[2 * i + 1])));
          }
          for (int q = 0; q < parts; ++q) {
            float f[kCount];
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
              const int local = min(first_local + i * kRowStep, rows_per - 1);
              asm volatile("ld.shared.f32 %0, [%1];"
                           : "=f"(f[i])
                           : "r"(smem_base + kRecv + static_cast<uint32_t>(q * rows_per + local) * (BN * 4) +
                                 place_of(column >> 2, local) * 16 + (column & 3) * 4)
                           : "memory");
            }
#pragma unroll
            for (int i = 0; i < kCount / 2; ++i) v[i] = __fadd2_rn(v[i], make_float2(f[2 * i], f[2 * i + 1]));
          }
          epilogue2(p, v, c);
          const int col = n0 + column;
          __half *d = p.D + static_cast<long long>(m0 + row_first + first_local) * p.N + col;
#pragma unroll
          for (int i = 0; i < kCount; ++i) {
            if (first_local + i * kRowStep < my_rows && col < p.N) *d = __float2half_rn(i & 1 ? v[i / 2].y : v[i / 2].x);
            d += static_cast<long long>(kRowStep) * p.N;
          }
        };
        if (rows_per > BM / 2) finish(std::integral_constant<int, kRows>());
        else if (rows_per > BM / 4) finish(std::integral_constant<int, kRows / 2>());
        else finish(std::integral_constant<int, kRows / 4>());
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <bool ALIGNED>
bool launch(const Problem &pb, int parts, cudaStream_t stream) {
  static std::atomic<bool> ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  auto kernel = gemm_mxf4_kernel<ALIGNED>;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (!check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes),
                    "cudaFuncSetAttribute(4-bit product)"))
      return false;
    ready[dev].store(true, std::memory_order_release);
  }
  const int64_t pitch = pb.blocks * 8;  // in two-byte elements, what the tensor maps count in
  const int64_t tile_cols = tile_cols_of(pb.blocks);
  CUtensorMap tmA, tmB, tmSA, tmSB;
  if (!gemm::make_tensor_map_2d(pb.A, pitch, pb.M, kStepBytes / 2, BM, &tmA) ||
      !gemm::make_tensor_map_2d(pb.B, pitch, pb.N, kStepBytes / 2, BN, &tmB) ||
      !gemm::make_tensor_map_scales(pb.scales_a, tile_cols, tile_rows_of(pb.M), kStepTiles, 1, &tmSA) ||
      !gemm::make_tensor_map_scales(pb.scales_b, tile_cols, tile_rows_of(pb.N), kStepTiles, 1, &tmSB))
    return false;
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
  const int64_t ctas = (pb.M + BM - 1) / BM * p.n_blocks * parts;
  LaunchScope scope(kOpGemm, product_flops(pb), product_bytes(pb));
  return check_cuda(launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmemBytes, stream,
                               static_cast<unsigned>(parts), tmA, tmB, tmSA, tmSB, p),
                    "4-bit product launch");
}

}  // namespace

// Measured per call in a chain of calls (us):
//   one wave of 128 x 64 tiles against the pairs' 256 x 256: 1024 x 1024 x 1024 3.7 / 5.7,
//   1024 x 1024 x 4096 6.1 / 9.3, 512 x 2304 x 768 3.6 / 5.5; more than one wave: 2048 x 768 x 768
//   6.5 / 5.4, 512 x 4096 x 1024 7.2 / 5.8;
//   K in one, two and four parts, 128 rows: 1024 columns and K = 1024 3.3 / 3.8 / 4.1, 2560 4.4 / 4.3 /
//   4.5, 4096 5.6 / 4.9 / 4.7, 8192 8.8 / 6.5 / 5.4; 1792 columns and K = 4096 5.6 / 5.0 / 5.4, 4096
//   columns 5.7 / 5.6 / 11.2 (the last no longer in one wave: clusters of four need SMs of one GPC);
//   32 rows, which are little to exchange, 256 columns and K = 1536 3.2 / 3.1 / 3.1, 2048 3.6 / 3.3 / 3.1.
bool run_product(const Problem &pb, cudaStream_t stream) {
  if (pb.M <= kMaxFewRows) return run_product_rows(pb, stream);
  const int64_t tiles = (pb.M + BM - 1) / BM * ((pb.N + BN - 1) / BN), sms = sm_count();
  if (tiles > sms) return run_product_pair(pb, stream);
  const int64_t steps = (pb.blocks + kStepBlocks - 1) / kStepBlocks;
  const bool few_rows = pb.M <= 32;
  int parts = 1;
  if (2 * tiles <= sms && steps >= (few_rows ? 6 : 3 * tiles <= sms ? 10 : 16)) parts = 2;
  if (8 * tiles <= sms && steps >= (few_rows ? 8 : 12)) parts = 4;
  return pb.N % 8 == 0 ? launch<true>(pb, parts, stream) : launch<false>(pb, parts, stream);
}

}  // namespace mxf4
}  // namespace hom
