// Product of one or two rows with a microscaled 4-bit weight (format: mxf4_sm100.cuh): the single
// token's form.  It reads the weight once and computes little, and what it takes is latency, so it
// does without tensor memory, TMA and barriers: a warp takes a row of B, a lane one block of 32
// values out of 32 (16 bytes, a warp 512 contiguous ones).
//
// Measured per call in a chain of calls, against the tensor-core kernel (us): one row of 768 values by
// 768 columns 1.9 / 2.7, two rows of 1024 by 4096 2.7 / 3.5.  The tensor-core kernel's time does not
// grow with the rows, this one's does.  Two or four rows of B for a warp were slower.
//
// Arithmetic is exact until the blocks are added: a product of two codes is at most 36 in quarters,
// so eight of them add up to at most 1152 quarters, which fp16 holds exactly (11 bits); the four
// sums of a block are added in fp32, multiplied by the two powers of two, and summed over the
// blocks in fp32 in a fixed order.
#include "mxf4_epilogue.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

namespace {

constexpr int kWarps = 8;

struct Params {
  const uint8_t *a, *scales_a, *b, *scales_b;
  const __half *c;
  __half *d;
  long long c_pitch;  // 0: one row for all
  float alpha, beta;
  int act;
  int n, blocks, tile_cols;
  int b_early;  // B is a declared constant: read before griddepcontrol.wait
};
static_assert(quick_to_launch<Params>, "see launch_pdl");

__device__ __forceinline__ void decode32(const uint4 &codes, __half2 (&v)[16]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h[4];
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t"
        "}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w[i]));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * i + j] = *reinterpret_cast<const __half2 *>(&h[j]);
  }
}

__device__ __forceinline__ int scale_at(const uint8_t *scales, int tile_cols, long long row, int block) {
  return scales[((row / kTileRows) * tile_cols + block / kTileBlocks) * kTileBytes + row % 32 * 16 + row / 32 % 4 * 4 +
                block % kTileBlocks];
}

// x * 2^(sa - 127) * 2^(sb - 127), in two steps whose exponents are the halves of the sum: rounded or
// out of range only where the result is.
__device__ __forceinline__ float apply_scales(float x, int sa, int sb) {
  if (sa == 255 || sb == 255) return __int_as_float(0x7fffffff);
  const int e = sa + sb - 254, e1 = e >> 1, e2 = e - e1;
  return x * __int_as_float((127 + e1) << 23) * __int_as_float((127 + e2) << 23);
}

template <int M>
__global__ void __launch_bounds__(32 * kWarps) gemm_mxf4_rows_kernel(const Params p) {
  hom::ptx::pdl_launch_dependents();
  if (!p.b_early) hom::ptx::pdl_wait();
  const int lane = threadIdx.x & 31;
  const int n = static_cast<int>(blockIdx.x) * kWarps + static_cast<int>(threadIdx.x >> 5);
  // blocks per lane whose loads are under way at once: as many as leave the registers for four CTAs
  constexpr int kInFlight = M == 1 ? 4 : 2;
  uint4 codes[kInFlight];
  int scale[kInFlight];
  auto load = [&](const uint8_t *from, const uint8_t *scales, int row, int block, uint4 *code, int *s) {
    *code = make_uint4(0, 0, 0, 0);
    *s = 0;
    if (block < p.blocks) {
      *code = *reinterpret_cast<const uint4 *>(from + (static_cast<long long>(row) * p.blocks + block) * 16);
      *s = scale_at(scales, p.tile_cols, row, block);
    }
  };
  if (n < p.n) {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) load(p.b, p.scales_b, n, lane + 32 * i, &codes[i], &scale[i]);
  }
  if (p.b_early) hom::ptx::pdl_wait();
  if (n >= p.n) return;

  float sum[M];
#pragma unroll
  for (int m = 0; m < M; ++m) sum[m] = 0.f;
  for (int first = lane; first - lane < p.blocks; first += 32 * kInFlight) {
    uint4 a_codes[kInFlight][M];
    int a_scale[kInFlight][M];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (first != lane) load(p.b, p.scales_b, n, first + 32 * i, &codes[i], &scale[i]);
#pragma unroll
      for (int m = 0; m < M; ++m) load(p.a, p.scales_a, m, first + 32 * i, &a_codes[i][m], &a_scale[i][m]);
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (first - lane + 32 * i >= p.blocks) break;  // the same for the whole warp
      __half2 bv[16];
      decode32(codes[i], bv);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        __half2 av[16];
        decode32(a_codes[i][m], av);
        __half2 s0 = __hmul2(av[0], bv[0]), s1 = __hmul2(av[8], bv[8]);
#pragma unroll
        for (int j = 1; j < 8; ++j) {
          s0 = __hfma2(av[j], bv[j], s0);
          s1 = __hfma2(av[8 + j], bv[8 + j], s1);
        }
        const float2 f0 = __half22float2(s0), f1 = __half22float2(s1);
        sum[m] += apply_scales((f0.x + f0.y) + (f1.x + f1.y), a_scale[i][m], scale[i]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], o);
    if (lane == m) {
      float v = p.alpha * sum[m];
      if (p.c != nullptr) v = fmaf(p.beta, __half2float(p.c[m * p.c_pitch + n]), v);
      if (p.act == 1) {
        float2 x[1] = {make_float2(v, 0.f)};
        gelu2(x);
        v = x[0].x;
      }
      p.d[static_cast<long long>(m) * p.n + n] = __float2half_rn(v);
    }
  }
}

}  // namespace

bool run_product_rows(const Problem &pb, cudaStream_t stream) {
  Params p = {};
  p.a = pb.A;
  p.scales_a = pb.scales_a;
  p.b = pb.B;
  p.scales_b = pb.scales_b;
  p.c = pb.c_mode == 0 ? nullptr : pb.C;
  p.d = pb.D;
  p.c_pitch = pb.c_mode == 1 ? pb.N : 0;
  p.alpha = pb.alpha;
  p.beta = pb.beta;
  p.act = pb.act;
  p.n = static_cast<int>(pb.N);
  p.blocks = static_cast<int>(pb.blocks);
  p.tile_cols = static_cast<int>(tile_cols_of(pb.blocks));
  p.b_early = pb.b_const ? 1 : 0;
  const unsigned grid = static_cast<unsigned>((pb.N + kWarps - 1) / kWarps);
  LaunchScope scope(kOpGemm, product_flops(pb), product_bytes(pb));
  return check_cuda(launch_pdl(pb.M == 1 ? gemm_mxf4_rows_kernel<1> : gemm_mxf4_rows_kernel<2>, dim3(grid),
                               dim3(32 * kWarps), 0, stream, 1, p),
                    "4-bit product launch (rows)");
}

}  // namespace mxf4
}  // namespace hom
