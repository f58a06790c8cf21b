// Host interface of the microscaled 4-bit floating-point operators: conversion (mxf4_convert.cu)
// and product (gemm_mxf4_sm100.cu).
//
// The format (the open MX one): 32 consecutive values along K share a power of two 2^(s - 127),
// s an unsigned byte (255: the block is NaN); each value is a 4-bit number with one sign, two
// exponent and one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.
// Codes: [rows, 16 * ceil(K / 32)] bytes, the even value of a pair in the low half; values beyond
// K are 0.  Scales: [ceil(rows / 128), ceil(blocks / 4), 512] bytes, byte
// (r % 32) * 16 + (r / 32) % 4 * 4 + b % 4 of tile (r / 128, b / 4) belongs to row r and block b:
// the order in which the tensor cores take a 128-row operand's scales, so that a tile goes from
// global to tensor memory without being touched.  Bytes of rows and blocks beyond the matrix are 0.
#pragma once

#include "hom_common.cuh"

namespace hom {
namespace mxf4 {

constexpr int kBlock = 32;            // values that share a scale
constexpr int kTileRows = 128;        // rows and
constexpr int kTileBlocks = 4;        // blocks of one scale tile
constexpr int kTileBytes = 512;

inline int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }
inline int64_t tile_rows_of(int64_t rows) { return (rows + kTileRows - 1) / kTileRows; }
inline int64_t tile_cols_of(int64_t blocks) { return (blocks + kTileBlocks - 1) / kTileBlocks; }

// x [rows, cols] -> codes, scales; with `transposed` x is [cols, rows] and the blocks still run
// along cols.
template <typename T>
bool quantize(const T *x, bool transposed, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols,
              cudaStream_t stream);
// out [rows, cols] <- codes, scales
template <typename T>
bool dequantize(const uint8_t *codes, const uint8_t *scales, T *out, int64_t rows, int64_t cols,
                cudaStream_t stream);

// D = act(alpha * A.B^T + beta * C); A [M, 32 * blocks], B [N, 32 * blocks].
struct Problem {
  int64_t M = 0, N = 0, blocks = 0;
  const uint8_t *A = nullptr, *scales_a = nullptr;
  const uint8_t *B = nullptr, *scales_b = nullptr;
  bool b_const = false;  // B and its scales lie in declared constant ranges
  const __half *C = nullptr;
  int c_mode = 0;  // 0 none, 1 full [M, N] (may alias D), 2 length-N row broadcast
  __half *D = nullptr;
  float alpha = 1.f, beta = 0.f;
  int act = 0;  // 1 = erf GELU
};
// What the product cannot do without.
inline double product_flops(const Problem &pb) { return 64.0 * pb.M * pb.N * pb.blocks; }
inline double product_bytes(const Problem &pb) {
  return (static_cast<double>(pb.M) + pb.N) * pb.blocks * 17.0 + 2.0 * pb.M * pb.N * (pb.c_mode == 1 ? 2 : 1) +
         (pb.c_mode == 2 ? 2.0 * pb.N : 0.0);
}
bool run_product(const Problem &pb, cudaStream_t stream);
// For one or two rows (gemm_mxf4_rows.cu).
constexpr int64_t kMaxFewRows = 2;
bool run_product_rows(const Problem &pb, cudaStream_t stream);
// On persistent CTA pairs, 256 x 256 tiles (gemm_mxf4_pair_sm100.cu).
bool run_product_pair(const Problem &pb, cudaStream_t stream);

}  // namespace mxf4
}  // namespace hom
