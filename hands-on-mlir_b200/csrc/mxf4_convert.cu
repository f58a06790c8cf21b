// Values to microscaled 4-bit floating point and back (format: mxf4_sm100.cuh).
//
// For a block of 32 values with largest magnitude a the scale is 2^(floor(log2 a) - 2), the power
// of two that puts a between 4 and 8, and every value over the scale is rounded to the nearest
// 4-bit number, ties to even, magnitudes above 6 to 6.  With the fp32 exponent field f of a the
// scale byte is max(f - 2, 0) and its reciprocal has the exponent field 254 - byte: both exact, so
// is the product with the value (a result too small for fp32 is far below the 0.25 that rounds to
// 0), and the only rounding is the one to four bits.
//
// Both directions move bytes and nothing else counts: 2.53 (fp16) or 4.53 (fp32) a value.
#include "bandwidth_kernels.cuh"
#include "mxf4_sm100.cuh"
#include "ptx_sm100.cuh"

namespace hom {
namespace mxf4 {

namespace {

constexpr int kWarps = 8;
constexpr int kLaneValues = 8;                     // consecutive values of a row that a lane holds
constexpr int kSegment = 32 * kLaneValues;         // a warp's part of a row: 8 blocks, 2 scale tiles wide
constexpr int kRowStep = kTileRows / 4;            // a warp works on rows r, r + 32, r + 64, r + 96

struct Params {
  const void *values;  // of the matrix that is read or written
  uint8_t *codes, *scales;
  long long rows, units;
  int cols, blocks;
  uint32_t segments;
  int fill[9];
};
static_assert(quick_to_launch<Params>, "see launch_pdl");

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale byte of a block whose largest magnitude has these bits (NaN and infinity compare
// above every number).
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const uint32_t field = bits >> 23;
  return field == 255u ? 255u : field < 2u ? 0u : field - 2u;
}

__device__ __forceinline__ float reciprocal_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0u : (254u - byte) << 23);
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fffffffu : byte << 23);
}

// Eight values to eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ void decode8(uint32_t codes, float (&v)[8]) {
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
      : "r"(codes));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(__half *p, const float (&v)[8]) {
  uint4 raw;
  __half2 *h = reinterpret_cast<__half2 *>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<uint4 *>(p) = raw;
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store1(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(float *p, float v) { *p = v; }

// Eight consecutive values of a row as they lie in memory, the bits of their largest magnitude as
// fp32 (NaN and infinity above all numbers), and their codes.
template <typename T>
struct Eight;
template <>
struct Eight<__half> {
  uint4 raw;
  __device__ __forceinline__ void load(const __half *p) { raw = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    __half2 *h = reinterpret_cast<__half2 *>(&raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
  }
  __device__ __forceinline__ void clear() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void keep(int n) {  // the first n values, zeros behind them
    uint32_t *word = reinterpret_cast<uint32_t *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) word[i] = 2 * i + 1 < n ? word[i] : 2 * i < n ? word[i] & 0xffffu : 0u;
  }
  __device__ __forceinline__ uint32_t largest() const {
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return magnitude_bits(__half2float(__hmax_nan(__low2half(m), __high2half(m))));
  }
  __device__ __forceinline__ uint32_t encode(float inv) const {
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(h[j]);
      v[2 * j] = f.x * inv;
      v[2 * j + 1] = f.y * inv;
    }
    return encode8(v);
  }
};
template <>
struct Eight<float> {
  float v[8];
  __device__ __forceinline__ void load(const float *p) { load8(p, v); }
  __device__ __forceinline__ void set(const float (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = w[j];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) bits = max(bits, magnitude_bits(v[j]));
    return bits;
  }
  __device__ __forceinline__ uint32_t encode(float inv) const {
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = v[j] * inv;
    return encode8(s);
  }
};

// Eight fp16 values that lie `shift` elements after a 16-byte boundary, in the two 16-byte pieces
// from there on.
struct ShiftedEight {
  uint32_t word[8];
  __device__ __forceinline__ void load(const uint4 *p) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 piece = p[h];
      word[4 * h] = piece.x, word[4 * h + 1] = piece.y, word[4 * h + 2] = piece.z, word[4 * h + 3] = piece.w;
    }
  }
  __device__ __forceinline__ Eight<__half> down(int shift) {
    if (shift & 4)
#pragma unroll
      for (int i = 0; i < 6; ++i) word[i] = word[i + 2];
    if (shift & 2)
#pragma unroll
      for (int i = 0; i < 5; ++i) word[i] = word[i + 1];
    if (shift & 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) word[i] = __funnelshift_r(word[i], word[i + 1], 16);
    Eight<__half> v;
    v.raw = make_uint4(word[0], word[1], word[2], word[3]);
    return v;
  }
};

// One warp converts a segment of 256 columns of the rows r, r + 32, r + 64 and r + 96 of a
// 128-row group: four independent loads in flight, and the scales of the four rows are the 16
// consecutive bytes of a scale tile.  A lane holds eight values, four lanes a block.  ALIGNED: rows
// start on 16 bytes (cols % 8 == 0).  Otherwise, fp16: a lane reads the two 16-byte pieces that its
// values lie in and moves them down, 20011 x 777 values 15.7 us, 37.9 element by element.  fp32: the
// warp reads element by element, coalesced, and sorts the values through shared memory, 16.3 us; in
// 16-byte pieces 24.5, and by 4-byte asynchronous copies 19.6.  (Slower too: a persistent form that
// requests the next unit's values early, whose registers cost more loads in flight than it gains; and
// for fp16 one 16-byte piece a lane, the second by a shuffle from the neighbour, 21 to 28 us.)  The
// memory would need 6.0 us for the fp16 values and 10.8 for the fp32 ones: a lane requests 32 bytes for
// its 16, or single elements.
//
// What the rows kernel needs is many loads in flight, so its registers are held down: 65536 x 4096
// fp16 values 119 us with room for five CTAs on an SM, 112 for eight (6.0 TB/s); 20011 x 776 fp32
// values 13.0 with five, 13.5 with six, 26 (spills) with eight.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps, sizeof(T) == 2 ? (ALIGNED ? 8 : 5) : 5)
quantize_rows_kernel(const Params p) {
  const T *x = static_cast<const T *>(p.values);
  const long long rows = p.rows, units = p.units;
  const int cols = p.cols, blocks = p.blocks;
  const uint32_t segments = p.segments;
  constexpr bool kShifted = !ALIGNED && sizeof(T) == 2, kSorted = !ALIGNED && sizeof(T) == 4;
  __shared__ __align__(16) T sorted[kSorted ? kWarps : 1][kSorted ? kSegment : 8];
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long unit = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (unit >= units) return;
  const long long row_unit = units <= INT32_MAX ? static_cast<uint32_t>(unit) / segments : unit / segments;
  const int segment = static_cast<int>(unit - row_unit * segments);
  const long long group = row_unit / kRowStep;
  const int r = static_cast<int>(row_unit % kRowStep);
  const long long row0 = group * kTileRows + r;
  const int col = segment * kSegment + lane * kLaneValues;

  Eight<T> v[4];
  ShiftedEight pieces[kShifted ? 4 : 1];
  bool whole = false;  // kShifted: the pieces of all rows lie inside the matrix
  int shift = 0;       // the same for all four rows, which are 32 rows apart
  if constexpr (kShifted) {
    const long long begin = row0 * cols + segment * kSegment;
    const long long last = begin + min(3LL, (rows - 1 - row0) / kRowStep) * kRowStep * cols;
    whole = row0 < rows && begin >= 8 && last + kSegment + 8 <= rows * cols;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(x + begin) / 2) & 7;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + i * kRowStep;
    if constexpr (ALIGNED) {
      if (row < rows && col < cols) v[i].load(x + row * cols + col);
      else v[i].clear();
    } else if (kShifted && whole) {
      if (row < rows && col < cols) {
        pieces[i].load(reinterpret_cast<const uint4 *>(x + row * cols + col - shift));
      } else {
#pragma unroll
        for (int w = 0; w < 8; ++w) pieces[i].word[w] = 0;
      }
    } else {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = kShifted ? col + j : segment * kSegment + j * 32 + lane;
        w[j] = row < rows && c < cols ? to_float(x[row * cols + c]) : 0.f;
      }
      v[i].set(w);
    }
  }
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kSorted) {
      // value j * 32 + lane of the segment in slot j of the lane -> eight consecutive ones
      const T *mine = reinterpret_cast<const T *>(&v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sorted[warp][j * 32 + lane] = mine[j];
      __syncwarp();
      v[i].load(&sorted[warp][lane * kLaneValues]);
      __syncwarp();
    }
    if constexpr (kShifted) {
      if (whole) {
        v[i] = pieces[i].down(shift);
        if (cols - col < kLaneValues) v[i].keep(cols - col);
      }
    }
    uint32_t bits = v[i].largest();
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    const uint32_t byte = scale_byte(bits);
    const uint32_t packed = byte == 255u ? 0u : v[i].encode(reciprocal_scale(byte));
    const long long row = row0 + i * kRowStep;
    if (row < rows && col < blocks * kBlock)
      *reinterpret_cast<uint32_t *>(p.codes + row * (blocks * 16LL) + col / 2) = packed;
    // the bytes of four neighbouring blocks become the word of one scale tile
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    words[i] = word;
  }
  const int tile_cols = (blocks + kTileBlocks - 1) / kTileBlocks;
  const int tile = segment * 2 + (lane >> 4);
  if ((lane & 15) == 0 && tile < tile_cols)
    *reinterpret_cast<uint4 *>(p.scales + (group * tile_cols + tile) * kTileBytes + r * 16) =
        make_uint4(words[0], words[1], words[2], words[3]);
}

// x stored [cols, rows]: a thread owns one block of COLUMNS rows of the result, that is 32 values of
// as many columns of x, all of them in flight; neighbouring threads read neighbouring elements.  A
// CTA makes one scale tile, whose bytes it gathers in shared memory.  Two columns for fp16 (rows even,
// x on 4 bytes): a [4096, 4096] weight takes 13.4 us (3.2 TB/s: pieces of 256 bytes out of rows of
// 8 KB); with one column, 2-byte loads, 4097 rows of 4096 values 16.4.  fp32 [4096, 4096] 16.0 us, 4.7
// TB/s (pieces of 512 bytes).
//
// The scale tiles along K are the grid's second dimension, which ends at 65535.  LONG: the third takes
// what is beyond.  (An instantiation of its own: the loads are scheduled so finely that the additional
// index took [4096, 4096] from 13.4 to 15.6 us, and one dimension with a division to 15.0.)
constexpr int64_t kMaxGridY = 65535;

template <typename T, int COLUMNS, bool LONG>
__global__ void __launch_bounds__(kTileRows * kTileBlocks / COLUMNS)
quantize_columns_kernel(const Params p) {
  const T *x = static_cast<const T *>(p.values);
  const long long rows = p.rows;
  const int cols = p.cols, blocks = p.blocks;
  __shared__ __align__(16) uint8_t tile_bytes[kTileBytes];
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  struct __align__(sizeof(T) * COLUMNS) Few {
    T v[COLUMNS];
  };
  const int r0 = static_cast<int>(threadIdx.x) * COLUMNS, b = threadIdx.y;
  const long long row0 = static_cast<long long>(blockIdx.x) * kTileRows + r0;
  const uint32_t tile_cols = LONG ? (blocks + kTileBlocks - 1) / kTileBlocks : gridDim.y;
  const uint32_t tile_col = LONG ? blockIdx.z * gridDim.y + blockIdx.y : blockIdx.y;
  if (LONG && tile_col >= tile_cols) return;
  const int block = static_cast<int>(tile_col) * kTileBlocks + b;
  const T *from = x + static_cast<long long>(block) * kBlock * rows + row0;
  Few v[kBlock];
#pragma unroll
  for (int j = 0; j < kBlock; ++j) {
    if (row0 < rows && block * kBlock + j < cols) {
      v[j] = *reinterpret_cast<const Few *>(from + j * rows);
    } else {
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c) v[j].v[c] = T(0.f);
    }
  }
  uint32_t largest[COLUMNS];
  if constexpr (COLUMNS == 2) {
    // both columns' maxima at once
    __half2 m = __float2half2_rn(0.f);
#pragma unroll
    for (int j = 0; j < kBlock; ++j) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2 *>(&v[j])));
    largest[0] = magnitude_bits(__low2float(m));
    largest[1] = magnitude_bits(__high2float(m));
  } else {
    largest[0] = 0;
#pragma unroll
    for (int j = 0; j < kBlock; ++j) largest[0] = max(largest[0], magnitude_bits(to_float(v[j].v[0])));
  }
#pragma unroll
  for (int c = 0; c < COLUMNS; ++c) {
    const uint32_t byte = scale_byte(largest[c]);
    const float inv = reciprocal_scale(byte);
    uint32_t packed[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float part[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) part[j] = to_float(v[q * 8 + j].v[c]) * inv;
      packed[q] = byte == 255u ? 0u : encode8(part);
    }
    if (row0 < rows && block < blocks)
      *reinterpret_cast<uint4 *>(p.codes + ((row0 + c) * blocks + block) * 16) =
          make_uint4(packed[0], packed[1], packed[2], packed[3]);
    const int r = r0 + c;
    tile_bytes[(r & 31) * 16 + (r >> 5) * 4 + b] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  const int t = static_cast<int>(threadIdx.y * blockDim.x + threadIdx.x);
  if (t < kTileBytes / 16)
    reinterpret_cast<uint4 *>(p.scales + (static_cast<long long>(blockIdx.x) * tile_cols + tile_col) * kTileBytes)[t] =
        reinterpret_cast<const uint4 *>(tile_bytes)[t];
}

// The way back, with the same division of work.  Where a lane's eight values are more than 16 bytes
// (fp32), or rows start anywhere, they go through shared memory, so that a store of the warp covers
// consecutive bytes (20011 x 776 fp32 values 13.8 us, with two half-filled stores a lane 16.4).  fp16
// 65536 x 4096 104.5 us, 6.5 TB/s, 4096 x 4096 8.5; rows that start anywhere are stored element by
// element, 20011 x 777 fp16 values 13.9 us where the memory needs 6.0, fp32 ones 14.7 (10.8).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps)
dequantize_kernel(const Params p) {
  T *out = static_cast<T *>(const_cast<void *>(p.values));
  const uint8_t *codes = p.codes, *scales = p.scales;
  const long long rows = p.rows, units = p.units;
  const int cols = p.cols, blocks = p.blocks, segments = static_cast<int>(p.segments);
  constexpr bool kDirect = ALIGNED && sizeof(T) == 2;
  __shared__ __align__(16) float sorted[kDirect ? 1 : kWarps][kDirect ? 4 : kSegment];
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long unit = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (unit >= units) return;
  const long long group = unit / segments / kRowStep;
  const int segment = static_cast<int>(unit % segments);
  const int r = static_cast<int>(unit / segments % kRowStep);
  const long long row0 = group * kTileRows + r;
  if (row0 >= rows) return;
  const int col = segment * kSegment + lane * kLaneValues;
  const int tile_cols = (blocks + kTileBlocks - 1) / kTileBlocks;
  const int tile = segment * 2 + (lane >> 4);

  uint32_t packed[4], words[4] = {0, 0, 0, 0};
  if (tile < tile_cols) {
    const uint4 w = *reinterpret_cast<const uint4 *>(scales + (group * tile_cols + tile) * kTileBytes + r * 16);
    words[0] = w.x, words[1] = w.y, words[2] = w.z, words[3] = w.w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + i * kRowStep;
    packed[i] = row < rows && col < blocks * kBlock
                    ? *reinterpret_cast<const uint32_t *>(codes + row * (blocks * 16LL) + col / 2)
                    : 0u;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + i * kRowStep;
    if (row >= rows) break;  // the same for the whole warp
    const float scale = scale_value((words[i] >> (8 * ((lane >> 2) & 3))) & 255u);
    float v[8];
    decode8(packed[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
    T *dst = out + row * cols;
    if constexpr (kDirect) {
      if (col < cols) store8(dst + col, v);
    } else {
      __syncwarp();
      store8(&sorted[warp][lane * kLaneValues], v);
      __syncwarp();
      if constexpr (ALIGNED) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = segment * kSegment + h * (kSegment / 2) + lane * 4;
          if (c < cols)
            *reinterpret_cast<float4 *>(dst + c) =
                *reinterpret_cast<const float4 *>(&sorted[warp][h * (kSegment / 2) + lane * 4]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = segment * kSegment + j * 32 + lane;
          if (c < cols) store1(dst + c, sorted[warp][j * 32 + lane]);
        }
      }
    }
  }
}

bool grid_fits(long long grid, const char *what) {
  if (grid <= INT32_MAX) return true;
  set_error(HOM_ERR_UNSUPPORTED, "%s: the matrix needs more than 2^31 - 1 thread blocks", what);
  return false;
}

bool is_aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

Params params(const void *values, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols) {
  Params p = {};
  p.values = values;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  p.blocks = static_cast<int>(blocks_of(cols));
  p.segments = static_cast<uint32_t>((cols + kSegment - 1) / kSegment);
  p.units = tile_rows_of(rows) * kRowStep * p.segments;
  return p;
}

double traffic(int64_t rows, int64_t cols, size_t element) {
  return static_cast<double>(rows) * (static_cast<double>(cols) * element + 16.5 * blocks_of(cols));
}

}  // namespace

template <typename T>
bool quantize(const T *x, bool transposed, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols,
              cudaStream_t stream) {
  const char *what = "4-bit quantisation launch";
  const int64_t tile_rows = tile_rows_of(rows);
  Params p = params(x, codes, scales, rows, cols);
  if (transposed) {
    const int64_t tile_cols = tile_cols_of(p.blocks);
    if (!grid_fits(tile_rows, what)) return false;
    const int64_t slices = (tile_cols + kMaxGridY - 1) / kMaxGridY;
    LaunchScope scope(kOpConvert, 0.0, traffic(rows, cols, sizeof(T)));
    constexpr int kColumns = sizeof(T) == 2 ? 2 : 1;
    const bool two = kColumns == 2 && slices == 1 && rows % 2 == 0 && (reinterpret_cast<uintptr_t>(x) & 3u) == 0;
    auto kernel = two          ? quantize_columns_kernel<T, kColumns, false>
                  : slices > 1 ? quantize_columns_kernel<T, 1, true>
                               : quantize_columns_kernel<T, 1, false>;
    return check_cuda(launch_pdl(kernel,
                                 dim3(static_cast<unsigned>(tile_rows), static_cast<unsigned>((tile_cols + slices - 1) / slices),
                                      static_cast<unsigned>(slices)),
                                 dim3(kTileRows / (two ? 2 : 1), kTileBlocks), 0, stream, 1, p),
                      what);
  }
  const long long grid = (p.units + kWarps - 1) / kWarps;
  if (!grid_fits(grid, what)) return false;
  auto kernel = cols % kLaneValues == 0 && is_aligned16(x) ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
  LaunchScope scope(kOpConvert, 0.0, traffic(rows, cols, sizeof(T)));
  return check_cuda(launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(32 * kWarps), 0, stream, 1, p), what);
}

template <typename T>
bool dequantize(const uint8_t *codes, const uint8_t *scales, T *out, int64_t rows, int64_t cols,
                cudaStream_t stream) {
  const char *what = "4-bit dequantisation launch";
  const Params p = params(out, const_cast<uint8_t *>(codes), const_cast<uint8_t *>(scales), rows, cols);
  const long long grid = (p.units + kWarps - 1) / kWarps;
  if (!grid_fits(grid, what)) return false;
  auto kernel = cols % kLaneValues == 0 && is_aligned16(out) ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
  LaunchScope scope(kOpConvert, 0.0, traffic(rows, cols, sizeof(T)));
  return check_cuda(launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(32 * kWarps), 0, stream, 1, p), what);
}

template bool quantize<__half>(const __half *, bool, uint8_t *, uint8_t *, int64_t, int64_t, cudaStream_t);
template bool quantize<float>(const float *, bool, uint8_t *, uint8_t *, int64_t, int64_t, cudaStream_t);
template bool dequantize<__half>(const uint8_t *, const uint8_t *, __half *, int64_t, int64_t, cudaStream_t);
template bool dequantize<float>(const uint8_t *, const uint8_t *, float *, int64_t, int64_t, cudaStream_t);

}  // namespace mxf4
}  // namespace hom
