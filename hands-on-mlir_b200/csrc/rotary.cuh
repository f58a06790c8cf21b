// Host interface of the rotary-position kernels (rotary.cu).
#pragma once

#include "hom_common.cuh"

namespace hom {
namespace rotary {

// [batch, seq, heads, dim] views whose last dimension is contiguous; strides in elements.
struct View {
  void *ptr = nullptr;
  int64_t stride_b = 0, stride_s = 0, stride_h = 0;
};

struct Problem {
  int64_t batch = 0, seq = 0, heads = 0, dim = 0;
  int64_t half = 0;  // pairs: the first 2 * half dimensions of a head are turned
  View x, out;       // out may be x
  const int64_t *positions = nullptr;  // null: 0 .. seq - 1
  int64_t positions_stride_b = 0;      // 0: the sequences share one row
  const double *frequencies = nullptr;
  bool interleaved = false;  // pairs (2i, 2i + 1) instead of (i, half + i)
  bool backward = false;
  float magnitude = 1.f;
};

constexpr int64_t kMaxHalf = 512;

template <typename T>
bool run(const Problem &pb, cudaStream_t stream);

// scaling: 0 none, 1 linear, 2 changed base, 3 by parts (see homRotaryFrequencies)
bool frequencies(double *out, int64_t half, double base, int scaling, double factor, double original_length,
                 double beta_fast, double beta_slow, cudaStream_t stream);

}  // namespace rotary
}  // namespace hom
