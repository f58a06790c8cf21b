// Rotary positions: the first r = 2 * half dimensions of every head are half pairs, and pair i of a
// token at position p is turned by the angle p * f_i and stretched by a magnitude m:
//   y0 = m (x0 cos - x1 sin),   y1 = m (x1 cos + x0 sin)
// (backward: the transpose, that is the sine with the other sign).  The other dimensions pass.
//
// The angle is formed in fp64: at position 2^20 an fp32 product is off by up to 0.06 radians.
// Taken as a number of turns, the whole turns fall away exactly and what is left, in [-1/2, 1/2],
// fits an fp32 sine and cosine to 2e-7 radians.  The rotation itself is fp32, rounded once.
#include "ptx_sm100.cuh"
#include "rotary.cuh"

namespace hom {
namespace rotary {

namespace {

constexpr int kWarps = 8;
constexpr int kBatch = 4;  // tasks whose loads a lane has in flight

struct Params {
  const void *x;
  void *out;
  long long x_b, x_s, x_h, out_b, out_s, out_h;
  const long long *positions;
  long long positions_b;
  const double *frequencies;
  long long tokens;
  int seq, heads, dim, half;
  int chunks, heads_per_chunk;  // a warp takes one token's heads [c * heads_per_chunk, ...)
  float magnitude, sign;
};

template <typename T, int VEC>
struct Vec;
template <typename T>
struct Vec<T, 1> {
  T v[1];
};
template <>
struct __align__(16) Vec<__half, 8> {
  __half v[8];
};
template <>
struct __align__(16) Vec<float, 4> {
  float v[4];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, float &o) { o = x; }
__device__ __forceinline__ void from_float(float x, __half &o) { o = __float2half_rn(x); }

// One warp per token (or per token and group of heads, where there are too few tokens to fill the
// chip).  The warp forms the token's sines and cosines once, in shared memory, and then walks over
// its heads; a task is VEC pairs of a head, two 16-byte vectors.  The first tasks' loads are under
// way while the sines are formed.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kWarps) rotary_kernel(const Params p) {
  extern __shared__ float2 turns[];
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  using V = Vec<T, VEC>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long unit = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (unit >= p.tokens * p.chunks) return;
  const long long token = unit / p.chunks;
  const long long b = token / p.seq, s = token % p.seq;
  const int head0 = static_cast<int>(unit % p.chunks) * p.heads_per_chunk;
  const int heads = min(p.heads_per_chunk, p.heads - head0);
  const T *x = static_cast<const T *>(p.x) + b * p.x_b + s * p.x_s + head0 * p.x_h;
  T *out = static_cast<T *>(p.out) + b * p.out_b + s * p.out_s + head0 * p.out_h;
  float2 *turn = turns + warp * p.half;

  const int per_head = p.half / VEC;
  const int tasks = heads * per_head;
  V first[kBatch], second[kBatch];
  auto place = [&](int task, int *head, int *pair) {
    *head = task / per_head;
    *pair = (task - *head * per_head) * VEC;
  };
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int task = base + i * 32 + lane;
      if (task < tasks) {
        int head, pair;
        place(task, &head, &pair);
        const T *src = x + head * p.x_h;
        first[i] = *reinterpret_cast<const V *>(src + (INTERLEAVED ? 2 * pair : pair));
        second[i] = *reinterpret_cast<const V *>(src + (INTERLEAVED ? 2 * pair + VEC : p.half + pair));
      }
    }
  };
  load(0);

  const long long position = p.positions ? p.positions[b * p.positions_b + s] : s;
  for (int i = lane; i < p.half; i += 32) {
    const double whole = static_cast<double>(position) * (p.frequencies[i] * 0.15915494309189533577);  // 1 / (2 pi)
    const float part = static_cast<float>(whole - rint(whole));
    float sine, cosine;
    sincospif(2.f * part, &sine, &cosine);
    turn[i] = make_float2(p.magnitude * cosine, p.magnitude * p.sign * sine);
  }
  __syncwarp();

  for (int base = 0; base < tasks; base += 32 * kBatch) {
    if (base) load(base);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int task = base + i * 32 + lane;
      if (task < tasks) {
        int head, pair;
        place(task, &head, &pair);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 t = turn[pair + k];
          // pair k of the two vectors: (first[k], second[k]), or two neighbours of their sequence
          T &e0 = !INTERLEAVED || VEC == 1 ? first[i].v[k] : 2 * k < VEC ? first[i].v[2 * k % VEC] : second[i].v[2 * k % VEC];
          T &e1 = !INTERLEAVED || VEC == 1 ? second[i].v[k]
                  : 2 * k < VEC            ? first[i].v[(2 * k + 1) % VEC]
                                           : second[i].v[(2 * k + 1) % VEC];
          const float x0 = to_float(e0), x1 = to_float(e1);
          from_float(x0 * t.x - x1 * t.y, e0);
          from_float(x1 * t.x + x0 * t.y, e1);
        }
        T *dst = out + head * p.out_h;
        *reinterpret_cast<V *>(dst + (INTERLEAVED ? 2 * pair : pair)) = first[i];
        *reinterpret_cast<V *>(dst + (INTERLEAVED ? 2 * pair + VEC : p.half + pair)) = second[i];
      }
    }
  }
  // the dimensions that are not turned
  if (p.out != p.x) {
    const int rest = (p.dim - 2 * p.half) / VEC;
    for (int task = lane; task < heads * rest; task += 32) {
      const int head = task / rest, d = 2 * p.half + (task - head * rest) * VEC;
      *reinterpret_cast<V *>(out + head * p.out_h + d) = *reinterpret_cast<const V *>(x + head * p.x_h + d);
    }
  }
}

__global__ void frequencies_kernel(double *out, int half, double base, int scaling, double factor,
                                   double original_length, double beta_fast, double beta_slow) {
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  const double r = 2.0 * half;
  if (scaling == 2 && half > 1) base *= pow(factor, r / (r - 2.0));
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    double f = pow(base, -2.0 * i / r);
    if (scaling == 1) f /= factor;
    if (scaling == 3) {
      const double turns = original_length * f * 0.15915494309189533577;
      const double keep = fmin(fmax((turns - beta_slow) / (beta_fast - beta_slow), 0.0), 1.0);
      f = f * (keep + (1.0 - keep) / factor);
    }
    out[i] = f;
  }
}

template <typename T, int VEC>
bool launch(const Problem &pb, cudaStream_t stream) {
  Params p;
  p.x = pb.x.ptr;
  p.out = pb.out.ptr;
  p.x_b = pb.x.stride_b, p.x_s = pb.x.stride_s, p.x_h = pb.x.stride_h;
  p.out_b = pb.out.stride_b, p.out_s = pb.out.stride_s, p.out_h = pb.out.stride_h;
  p.positions = reinterpret_cast<const long long *>(pb.positions);
  p.positions_b = pb.positions_stride_b;
  p.frequencies = pb.frequencies;
  p.tokens = pb.batch * pb.seq;
  p.seq = static_cast<int>(pb.seq);
  p.heads = static_cast<int>(pb.heads);
  p.dim = static_cast<int>(pb.dim);
  p.half = static_cast<int>(pb.half);
  p.magnitude = pb.magnitude;
  p.sign = pb.backward ? -1.f : 1.f;
  // Few tokens: their heads are spread over more warps, each of which forms the sines anew.
  const long long want = 16LL * sm_count();
  long long chunks = p.tokens >= want ? 1 : (want + p.tokens - 1) / p.tokens;
  if (chunks > p.heads) chunks = p.heads;
  p.heads_per_chunk = static_cast<int>((p.heads + chunks - 1) / chunks);
  p.chunks = (p.heads + p.heads_per_chunk - 1) / p.heads_per_chunk;
  const long long grid = (p.tokens * p.chunks + kWarps - 1) / kWarps;
  if (grid > INT32_MAX) {
    set_error(HOM_ERR_UNSUPPORTED, "rotary positions: more than 2^31 - 1 thread blocks");
    return false;
  }
  auto kernel = pb.interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>;
  const double elements = static_cast<double>(p.tokens) * p.heads * p.dim;
  LaunchScope scope(kOpRotary, 0.0, 2.0 * sizeof(T) * elements);
  return check_cuda(launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(32 * kWarps),
                               kWarps * p.half * sizeof(float2), stream, 1, p),
                    "rotary positions launch");
}

}  // namespace

template <typename T>
bool run(const Problem &pb, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  auto fits = [&](const View &v) {
    return (reinterpret_cast<uintptr_t>(v.ptr) & 15u) == 0 && (pb.batch == 1 || v.stride_b % VEC == 0) &&
           (pb.seq == 1 || v.stride_s % VEC == 0) && (pb.heads == 1 || v.stride_h % VEC == 0);
  };
  const bool vectors = pb.half % VEC == 0 && (pb.dim - 2 * pb.half) % VEC == 0 && fits(pb.x) && fits(pb.out);
  return vectors ? launch<T, VEC>(pb, stream) : launch<T, 1>(pb, stream);
}

template bool run<__half>(const Problem &, cudaStream_t);
template bool run<float>(const Problem &, cudaStream_t);

bool frequencies(double *out, int64_t half, double base, int scaling, double factor, double original_length,
                 double beta_fast, double beta_slow, cudaStream_t stream) {
  LaunchScope scope(kOpRotary, 0.0, 8.0 * half);
  return check_cuda(launch_pdl(frequencies_kernel, dim3(1), dim3(128), 0, stream, 1, out, static_cast<int>(half), base,
                               scaling, factor, original_length, beta_fast, beta_slow),
                    "rotary frequencies launch");
}

}  // namespace rotary
}  // namespace hom
