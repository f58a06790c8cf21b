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
constexpr int kBatch = 2;  // tasks whose loads a lane has in flight

struct Params {
  const void *x;
  void *out;
  long long x_b, x_s, x_h, out_b, out_s, out_h;
  const long long *positions;
  long long positions_b;
  const double *frequencies;
  uint32_t tokens, seq;
  int heads, dim, half;
  uint32_t chunks;              // a warp takes one token's heads
  int heads_per_chunk;          // [c * heads_per_chunk, ...)
  float magnitude, sign;
  int fill[8];
};
static_assert(quick_to_launch<Params>, "see launch_pdl");

template <typename T, int VEC>
struct __align__(sizeof(T) * VEC) Vec {
  T v[VEC];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, float &o) { o = x; }
__device__ __forceinline__ void from_float(float x, __half &o) { o = __float2half_rn(x); }

// The sines and cosines of one token, formed by one warp; `frequency` is the lane's first one, asked
// for before the values were (one token of 16 heads 1.77 us, 1.97 when it is asked for here).
__device__ __forceinline__ void form_turns(const Params &p, long long position, double frequency, float2 *turn, int lane) {
  for (int i = lane; i < p.half; i += 32) {
    if (i != lane) frequency = p.frequencies[i];
    const double whole = static_cast<double>(position) * (frequency * 0.15915494309189533577);  // 1 / (2 pi)
    const float part = static_cast<float>(whole - rint(whole));
    float sine, cosine;
    sincospif(2.f * part, &sine, &cosine);
    turn[i] = make_float2(p.magnitude * cosine, p.magnitude * p.sign * sine);
  }
  __syncwarp();
}

// Turns VEC pairs held in two vectors: pair k is (first[k], second[k]), or, interleaved, the k-th two
// neighbours of their sequence.
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void apply_turns(Vec<T, VEC> &first, Vec<T, VEC> &second, const float2 *turn) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float2 t = turn[k];
    T &e0 = !INTERLEAVED || VEC == 1 ? first.v[k] : 2 * k < VEC ? first.v[2 * k % VEC] : second.v[2 * k % VEC];
    T &e1 = !INTERLEAVED || VEC == 1 ? second.v[k] : 2 * k < VEC ? first.v[(2 * k + 1) % VEC] : second.v[(2 * k + 1) % VEC];
    const float x0 = to_float(e0), x1 = to_float(e1);
    from_float(x0 * t.x - x1 * t.y, e0);
    from_float(x1 * t.x + x0 * t.y, e1);
  }
}

// One warp per token, or per token and group of heads where there are too few tokens to fill the
// chip.  The warp forms the token's sines and cosines once, in shared memory, and walks over its
// heads; a task is VEC pairs of a head, two vectors of up to 16 bytes, or two vectors of its other
// dimensions, which are copied.  The first tasks' loads are under way while the sines are formed.
//
// FIXED: the tasks of a head are a power of two up to 32 and all turn pairs, so that a lane works on
// the same pairs of every head and keeps their sines and cosines in registers (64 x 512 tokens of 32
// heads: 65 us without).
//
// Bound by memory where FIXED holds and the vectors have 16 bytes: each element is read and written
// once, 64 x 512 tokens of 32 heads of 64 fp16 values in 41.1 us, 6.5 TB/s, 32 x 512 tokens of 24 heads
// of 128 in 32.9, 6.1 TB/s.  Four CTAs on an SM with two tasks a lane in flight; three CTAs with four
// took 47 us, six with one 45.  Otherwise by instructions, and by the few bytes that a lane has in
// flight: every task finds its place and reads its sines from shared memory, for VEC pairs at a time.
// 32 x 512 tokens of 24 fp16 heads, us, and the time that the memory needs: of 80 32.0 / 19.2, of 96
// 36.6 / 23.1; by vectors of four elements of 72 36.5 / 17.3, of 88 43.2 / 21.2; of two of 68 52.7 /
// 16.4, of 100 74 / 24; of one of 50 48.3 / 12.0.
template <typename T, int VEC, bool INTERLEAVED, bool FIXED>
__global__ void __launch_bounds__(32 * kWarps, 4) rotary_kernel(const Params p) {
  extern __shared__ float2 turns[];
  hom::ptx::pdl_launch_dependents();
  hom::ptx::pdl_wait();
  using V = Vec<T, VEC>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t unit = blockIdx.x * kWarps + warp;
  const uint32_t token = unit / p.chunks;
  if (token >= p.tokens) return;
  const uint32_t b = token / p.seq, s = token - b * p.seq;
  const int head0 = static_cast<int>(unit - token * p.chunks) * p.heads_per_chunk;
  const int heads = min(p.heads_per_chunk, p.heads - head0);
  const T *x = static_cast<const T *>(p.x) + b * p.x_b + s * p.x_s + head0 * p.x_h;
  T *out = static_cast<T *>(p.out) + b * p.out_b + s * p.out_s + head0 * p.out_h;
  float2 *turn = turns + warp * p.half;
  const long long position = p.positions ? p.positions[b * p.positions_b + s] : s;

  const double frequency = lane < p.half ? p.frequencies[lane] : 0.0;

  V first[kBatch], second[kBatch];
  if constexpr (FIXED) {
    const int per_head = p.half / VEC;  // a power of two
    const int pair = (lane & (per_head - 1)) * VEC, at_once = 32 / per_head;
    const int off0 = INTERLEAVED ? 2 * pair : pair, off1 = INTERLEAVED ? 2 * pair + VEC : p.half + pair;
    int head = lane / per_head;
    auto load = [&]() {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (head + i * at_once < heads) {
          const T *src = x + (head + i * at_once) * p.x_h;
          first[i] = *reinterpret_cast<const V *>(src + off0);
          second[i] = *reinterpret_cast<const V *>(src + off1);
        }
      }
    };
    load();
    form_turns(p, position, frequency, turn, lane);
    float2 mine[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) mine[k] = turn[pair + k];
    while (head < heads) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (head + i * at_once < heads) {
          apply_turns<T, VEC, INTERLEAVED>(first[i], second[i], mine);
          T *dst = out + (head + i * at_once) * p.out_h;
          *reinterpret_cast<V *>(dst + off0) = first[i];
          *reinterpret_cast<V *>(dst + off1) = second[i];
        }
      }
      head += kBatch * at_once;
      load();
    }
  } else {
    // tasks of a head: its pairs, then two vectors at a time of what is copied
    const int pairs = p.half / VEC, rest = p.out != p.x ? (p.dim - 2 * p.half) / VEC : 0;
    const int per_head = pairs + (rest + 1) / 2;
    const int tasks = heads * per_head;
    const float inverse = 1.f / static_cast<float>(per_head);
    // head and offsets of a task; the quotient by way of fp32 is off by little for a large task and
    // put right
    struct Place {
      int head, pair, off0, off1;
      bool two;
    };
    auto place = [&](int task) {
      Place at;
      at.head = static_cast<int>(static_cast<float>(task) * inverse);
      int i = task - at.head * per_head;
      while (i < 0) i += per_head, --at.head;
      while (i >= per_head) i -= per_head, ++at.head;
      at.pair = i < pairs ? i * VEC : -1;
      at.off0 = i >= pairs ? 2 * p.half + (i - pairs) * 2 * VEC : INTERLEAVED ? 2 * i * VEC : i * VEC;
      at.off1 = i >= pairs || INTERLEAVED ? at.off0 + VEC : p.half + i * VEC;
      at.two = i < pairs || (i - pairs) * 2 + 1 < rest;
      return at;
    };
    Place at[kBatch];
    auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int task = base + i * 32 + lane;
        if (task < tasks) {
          at[i] = place(task);
          const T *src = x + at[i].head * p.x_h;
          first[i] = *reinterpret_cast<const V *>(src + at[i].off0);
          if (at[i].two) second[i] = *reinterpret_cast<const V *>(src + at[i].off1);
        }
      }
    };
    load(0);
    form_turns(p, position, frequency, turn, lane);
    for (int base = 0; base < tasks; base += 32 * kBatch) {
      if (base) load(base);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int task = base + i * 32 + lane;
        if (task < tasks) {
          if (at[i].pair >= 0) apply_turns<T, VEC, INTERLEAVED>(first[i], second[i], turn + at[i].pair);
          T *dst = out + at[i].head * p.out_h;
          *reinterpret_cast<V *>(dst + at[i].off0) = first[i];
          if (at[i].two) *reinterpret_cast<V *>(dst + at[i].off1) = second[i];
        }
      }
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
  Params p = {};
  p.x = pb.x.ptr;
  p.out = pb.out.ptr;
  p.x_b = pb.x.stride_b, p.x_s = pb.x.stride_s, p.x_h = pb.x.stride_h;
  p.out_b = pb.out.stride_b, p.out_s = pb.out.stride_s, p.out_h = pb.out.stride_h;
  p.positions = reinterpret_cast<const long long *>(pb.positions);
  p.positions_b = pb.positions_stride_b;
  p.frequencies = pb.frequencies;
  p.tokens = static_cast<uint32_t>(pb.batch * pb.seq);
  p.seq = static_cast<uint32_t>(pb.seq);
  p.heads = static_cast<int>(pb.heads);
  p.dim = static_cast<int>(pb.dim);
  p.half = static_cast<int>(pb.half);
  p.magnitude = pb.magnitude;
  p.sign = pb.backward ? -1.f : 1.f;
  // Few tokens: their heads are spread over more warps, each of which forms the sines anew.
  const long long want = 16LL * sm_count();
  const long long tokens = p.tokens;
  long long chunks = tokens >= want ? 1 : (want + tokens - 1) / tokens;
  if (chunks > p.heads) chunks = p.heads;
  p.heads_per_chunk = static_cast<int>((p.heads + chunks - 1) / chunks);
  p.chunks = static_cast<uint32_t>((p.heads + p.heads_per_chunk - 1) / p.heads_per_chunk);
  const long long grid = (static_cast<long long>(p.tokens) * p.chunks + kWarps - 1) / kWarps;
  const int per_head = p.half / VEC;
  const bool fixed = per_head <= 32 && (per_head & (per_head - 1)) == 0 && (p.dim == 2 * p.half || p.out == p.x);
  auto kernel = pb.interleaved ? (fixed ? rotary_kernel<T, VEC, true, true> : rotary_kernel<T, VEC, true, false>)
                               : (fixed ? rotary_kernel<T, VEC, false, true> : rotary_kernel<T, VEC, false, false>);
  const double elements = static_cast<double>(pb.batch) * pb.seq * pb.heads * pb.dim;
  LaunchScope scope(kOpRotary, 0.0, 2.0 * sizeof(T) * elements);
  return check_cuda(launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(32 * kWarps),
                               kWarps * p.half * sizeof(float2), stream, 1, p),
                    "rotary positions launch");
}

}  // namespace

template <typename T>
bool run(const Problem &pb, cudaStream_t stream) {
  // The widest vectors, up to 16 bytes, that heads, their parts and all strides are whole ones of.
  auto fits = [&](int64_t vec) {
    auto view = [&](const View &v) {
      return reinterpret_cast<uintptr_t>(v.ptr) % (vec * sizeof(T)) == 0 && (pb.batch == 1 || v.stride_b % vec == 0) &&
             (pb.seq == 1 || v.stride_s % vec == 0) && (pb.heads == 1 || v.stride_h % vec == 0);
    };
    return pb.half % vec == 0 && (pb.dim - 2 * pb.half) % vec == 0 && view(pb.x) && view(pb.out);
  };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return launch<T, 8>(pb, stream);
  if (fits(4)) return launch<T, 4>(pb, stream);
  return fits(2) ? launch<T, 2>(pb, stream) : launch<T, 1>(pb, stream);
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
