// extern "C" entry points of the 4-bit floating-point operators and of the rotary positions:
// argument validation and dispatch.  A rejected call records an error and launches nothing.
#include <cmath>

#include "hom_common.cuh"
#include "mxf4_sm100.cuh"
#include "rotary.cuh"

namespace {

using hom::MemRefView;
using hom::set_error;
using hom::view_memref;
namespace mxf4 = hom::mxf4;

// Largest extent of a dimension: index arithmetic inside a matrix row and tile is 32-bit.
constexpr int64_t kMaxExtent = int64_t{1} << 30;

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A descriptor over no elements may carry a null pointer.
bool usable(const MemRefView &v) { return v.valid || (v.rank > 0 && v.numel() == 0); }

// [rank 2 or 3] flattened to rows x cols (a rank-3 operand's leading dimensions together).
bool as_matrix(const char *name, const char *what, const MemRefView &v, int64_t *rows, int64_t *cols) {
  if (!usable(v) || (v.rank != 2 && v.rank != 3)) {
    set_error(HOM_ERR_INVALID, "%s: %s must be a memref of rank 2 or 3", name, what);
    return false;
  }
  for (int64_t i = 0; i < v.rank; ++i) {
    if (v.sizes[i] > kMaxExtent) {
      set_error(HOM_ERR_UNSUPPORTED, "%s: a dimension of %s exceeds 2^30", name, what);
      return false;
    }
  }
  *cols = v.sizes[v.rank - 1];
  *rows = v.rank == 3 ? v.sizes[0] * v.sizes[1] : v.sizes[0];
  if (*rows > kMaxExtent) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: %s has more than 2^30 rows", name, what);
    return false;
  }
  if (*rows != 0 && *cols != 0 && !v.contiguous()) {
    set_error(HOM_ERR_INVALID, "%s: %s must be row-major contiguous", name, what);
    return false;
  }
  return true;
}

// Codes [rows, 16 * blocks] with their scales [row tiles, block tiles, 512].
bool coded_operand(const char *name, const char *what, const MemRefView &q, const MemRefView &s, int64_t *rows,
                   int64_t *blocks) {
  int64_t pitch = 0;
  if (!as_matrix(name, what, q, rows, &pitch)) return false;
  if (pitch % 16 != 0) {
    set_error(HOM_ERR_INVALID, "%s: rows of %s must be whole blocks of 16 bytes, got %lld", name, what,
              static_cast<long long>(pitch));
    return false;
  }
  *blocks = pitch / 16;
  const int64_t tile_rows = mxf4::tile_rows_of(*rows), tile_cols = mxf4::tile_cols_of(*blocks);
  if (!usable(s) || s.rank != 3 || s.sizes[0] != tile_rows || s.sizes[1] != tile_cols ||
      s.sizes[2] != mxf4::kTileBytes || (s.numel() != 0 && !s.contiguous())) {
    set_error(HOM_ERR_INVALID, "%s: the scales of %s must be contiguous [%lld, %lld, %d]", name, what,
              static_cast<long long>(tile_rows), static_cast<long long>(tile_cols), mxf4::kTileBytes);
    return false;
  }
  if (!aligned(q.ptr, 16) || !aligned(s.ptr, 16)) {
    set_error(HOM_ERR_INVALID, "%s: %s and its scales must be 16-byte aligned", name, what);
    return false;
  }
  return true;
}

bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(b_bytes) && y < x + static_cast<uintptr_t>(a_bytes);
}

bool reject_overlap(const char *name) {
  set_error(HOM_ERR_INVALID, "%s: an output overlaps another operand", name);
  return false;
}

template <typename T>
void quantize_entry(const char *name, int64_t rankX, void *dstX, bool transposed, int64_t rankQ, void *dstQ,
                    int64_t rankS, void *dstS) {
  const MemRefView X = view_memref(rankX, dstX, sizeof(T)), Q = view_memref(rankQ, dstQ, 1);
  const MemRefView S = view_memref(rankS, dstS, 1);
  int64_t rows = 0, cols = 0, q_rows = 0, blocks = 0;
  if (!as_matrix(name, "X", X, &rows, &cols)) return;
  if (transposed) {
    if (X.rank == 3 && X.sizes[0] != 1) {
      set_error(HOM_ERR_UNSUPPORTED, "%s: a transposed X must be [K, N] or [1, K, N]", name);
      return;
    }
    const int64_t k = rows;
    rows = cols;
    cols = k;
  }
  if (!coded_operand(name, "Q", Q, S, &q_rows, &blocks)) return;
  if (q_rows != rows || blocks != mxf4::blocks_of(cols)) {
    set_error(HOM_ERR_INVALID, "%s: %lld x %lld values need codes [%lld, %lld]", name, static_cast<long long>(rows),
              static_cast<long long>(cols), static_cast<long long>(rows),
              static_cast<long long>(16 * mxf4::blocks_of(cols)));
    return;
  }
  if (rows == 0 || cols == 0) return;
  if (!aligned(X.ptr, sizeof(T))) {
    set_error(HOM_ERR_INVALID, "%s: X is not aligned to its elements", name);
    return;
  }
  const int64_t x_bytes = X.numel() * static_cast<int64_t>(sizeof(T));
  if (overlap(X.ptr, x_bytes, Q.ptr, Q.numel()) || overlap(X.ptr, x_bytes, S.ptr, S.numel()) ||
      overlap(Q.ptr, Q.numel(), S.ptr, S.numel())) {
    reject_overlap(name);
    return;
  }
  // A product that requested these early would read them while they are written.
  hom::withdraw_constant_ranges({{Q.ptr, static_cast<size_t>(Q.numel())}, {S.ptr, static_cast<size_t>(S.numel())}});
  mxf4::quantize(reinterpret_cast<const T *>(X.ptr), transposed, reinterpret_cast<uint8_t *>(Q.ptr),
                 reinterpret_cast<uint8_t *>(S.ptr), rows, cols, hom::current_stream());
}

template <typename T>
void dequantize_entry(const char *name, int64_t rankQ, void *dstQ, int64_t rankS, void *dstS, int64_t rankOut,
                      void *dstOut) {
  const MemRefView Q = view_memref(rankQ, dstQ, 1), S = view_memref(rankS, dstS, 1);
  const MemRefView O = view_memref(rankOut, dstOut, sizeof(T));
  int64_t rows = 0, cols = 0, q_rows = 0, blocks = 0;
  if (!coded_operand(name, "Q", Q, S, &q_rows, &blocks) || !as_matrix(name, "Out", O, &rows, &cols)) return;
  if (q_rows != rows || blocks != mxf4::blocks_of(cols)) {
    set_error(HOM_ERR_INVALID, "%s: codes [%lld, %lld] do not hold %lld x %lld values", name,
              static_cast<long long>(q_rows), static_cast<long long>(16 * blocks), static_cast<long long>(rows),
              static_cast<long long>(cols));
    return;
  }
  if (rows == 0 || cols == 0) return;
  if (!aligned(O.ptr, sizeof(T))) {
    set_error(HOM_ERR_INVALID, "%s: Out is not aligned to its elements", name);
    return;
  }
  const int64_t o_bytes = O.numel() * static_cast<int64_t>(sizeof(T));
  if (overlap(O.ptr, o_bytes, Q.ptr, Q.numel()) || overlap(O.ptr, o_bytes, S.ptr, S.numel())) {
    reject_overlap(name);
    return;
  }
  mxf4::dequantize(reinterpret_cast<const uint8_t *>(Q.ptr), reinterpret_cast<const uint8_t *>(S.ptr),
                   reinterpret_cast<T *>(O.ptr), rows, cols, hom::current_stream());
}

// Row-major order is not asked for, but two places of the view must never be one element.
bool distinct_elements(const MemRefView &v) {
  int order[HOM_MAX_RANK];
  int n = 0;
  for (int i = 0; i < v.rank; ++i)
    if (v.sizes[i] > 1) order[n++] = i;
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && v.strides[order[j]] < v.strides[order[j - 1]]; --j) {
      const int t = order[j];
      order[j] = order[j - 1];
      order[j - 1] = t;
    }
  int64_t span = 1;  // elements from the first to the last of the dimensions so far
  for (int i = 0; i < n; ++i) {
    if (v.strides[order[i]] < span) return false;
    span += v.strides[order[i]] * (v.sizes[order[i]] - 1);
  }
  return true;
}

int64_t span_elements(const MemRefView &v) {
  int64_t span = 1;
  for (int64_t i = 0; i < v.rank; ++i) span += (v.sizes[i] - 1) * v.strides[i];
  return span;
}

template <typename T>
void rotary_entry(const char *name, int64_t rankX, void *dstX, int64_t rankPos, void *dstPos, int64_t rankFreq,
                  void *dstFreq, int64_t rankOut, void *dstOut, bool interleaved, bool backward, float magnitude) {
  const MemRefView X = view_memref(rankX, dstX, sizeof(T)), O = view_memref(rankOut, dstOut, sizeof(T));
  const MemRefView P = view_memref(rankPos, dstPos, 8), F = view_memref(rankFreq, dstFreq, 8);
  if (!usable(X) || !usable(O) || X.rank != 4 || O.rank != 4) {
    set_error(HOM_ERR_INVALID, "%s: X and Out must be memrefs [bs, seq, heads, d]", name);
    return;
  }
  if (!F.valid || F.rank != 1 || F.sizes[0] < 1 || !F.contiguous() || !aligned(F.ptr, 8)) {
    set_error(HOM_ERR_INVALID, "%s: Frequencies must be a contiguous fp64 memref of rank 1", name);
    return;
  }
  int64_t total = 1;
  for (int i = 0; i < 4; ++i) {
    if (X.sizes[i] != O.sizes[i]) {
      set_error(HOM_ERR_INVALID, "%s: X and Out have different shapes", name);
      return;
    }
    if (X.sizes[i] > kMaxExtent) {
      set_error(HOM_ERR_UNSUPPORTED, "%s: a dimension exceeds 2^30", name);
      return;
    }
    for (const MemRefView *v : {&X, &O}) {
      if (v->sizes[i] > 1 && (v->strides[i] < 0 || v->strides[i] > INT64_MAX / 16 / v->sizes[i])) {
        set_error(HOM_ERR_UNSUPPORTED, "%s: negative or too large strides", name);
        return;
      }
    }
    if (X.sizes[i] != 0 && total > INT64_MAX / X.sizes[i]) {
      set_error(HOM_ERR_UNSUPPORTED, "%s: too many elements", name);
      return;
    }
    total *= X.sizes[i];
  }
  const int64_t bs = X.sizes[0], seq = X.sizes[1], heads = X.sizes[2], dim = X.sizes[3], half = F.sizes[0];
  if (half > hom::rotary::kMaxHalf) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: more than %lld frequencies", name,
              static_cast<long long>(hom::rotary::kMaxHalf));
    return;
  }
  if (dim > 0 && 2 * half > dim) {
    set_error(HOM_ERR_INVALID, "%s: %lld frequencies turn %lld dimensions, a head has %lld", name,
              static_cast<long long>(half), static_cast<long long>(2 * half), static_cast<long long>(dim));
    return;
  }
  const bool positions = dstPos != nullptr;
  if (positions && (!usable(P) || P.rank != 2 || (P.sizes[0] != bs && P.sizes[0] != 1) || P.sizes[1] != seq ||
                    (P.numel() != 0 && !P.contiguous()) || !aligned(P.ptr, 8))) {
    set_error(HOM_ERR_INVALID, "%s: Positions must be contiguous int64 [bs, seq] or [1, seq], or absent", name);
    return;
  }
  if (!std::isfinite(magnitude)) {
    set_error(HOM_ERR_INVALID, "%s: the magnitude is not a number", name);
    return;
  }
  if (total == 0) return;
  if (dim > 1 && (X.strides[3] != 1 || O.strides[3] != 1)) {
    set_error(HOM_ERR_INVALID, "%s: the last dimension must be contiguous", name);
    return;
  }
  if (heads * dim > INT32_MAX || bs * seq > INT32_MAX) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens, or elements in a token", name);
    return;
  }
  if (!aligned(X.ptr, sizeof(T)) || !aligned(O.ptr, sizeof(T))) {
    set_error(HOM_ERR_INVALID, "%s: X or Out is not aligned to its elements", name);
    return;
  }
  if (!distinct_elements(O)) {
    set_error(HOM_ERR_INVALID, "%s: elements of Out share memory", name);
    return;
  }
  bool in_place = X.ptr == O.ptr;
  for (int i = 0; i < 4; ++i) in_place = in_place && (X.sizes[i] == 1 || X.strides[i] == O.strides[i]);
  const int64_t o_bytes = span_elements(O) * static_cast<int64_t>(sizeof(T));
  if ((!in_place && overlap(X.ptr, span_elements(X) * static_cast<int64_t>(sizeof(T)), O.ptr, o_bytes)) ||
      overlap(F.ptr, half * 8, O.ptr, o_bytes) || (positions && overlap(P.ptr, P.numel() * 8, O.ptr, o_bytes))) {
    reject_overlap(name);
    return;
  }
  hom::rotary::Problem pb;
  pb.batch = bs;
  pb.seq = seq;
  pb.heads = heads;
  pb.dim = dim;
  pb.half = half;
  pb.x = {X.ptr, X.strides[0], X.strides[1], X.strides[2]};
  pb.out = {O.ptr, O.strides[0], O.strides[1], O.strides[2]};
  pb.positions = positions ? reinterpret_cast<const int64_t *>(P.ptr) : nullptr;
  pb.positions_stride_b = positions && P.sizes[0] != 1 ? seq : 0;
  pb.frequencies = reinterpret_cast<const double *>(F.ptr);
  pb.interleaved = interleaved;
  pb.backward = backward;
  pb.magnitude = magnitude;
  hom::rotary::run<T>(pb, hom::current_stream());
}

}  // namespace

extern "C" {

void homQuantizeMxF4F16(int64_t rankX, void *dstX, bool transposed, int64_t rankQ, void *dstQ, int64_t rankS,
                        void *dstS) {
  quantize_entry<__half>("homQuantizeMxF4F16", rankX, dstX, transposed, rankQ, dstQ, rankS, dstS);
}
void homQuantizeMxF4F32(int64_t rankX, void *dstX, bool transposed, int64_t rankQ, void *dstQ, int64_t rankS,
                        void *dstS) {
  quantize_entry<float>("homQuantizeMxF4F32", rankX, dstX, transposed, rankQ, dstQ, rankS, dstS);
}
void homDequantizeMxF4F16(int64_t rankQ, void *dstQ, int64_t rankS, void *dstS, int64_t rankOut, void *dstOut) {
  dequantize_entry<__half>("homDequantizeMxF4F16", rankQ, dstQ, rankS, dstS, rankOut, dstOut);
}
void homDequantizeMxF4F32(int64_t rankQ, void *dstQ, int64_t rankS, void *dstS, int64_t rankOut, void *dstOut) {
  dequantize_entry<float>("homDequantizeMxF4F32", rankQ, dstQ, rankS, dstS, rankOut, dstOut);
}

void homGemmMxF4F16(int64_t rankA, void *dstA, int64_t rankSA, void *dstSA, int64_t rankB, void *dstB, int64_t rankSB,
                    void *dstSB, int64_t rankC, void *dstC, int64_t rankD, void *dstD, int64_t activation,
                    float alpha, float beta) {
  const char *name = "homGemmMxF4F16";
  const MemRefView A = view_memref(rankA, dstA, 1), SA = view_memref(rankSA, dstSA, 1);
  const MemRefView B = view_memref(rankB, dstB, 1), SB = view_memref(rankSB, dstSB, 1);
  const MemRefView C = view_memref(rankC, dstC, 2), D = view_memref(rankD, dstD, 2);
  mxf4::Problem pb;
  int64_t d_rows = 0, d_cols = 0, b_blocks = 0;
  if (!coded_operand(name, "A", A, SA, &pb.M, &pb.blocks) || !coded_operand(name, "B", B, SB, &pb.N, &b_blocks) ||
      !as_matrix(name, "D", D, &d_rows, &d_cols))
    return;
  if (B.rank == 3 && B.sizes[0] != 1) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: B must have batch 1 (weights are shared by the batch)", name);
    return;
  }
  if (b_blocks != pb.blocks) {
    set_error(HOM_ERR_INVALID, "%s: inner dimensions differ (A has %lld blocks of 32, B has %lld)", name,
              static_cast<long long>(pb.blocks), static_cast<long long>(b_blocks));
    return;
  }
  if (d_rows != pb.M || d_cols != pb.N || D.rank != A.rank || (A.rank == 3 && A.sizes[0] != D.sizes[0])) {
    set_error(HOM_ERR_INVALID, "%s: D must be [%lld x %lld] with the leading dimensions of A", name,
              static_cast<long long>(pb.M), static_cast<long long>(pb.N));
    return;
  }
  if (activation != 0 && activation != 1) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: activation %lld (0 = none, 1 = erf GELU)", name,
              static_cast<long long>(activation));
    return;
  }
  if (pb.M == 0 || pb.N == 0) return;
  if (pb.blocks == 0) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: K == 0", name);
    return;
  }
  const size_t need = pb.N % 8 == 0 ? 16 : 2;  // whole 16-byte rows travel in 16-byte pieces
  const int64_t d_bytes = 2 * pb.M * pb.N;
  if (beta != 0.f) {
    if (!C.valid || !C.contiguous() || C.rank < 1 || C.sizes[C.rank - 1] != pb.N) {
      set_error(HOM_ERR_INVALID, "%s: beta != 0 needs a contiguous C [%lld x %lld] or a length-%lld row", name,
                static_cast<long long>(pb.M), static_cast<long long>(pb.N), static_cast<long long>(pb.N));
      return;
    }
    int64_t c_rows = 1;
    for (int64_t i = 0; i + 1 < C.rank; ++i) {
      if (C.sizes[i] > kMaxExtent || c_rows > kMaxExtent) {
        set_error(HOM_ERR_UNSUPPORTED, "%s: a dimension of C exceeds 2^30", name);
        return;
      }
      c_rows *= C.sizes[i];
    }
    if (c_rows != pb.M && c_rows != 1) {
      set_error(HOM_ERR_INVALID, "%s: C must be [%lld x %lld] or a length-%lld row", name,
                static_cast<long long>(pb.M), static_cast<long long>(pb.N), static_cast<long long>(pb.N));
      return;
    }
    pb.c_mode = c_rows == pb.M ? 1 : 2;
    pb.C = reinterpret_cast<const __half *>(C.ptr);
    if (!aligned(C.ptr, need)) {
      set_error(HOM_ERR_INVALID, "%s: C is not %d-byte aligned", name, static_cast<int>(need));
      return;
    }
    const int64_t c_bytes = 2 * c_rows * pb.N;
    if (overlap(C.ptr, c_bytes, D.ptr, d_bytes) && !(pb.c_mode == 1 && C.ptr == D.ptr)) {
      reject_overlap(name);
      return;
    }
  }
  if (!aligned(D.ptr, need)) {
    set_error(HOM_ERR_INVALID, "%s: D is not %d-byte aligned", name, static_cast<int>(need));
    return;
  }
  for (const MemRefView *v : {&A, &SA, &B, &SB}) {
    if (overlap(v->ptr, v->numel(), D.ptr, d_bytes)) {
      reject_overlap(name);
      return;
    }
  }
  pb.A = reinterpret_cast<const uint8_t *>(A.ptr);
  pb.scales_a = reinterpret_cast<const uint8_t *>(SA.ptr);
  pb.B = reinterpret_cast<const uint8_t *>(B.ptr);
  pb.scales_b = reinterpret_cast<const uint8_t *>(SB.ptr);
  pb.b_const = hom::is_constant_range(B.ptr, static_cast<size_t>(B.numel())) &&
               hom::is_constant_range(SB.ptr, static_cast<size_t>(SB.numel()));
  pb.D = reinterpret_cast<__half *>(D.ptr);
  pb.alpha = alpha;
  pb.beta = beta;
  pb.act = static_cast<int>(activation);
  mxf4::run_product(pb, hom::current_stream());
}

void homRotaryF16(int64_t rankX, void *dstX, int64_t rankPos, void *dstPos, int64_t rankFreq, void *dstFreq,
                  int64_t rankOut, void *dstOut, bool interleaved, bool backward, float magnitude) {
  rotary_entry<__half>("homRotaryF16", rankX, dstX, rankPos, dstPos, rankFreq, dstFreq, rankOut, dstOut, interleaved,
                       backward, magnitude);
}
void homRotaryF32(int64_t rankX, void *dstX, int64_t rankPos, void *dstPos, int64_t rankFreq, void *dstFreq,
                  int64_t rankOut, void *dstOut, bool interleaved, bool backward, float magnitude) {
  rotary_entry<float>("homRotaryF32", rankX, dstX, rankPos, dstPos, rankFreq, dstFreq, rankOut, dstOut, interleaved,
                      backward, magnitude);
}

void homRotaryFrequencies(int64_t rankFreq, void *dstFreq, double base, int32_t scaling, double factor,
                          double originalLength, double betaFast, double betaSlow) {
  const char *name = "homRotaryFrequencies";
  const MemRefView F = view_memref(rankFreq, dstFreq, 8);
  if (!F.valid || F.rank != 1 || F.sizes[0] < 1 || !F.contiguous() || !aligned(F.ptr, 8)) {
    set_error(HOM_ERR_INVALID, "%s: Frequencies must be a contiguous fp64 memref of rank 1", name);
    return;
  }
  if (F.sizes[0] > hom::rotary::kMaxHalf) {
    set_error(HOM_ERR_UNSUPPORTED, "%s: more than %lld frequencies", name,
              static_cast<long long>(hom::rotary::kMaxHalf));
    return;
  }
  if (!(base > 0.0) || !std::isfinite(base) || scaling < 0 || scaling > 3 ||
      (scaling != 0 && (!(factor > 0.0) || !std::isfinite(factor))) ||
      (scaling == 3 && (!(originalLength > 0.0) || !std::isfinite(originalLength) || !std::isfinite(betaFast) ||
                        !std::isfinite(betaSlow) || !(betaFast > betaSlow)))) {
    set_error(HOM_ERR_INVALID,
              "%s: needs a positive base and factor, scaling 0 to 3, and for 3 a positive original length and "
              "betaFast > betaSlow",
              name);
    return;
  }
  hom::rotary::frequencies(reinterpret_cast<double *>(F.ptr), F.sizes[0], base, scaling, factor, originalLength,
                           betaFast, betaSlow, hom::current_stream());
}

}  // extern "C"
