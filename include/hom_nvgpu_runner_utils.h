/* C ABI of libhands_on_mlir_nvgpu_runner_utils.so, the runtime kernel layer that a
 * BERT model lowered by Hands-on-MLIR calls into.
 *
 * Part 1 declares, with identical names and argument lists, every entry point of
 * the reference's include/ExecutionEngine/HandsOnNVGPURunnerUtils.h:70-164 (the
 * symbol names the lowering emits are listed in
 * include/Conversions/Function/FunctionUtils.h:12-49).  A model .so produced by
 * the reference's compiler links against this library unchanged.
 *
 * Part 2 declares additions (prefix `hom`) that have no counterpart in the
 * reference: an error side channel (the reference aborts the process instead),
 * stream selection (the reference always uses the null stream), the
 * residual+affine LayerNorm of the op-level benchmark configuration, and
 * measurement hooks.
 *
 * Conventions shared by all compute entry points:
 *  - tensors are `(int64_t rank, void *descriptor)` pairs, see hom_memref.h;
 *    data must be row-major contiguous; `offset` is honoured.
 *  - work is enqueued on the library's current stream (null stream unless
 *    homSetStream() was called) of the current CUDA device and is not awaited.
 *  - nothing is returned; a rejected call launches nothing and records an error
 *    that homGetLastError() reports.  The process is never aborted.
 */
#ifndef HOM_NVGPU_RUNNER_UTILS_H
#define HOM_NVGPU_RUNNER_UTILS_H

#include <stdbool.h>
#include <stdint.h>

#include "hom_memref.h"

#if defined(__GNUC__)
#define HOM_EXPORT __attribute__((visibility("default")))
#else
#define HOM_EXPORT
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ===================================================================== Part 1 */

/* D = epilogue(alpha * A.B + beta * C); A [Bs,M,K], B [1,K,N], C/D [Bs,M,N], fp16 in and
 * out, fp32 accumulate and epilogue.  `activation` 1 = erf GELU, 0 = identity.  D may alias C.
 * C may also be [1,1,N] (bias broadcast over rows, as the reference's CPU matmulAddF32 does,
 * lib/ExecutionEngine/HandsOnRunnerUtils.cpp:258-266).  `gemmNum` 1..6 selects a row of the
 * sm_100a tile table (1-4: one CTA per 128 x {64,128,192,256} tile; 5-6: one CTA pair per
 * 256 x {128,256} tile; 0 or any other number = automatic); `splitKFactor` is a hint.
 * Replaces lib/ExecutionEngine/HandsOnNVGPURunnerUtils.cu:104-116 and
 * include/NVGPUKernels/GemmRunner.h:244-310. */
HOM_EXPORT void cutlassGemmF16(int64_t rankA, void *dstA, bool transa, int64_t rankB, void *dstB,
                               bool transb, int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                               int64_t activation, float alpha, float beta, int32_t gemmNum,
                               int32_t splitKFactor);

/* Empty stub in the reference (HandsOnNVGPURunnerUtils.cu:80-102); records "unsupported". */
HOM_EXPORT void cutlassGemmF32(int64_t rankA, void *dstA, bool transa, int64_t rankB, void *dstB,
                               bool transb, int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                               int64_t activation, float alpha, float beta);

/* D = act(A.B^T) (+ D when beta == 1 and C aliases D); A [Bs,M,K], B [1,N,K] with
 * transb == true, transa == false, alpha == 1, beta in {0,1}.  The reference ignores the two
 * trailing integers; here the first is a tile-table row hint like cutlassGemmF16's gemmNum.
 * Replaces HandsOnNVGPURunnerUtils.cu:172-183 and GemmRunner.h:322-426. */
HOM_EXPORT void nvteGemmF16(int64_t rankA, void *dstA, bool transa, int64_t rankB, void *dstB,
                            bool transb, int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                            int64_t activation, float alpha, float beta, int32_t gemmNum,
                            int32_t unused);

/* The GEMM <-> LayerNorm-statistics pair (HandsOnNVGPURunnerUtils.cu:118-170, :191-222;
 * include/NVGPUKernels/LayernormGemmRunner.h, Layernorm.h:107-194).
 * cutlassGemmWithVarMeanF16: D = alpha * A.B + beta * C, then for every row r of D
 *   Var[r] = 1 / sqrt(E[x^2] - mean^2 + eps), Mean[r] = -mean * Var[r]   (fp16, rank 1,
 *   at least Bs*M entries; `activation` is ignored as in the reference).
 * cutlassLayernormGemmF16: D = alpha * (A * Var[r] + Mean[r]).B + beta * C, i.e. the GEMM of
 *   the LayerNorm of A (scale 1, shift 0) with those statistics.
 * Neither is emitted by the compiler for BERT.  cutlassLayernormGemmF32 is an empty stub in
 * the reference and records "unsupported". */
HOM_EXPORT void cutlassGemmWithVarMeanF16(int64_t rankA, void *dstA, int64_t rankB, void *dstB,
                                          int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                                          int64_t rankVar, void *dstVar, int64_t rankMean,
                                          void *dstMean, float alpha, float beta,
                                          int64_t activation, float eps);
HOM_EXPORT void cutlassLayernormGemmF32(int64_t rankA, void *dstA, int64_t rankB, void *dstB,
                                        int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                                        int64_t rankVar, void *dstVar, int64_t rankMean,
                                        void *dstMean, float alpha, float beta,
                                        int64_t activation);
HOM_EXPORT void cutlassLayernormGemmF16(int64_t rankA, void *dstA, int64_t rankB, void *dstB,
                                        int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                                        int64_t rankVar, void *dstVar, int64_t rankMean,
                                        void *dstMean, float alpha, float beta,
                                        int64_t activation);

/* In-place x <- (x - mean) * rsqrt(var + eps) over the last dimension, biased variance,
 * fp32 statistics, no affine; rank 2 or 3.
 * Replaces HandsOnNVGPURunnerUtils.cu:300-310 and include/NVGPUKernels/Layernorm.h:584-694. */
HOM_EXPORT void nvteLayernormF32(int64_t rankA, void *dstA, float eps);
HOM_EXPORT void nvteLayernormF16(int64_t rankA, void *dstA, float eps);

/* O = softmax(scale * Q.K^T + padding mask).V per (batch, head), bidirectional.
 * A = packed QKV [bs, seq, 3*heads*d] with innermost order [3][heads][d];
 * Seqlen = int32 [bs+1] prefix sums of valid lengths; Out [bs, seq, heads*d].
 * Rows at padded query positions are written as zeros.
 * Replaces HandsOnNVGPURunnerUtils.cu:312-328 and
 * include/NVGPUKernels/BertAttentionRunner.h:19-137. */
HOM_EXPORT void nvteBertAttentionF32(int64_t rankA, void *dstA, int64_t rankSeqlen,
                                     void *dstSeqlen, int64_t rankOut, void *dstOut, float scale,
                                     int64_t headNum);
HOM_EXPORT void nvteBertAttentionF16(int64_t rankA, void *dstA, int64_t rankSeqlen,
                                     void *dstSeqlen, int64_t rankOut, void *dstOut, float scale,
                                     int64_t headNum);

/* Device allocation.  The descriptor is malloc()ed (callers free() it); the buffer is
 * released by dealloc*.  allocConstant* reads "<dir>/<idx>.txt" (first line: three
 * dimensions; then the values as text) and uploads it, converting to fp16 with
 * round-to-nearest-even for the F16 variant.
 * Replaces HandsOnNVGPURunnerUtils.cu:224-355 and allocHelper,
 * include/ExecutionEngine/HandsOnRunnerUtils.h:46-73. */
HOM_EXPORT HomUnrankedMemRef allocConstantNVGPUF32(int32_t idx);
HOM_EXPORT HomUnrankedMemRef allocConstantNVGPUF16(int32_t idx);
HOM_EXPORT HomUnrankedMemRef alloc3DMemRefNVGPUF32(int32_t a, int32_t b, int32_t c);
HOM_EXPORT HomUnrankedMemRef alloc3DMemRefNVGPUF16(int32_t a, int32_t b, int32_t c);
HOM_EXPORT HomUnrankedMemRef alloc1DMemRefNVGPUI32(int32_t n);
HOM_EXPORT void deallocNVGPUF32(int64_t rank, void *dst);
HOM_EXPORT void deallocNVGPUF16(int64_t rank, void *dst);
HOM_EXPORT void deallocNVGPUI32(int64_t rank, void *dst);

/* Out = A op B; same rank; B may have size-1 (broadcast) dimensions; arithmetic in the
 * element type.  Replaces HandsOnNVGPURunnerUtils.cu:357-365 and
 * include/NVGPUKernels/ElementwiseRunner.h:120-153. */
HOM_EXPORT void thrustElementwiseAddF32(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseSubF32(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseMulF32(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseDivF32(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseAddF16(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseSubF16(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseMulF16(int64_t, void *, int64_t, void *, int64_t, void *);
HOM_EXPORT void thrustElementwiseDivF16(int64_t, void *, int64_t, void *, int64_t, void *);

/* out[b,s,:] = table[0, indices[b,s], :]; indices int64 [bs,seq]; table [1,V,H].
 * Replaces HandsOnNVGPURunnerUtils.cu:367-368 and include/NVGPUKernels/GatherRunner.h:46-77. */
HOM_EXPORT void thrustGatherF32(int64_t rankIndices, void *desIndices, int64_t rankValue,
                                void *desValue, int64_t rankOut, void *desOut);
HOM_EXPORT void thrustGatherF16(int64_t rankIndices, void *desIndices, int64_t rankValue,
                                void *desValue, int64_t rankOut, void *desOut);

/* out[0] = 0; out[b+1] = sum over rows <= b of sum_j mask[row][j]; mask [bs,seq] int32/int64,
 * out int32 [bs+1].  Replaces HandsOnNVGPURunnerUtils.cu:370-371 and
 * include/NVGPUKernels/CuSeqLen.h:48-74. */
HOM_EXPORT void thrustCuSeqLenI32(int64_t rankInput, void *desInput, int64_t rankOut, void *desOut);
HOM_EXPORT void thrustCuSeqLenI64(int64_t rankInput, void *desInput, int64_t rankOut, void *desOut);

/* Prints "Print inside: <sizes>" to stderr (HandsOnNVGPURunnerUtils.h:58-68). */
HOM_EXPORT void printMemrefSizeF32(int64_t rank, void *descriptor);
HOM_EXPORT void printMemrefSizeF16(int64_t rank, void *descriptor);
HOM_EXPORT void printMemrefSizeI64(int64_t rank, void *descriptor);
HOM_EXPORT void printMemrefSizeI32(int64_t rank, void *descriptor);

/* ===================================================================== Part 2 */

/* Error side channel (per host thread).  Codes: 0 ok, 1 invalid argument, 2 unsupported,
 * 3 CUDA runtime error, 4 device-side wait expired, 5 I/O error. */
enum {
  HOM_OK = 0,
  HOM_ERR_INVALID = 1,
  HOM_ERR_UNSUPPORTED = 2,
  HOM_ERR_CUDA = 3,
  HOM_ERR_DEVICE_TIMEOUT = 4,
  HOM_ERR_IO = 5
};
HOM_EXPORT int homGetLastError(void);
HOM_EXPORT const char *homGetLastErrorString(void);
HOM_EXPORT void homClearLastError(void);

/* Stream used by this host thread's subsequent calls (a cudaStream_t; NULL = null stream). */
HOM_EXPORT void homSetStream(void *stream);
HOM_EXPORT void *homGetStream(void);
/* Waits for the stream, then folds the device status word into the error channel.
 * Returns the error code. */
HOM_EXPORT int homSynchronize(void);

/* Declares that no kernel will write [ptr, ptr + bytes) while GEMMs read it as their B operand
 * (model weights).  Kernels of this library are launched so that one may start while the previous
 * kernel of the stream is still finishing; a GEMM requests its first tiles of a DECLARED B before
 * that previous kernel is known to be complete, and those of any other B only afterwards, so a B
 * that an earlier call on the stream produced is always read after it was written.  What writes a
 * buffer must therefore be complete (homSynchronize) before the first call that reads it as
 * declared.  Buffers returned by allocConstantNVGPU* are declared by the library; callers that bring their own
 * weight buffers may declare them to get the earlier prefetch.  homForgetWeights() withdraws a
 * declaration (call it before the buffer is freed or reused).  What the library derives from a
 * declared weight and keeps (a re-pitched copy for N % 8 != 0; column sums for
 * cutlassLayernormGemmF16 and the deferred LayerNorm) is dropped when the weight is forgotten and
 * when it is declared again: declare a buffer again after rewriting its contents.  The first call
 * that derives something allocates and waits for its stream.  A captured cutlassLayernormGemmF16
 * computes its sums inside the graph; a graph captured with one of the other kept buffers shares
 * their ownership, so it stays valid, but has to be captured again to follow a new declaration.
 * No counterpart in the reference, whose launches are fully serialised on the null stream. */
HOM_EXPORT void homDeclareWeights(const void *ptr, int64_t bytes);
HOM_EXPORT void homForgetWeights(const void *ptr);

/* Directory that allocConstantNVGPU* reads "<idx>.txt" from (default: $HOM_CONSTANT_DIR,
 * else the current directory). */
HOM_EXPORT void homSetConstantDir(const char *dir);
/* Opt-in binary cache of parsed constants: with enable != 0 (or HOM_CONSTANT_CACHE=1)
 * allocConstantNVGPU* writes `<idx>.txt.homcache` (parsed fp32 values) beside the text file on
 * first use and reads it afterwards while the text file's size and modification time are
 * unchanged.  A weight directory that cannot be written just runs uncached. */
HOM_EXPORT void homSetConstantCache(int enable);

/* D = LayerNorm(fp16(A.B + R)) over the last dimension, no affine: what a GEMM with the
 * residual as C (beta 1) followed by nvteLayernormF16 leaves in D, in one launch.  The CTAs that
 * hold the column tiles of the same 128 rows form a thread-block cluster and exchange their row
 * sums through distributed shared memory, so the normalised rows are the only thing written.
 * A [.., M, K] fp16; B [1, K, N] (weightsNK false) or [1, N, K] (true); R [.., M, N] or a rank-0
 * descriptor (absent), may alias D; N must be c x {64,128,192,256} with c in {1,2,4,8} (256, 512,
 * 768, 1024, 1536, 2048, ...).  Statistics in fp32 from the fp16-rounded values (sum and sum of
 * squares).  No counterpart in the reference: it fuses the call pairs out-projection + LayerNorm
 * and FFN2 + LayerNorm of the lowered encoder layer. */
HOM_EXPORT void homGemmResidualLayernormF16(int64_t rankA, void *dstA, int64_t rankB, void *dstB,
                                            bool weightsNK, int64_t rankR, void *dstR, int64_t rankD,
                                            void *dstD, float eps);

/* The embedding stage of the lowered BERT in one launch: what the five calls
 * thrustGatherF16(ids, word) ; thrustGatherF16(types, typeEmb) ; thrustElementwiseAddF16 x2 ;
 * nvteLayernormF16 leave in Out, bit for bit (each fp16 addition rounded, fp32 statistics, no
 * affine).  ids, types int64 [bs,seq]; word [1,V,H], pos [1,seq,H], typeEmb [1,T,H], Out
 * [bs,seq,H] fp16; out-of-range indices read as zero rows.  No counterpart in the reference:
 * a compiler pass would have to emit it in place of the five calls. */
HOM_EXPORT void homBertEmbeddingF16(int64_t rankIds, void *dstIds, int64_t rankTypes, void *dstTypes,
                                    int64_t rankWord, void *dstWord, int64_t rankPos, void *dstPos,
                                    int64_t rankTypeEmb, void *dstTypeEmb, int64_t rankOut,
                                    void *dstOut, float eps);

/* GEMM with the LayerNorms around it deferred into its epilogue, so that a post-LayerNorm
 * transformer layer needs no LayerNorm launch at all:
 *   D = act( LN?(A).B + LN?(R) ),  and optionally the row statistics of D for the next call.
 * Every tensor that is "raw" (not yet normalised) travels with fp32 partial sums of its rows,
 * shape [ceil(width / 64), rows, 2] = {sum, sum of squares} per 64-column group, exactly what a
 * previous call wrote through StatsD.  StatsA given: A is raw and the epilogue computes
 * LN(A).B as rstd * (A.B) - mean * rstd * colsum(B) (column sums of a declared weight are kept).
 * StatsR given: the residual added is LN(R) = rstd * R - mean * rstd (R raw; R may alias D).
 * StatsD given: the epilogue writes D's partial sums (of the fp16-rounded values) there.  Absent
 * operands are rank-0 / null descriptors.  LayerNorm is the reference's (no affine, biased
 * variance, eps inside the square root); statistics stay in fp32 - the sm_100a form of the
 * reference's experimental cutlassGemmWithVarMeanF16 / cutlassLayernormGemmF16 pair
 * (include/NVGPUKernels/LayernormGemmRunner.h:17-361), which stores them in fp16 and cannot
 * express BERT's normalised residual.  A [.., M, K], B [1, K, N] or [1, N, K] (weightsNK),
 * R, D [.., M, N], N % 8 == 0; activation 0 or 1 (erf GELU).  StatsD must not be the buffer
 * of StatsA or StatsR (other tiles still read them).  With StatsA, the first call for a declared
 * weight computes and caches its column sums (allocates device memory and waits for the stream).
 * For any other B, and for a declared weight that is first seen under stream capture, an extra
 * launch recomputes them on every call or replay (N <= 65536). */
HOM_EXPORT void homGemmDeferredLayernormF16(int64_t rankA, void *dstA, int64_t rankStatsA, void *dstStatsA,
                                            int64_t rankB, void *dstB, bool weightsNK, int64_t rankR,
                                            void *dstR, int64_t rankStatsR, void *dstStatsR, int64_t rankD,
                                            void *dstD, int64_t rankStatsD, void *dstStatsD,
                                            int64_t activation, float eps);

/* Out = LayerNorm(X + R) * gamma + beta over the last dimension; X, R, Out [rows.., H]
 * fp16 (R, gamma, beta may be rank-0 descriptors = absent), fp32 sum and statistics,
 * one fp16 rounding at the store.  Out may alias X. */
HOM_EXPORT void homResidualLayernormF16(int64_t rankX, void *dstX, int64_t rankR, void *dstR,
                                        int64_t rankGamma, void *dstGamma, int64_t rankBeta,
                                        void *dstBeta, int64_t rankOut, void *dstOut, float eps);

/* cutlassLayernormGemmF16 for callers that must not allocate device memory - a process whose
 * memory was budgeted once at start-up, a plug-in running under a framework where cudaMalloc
 * would stall every stream of the device, a latency-critical loop.  Same operands and result:
 * D = alpha * (A * Var[r] + Mean[r]).B + beta * C (A [Bs,M,K], B [1,K,N], C [Bs,M,N] or
 * [1,1,N] or unused when beta == 0, D [Bs,M,N], Var/Mean fp16 [>= Bs*M]).  The column sums of
 * B that the computation needs live in a fixed 64 KB array inside the library image instead
 * of a cudaMalloc'ed buffer, so N is limited to 16384 columns (larger N: error 2, nothing is
 * launched) and every GPU that loads the library carries those 64 KB until the process ends.
 * The call performs no cudaMalloc / cudaFree / cudaHostAlloc and uses no allocating library.
 * The first call on each device looks up the array's device address (with that device
 * current); make that first call outside of any stream capture.  All calls share the one
 * array: each call rewrites the entries it uses before reading them, so nothing needs
 * clearing between calls, but two calls whose kernels overlap on the GPU (different streams,
 * or host threads on one device) would overwrite each other's sums - issue them on one stream.
 * Its launches are counted but never timed by homOpTimingEnable (timing allocates events), and
 * an expired device-side wait is reported by homSynchronize() only if some other entry point of
 * this library has run on the device before (that is what creates the status word; this one
 * will not allocate it).  This entry point has no counterpart in the reference. */
HOM_EXPORT void homLayernormGemmF16NoAlloc(int64_t rankA, void *dstA, int64_t rankB, void *dstB,
                                           int64_t rankC, void *dstC, int64_t rankD, void *dstD,
                                           int64_t rankVar, void *dstVar, int64_t rankMean,
                                           void *dstMean, float alpha, float beta);

/* Microscaled 4-bit floating point: 32 consecutive values along K share a power of two, each is one
 * of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it.  A matrix [rows, K] is held as two uint8 memrefs:
 *   Q  [.., rows, 16 * ceil(K / 32)]: two codes to a byte, the even column in the low half (sign,
 *      two exponent bits, one mantissa bit); columns beyond K are 0;
 *   S  [ceil(rows / 128), ceil(ceil(K / 32) / 4), 512]: the scale byte s of row r and block b,
 *      meaning 2^(s - 127) (255: NaN), is byte (r % 32) * 16 + (r / 32) % 4 * 4 + b % 4 of tile
 *      (r / 128, b / 4); bytes of rows and blocks beyond the matrix are 0.
 * Both 16-byte aligned.  Leading dimensions of a rank-3 operand count as rows.  K and rows may be
 * anything from 1 to 2^30; a matrix without elements is a call without effect.  An output must not
 * overlap another operand (C may be D).
 *
 * homQuantizeMxF4*: the block's power of two is 2^(floor(log2 max|x|) - 2), at least 2^-127; values
 * over it are rounded to the nearest code, ties to even, magnitudes above 6 to 6.  A block that
 * holds a NaN or an infinity becomes NaN as a whole.  X [.., rows, K] (any element alignment), or
 * [K, rows] / [1, K, rows] with `transposed` (a weight stored [1,K,N]): the blocks run along K
 * either way.  All of Q and S is written, and a declaration (homDeclareWeights) that holds any of
 * it is withdrawn: products after this call read it only after it was written, and fetch it early
 * again once it is declared anew.
 * homDequantizeMxF4*: Out [.., rows, K] = the values; exact in fp32, in fp16 wherever the values
 * came from fp16.
 * No counterpart in the reference, whose path is fp16 throughout. */
HOM_EXPORT void homQuantizeMxF4F16(int64_t rankX, void *dstX, bool transposed, int64_t rankQ, void *dstQ,
                                   int64_t rankS, void *dstS);
HOM_EXPORT void homQuantizeMxF4F32(int64_t rankX, void *dstX, bool transposed, int64_t rankQ, void *dstQ,
                                   int64_t rankS, void *dstS);
HOM_EXPORT void homDequantizeMxF4F16(int64_t rankQ, void *dstQ, int64_t rankS, void *dstS, int64_t rankOut,
                                     void *dstOut);
HOM_EXPORT void homDequantizeMxF4F32(int64_t rankQ, void *dstQ, int64_t rankS, void *dstS, int64_t rankOut,
                                     void *dstOut);

/* D = epilogue(alpha * A.B^T + beta * C) of two such matrices, A [.., M, K] and B [N, K] or
 * [1, N, K] with equal numbers of blocks: the 4-bit counterpart of nvteGemmF16 with its epilogue
 * (fp32 accumulation; fp16 C and D; C [.., M, N], which may be D, or one row of N; unused when
 * beta == 0; `activation` 1 = erf GELU).  D (and C) 16-byte aligned when N % 8 == 0.  Q and S of
 * the weight may be declared (homDeclareWeights, one declaration each) to be fetched early: after
 * the stream that quantised them was waited for. */
HOM_EXPORT void homGemmMxF4F16(int64_t rankA, void *dstA, int64_t rankSA, void *dstSA, int64_t rankB,
                               void *dstB, int64_t rankSB, void *dstSB, int64_t rankC, void *dstC,
                               int64_t rankD, void *dstD, int64_t activation, float alpha, float beta);

/* Rotary positions.  The first 2F dimensions of every head, F = entries of Frequencies, are F pairs
 * (i, F + i), or (2i, 2i + 1) with `interleaved`; pair i of a token at position p is turned by
 * p * Frequencies[i] radians and multiplied by `magnitude`:
 *   y0 = magnitude * (x0 cos - x1 sin),   y1 = magnitude * (x1 cos + x0 sin).
 * `backward` applies the transpose, which takes the gradient of Out to that of X.  Dimensions
 * beyond 2F are copied.  X, Out [bs, seq, heads, d] with any non-negative strides and a contiguous
 * last dimension - the query and key heads of a packed [bs, seq, 3*heads*d] are the view
 * [bs, seq, 2*heads, d] of it -.  Out may be X; otherwise its addresses, from the first to the last
 * element, must not meet those of X (which those of two groups of heads of one packed buffer do),
 * nor in any case those of Positions and Frequencies; and its dimensions, in the order of their
 * strides, must each lie within one step of the next.  Positions int64 [bs, seq] or [1, seq], absent
 * (rank 0 / null): 0 .. seq - 1; bs * seq and heads * d below 2^31.  Frequencies fp64 [F], F <= 512;
 * angles are formed in 64 bits, so that far positions keep their fractions of a turn.  The
 * rotation is fp32, rounded once.
 * No counterpart in the reference, whose model adds a position table. */
HOM_EXPORT void homRotaryF16(int64_t rankX, void *dstX, int64_t rankPos, void *dstPos, int64_t rankFreq,
                             void *dstFreq, int64_t rankOut, void *dstOut, bool interleaved, bool backward,
                             float magnitude);
HOM_EXPORT void homRotaryF32(int64_t rankX, void *dstX, int64_t rankPos, void *dstPos, int64_t rankFreq,
                             void *dstFreq, int64_t rankOut, void *dstOut, bool interleaved, bool backward,
                             float magnitude);
/* Fills Frequencies (fp64 [F], on the device) with f_i = base^(-i / F).  `scaling` for contexts that
 * are `factor` times longer: 0 none; 1 linear: f_i / factor; 2 changed base: base * factor^(F / (F - 1))
 * instead of base, which leaves the fastest pair alone and slows the slowest by factor; 3 by parts:
 * a pair that makes t = originalLength * f_i / (2 pi) turns keeps the share
 * g = clamp((t - betaSlow) / (betaFast - betaSlow), 0, 1) of its frequency and has the rest divided:
 * f_i * (g + (1 - g) / factor). */
HOM_EXPORT void homRotaryFrequencies(int64_t rankFreq, void *dstFreq, double base, int32_t scaling, double factor,
                                     double originalLength, double betaFast, double betaSlow);

/* Number of kernels this library has launched since load (all threads). */
HOM_EXPORT int64_t homKernelLaunchCount(void);

/* Per-launch timing: while enabled every entry point brackets its kernel with events on
 * the current stream.  homOpTimingCollect() synchronises, writes up to `capacity` records
 * (kind: 1 gemm, 2 layernorm, 3 attention, 4 elementwise, 5 gather, 6 cu_seqlen, 7 conversion
 * to or from 4 bits, 8 rotary; ms; and the algorithmic flop and byte counts of that launch), clears the log and returns the
 * number of records that were available. */
typedef struct HomOpTiming {
  int32_t kind;
  float ms;
  double flops;
  double bytes;
} HomOpTiming;
HOM_EXPORT void homOpTimingEnable(int enable);
HOM_EXPORT int64_t homOpTimingCollect(HomOpTiming *out, int64_t capacity);
/* The same read-out without releasing the records: for launches that were captured into a CUDA
 * graph while timing was enabled (their event records became graph nodes), call it after each
 * replay; call homOpTimingCollect once the graph is gone. */
HOM_EXPORT int64_t homOpTimingPeek(HomOpTiming *out, int64_t capacity);

/* The tile the GEMM family would run for (M, N, K, activation): the tile's N extent,
 * pipeline stages and split-K.  Returns the tile-table row number (usable as gemmNum). */
HOM_EXPORT int32_t homGemmQueryTile(int64_t m, int64_t n, int64_t k, int64_t activation,
                                    int32_t *bn, int32_t *stages, int32_t *splitK);

/* Run-time tuner with the contract of GemmProfiler::profile
 * (lib/NVGPUKernels/GemmProfiler.cu:143-236, include/NVGPUKernels/GemmProfiler.h:39-57): times every
 * row of the tile table for fp16 (M, N, K, activation, alpha, beta) on scratch operands it
 * allocates and frees (beta != 0 reads C = D), returns the fastest row in *tile_row (usable as
 * gemmNum; the autotune pass writes it to `kernel_name`) and 1 in *split_k, and remembers the
 * result so that later calls with an automatic gemmNum use it.  weights_nk != 0 times the
 * [1,N,K] weight layout.  row_us, if not null, receives the six per-row times in microseconds.
 * Blocks until the measurements are done; call it outside stream capture.  Returns the error
 * code (0 = ok). */
HOM_EXPORT int32_t homGemmTune(int64_t m, int64_t n, int64_t k, int64_t activation, float alpha,
                               float beta, int32_t weights_nk, int32_t iterations,
                               int32_t *tile_row, int32_t *split_k, float *best_us, float *row_us);
/* The tuned table as text, one "M N K activation row" line per shape (the reference keeps its
 * timing cache in memory only).  Return the number of entries, or -1 if the file cannot be
 * opened.  $HOM_TUNE_CACHE names a file that is loaded on first use. */
HOM_EXPORT int32_t homGemmTuneSave(const char *path);
HOM_EXPORT int32_t homGemmTuneLoad(const char *path);

#ifdef __cplusplus
}
#endif

#endif /* HOM_NVGPU_RUNNER_UTILS_H */
