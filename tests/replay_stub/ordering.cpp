// The replay program on a runtime that computes nothing and only keeps account of order: which of the work issued so far a
// stream has waited for when it is given the next piece.  Every call of a program works on the program's buffers, so a
// piece that does not come after all the others is a race.  Linked with bert_replay.cpp in place of the CUDA runtime and
// of the kernel library; prints what is wrong, or `ok`.
//   usage: ordering <scenario>
#include <cuda_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <string>

#include "hom_bert_replay.h"
#include "hom_nvgpu_runner_utils.h"

namespace {

using Seen = std::set<int>;
std::map<void *, Seen> stream_seen;  // by stream: pieces that are over before what is issued next
std::map<void *, Seen> event_seen;
Seen host_seen;                      // what the host has waited for
std::set<void *> capturing;
std::map<void *, int> graph_bound_at;  // by graph: how many weights had been bound when it was captured
int issued = 0, bound = 0, streams_made = 0, graphs_launched = 0, faults = 0;
bool pinned = true;
void *current = nullptr;
uintptr_t next_handle = 0x1000;

void *handle() { return reinterpret_cast<void *>(next_handle += 16); }

void piece(void *stream, const char *what) {
  if (capturing.count(stream)) return;
  Seen &seen = stream_seen[stream];
  seen.insert(host_seen.begin(), host_seen.end());
  if (static_cast<int>(seen.size()) != issued) {
    std::printf("%s on stream %p does not wait for %d earlier pieces\n", what, stream,
                issued - static_cast<int>(seen.size()));
    ++faults;
    for (int i = 0; i < issued; ++i) seen.insert(i);  // report it once
  }
  seen.insert(issued++);
}

HomUnrankedMemRef memref(std::initializer_list<int64_t> sizes) {
  const int64_t rank = static_cast<int64_t>(sizes.size());
  auto *words = static_cast<int64_t *>(std::calloc(3 + 2 * rank, 8));
  words[0] = words[1] = reinterpret_cast<int64_t>(handle());
  int64_t i = 0, stride = 1;
  for (int64_t s : sizes) words[3 + i++] = s;
  for (i = rank - 1; i >= 0; --i) words[3 + rank + i] = stride, stride *= words[3 + i];
  return HomUnrankedMemRef{rank, words};
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------- CUDA runtime
void **__cudaRegisterFatBinary(void *) { static void *p; return &p; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *, dim3 *, int *) {}
static void *launch_stream;
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t stream) { launch_stream = stream; return 0; }
cudaError_t __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *stream) {
  *static_cast<void **>(stream) = launch_stream;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t stream) {
  piece(stream, "a staging kernel");
  return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void *, const void *, size_t, cudaMemcpyKind kind, cudaStream_t stream) {
  // (a delivery to the host beside the next step is meant to overlap with it: not a piece)
  if (kind == cudaMemcpyHostToDevice || stream == current) piece(stream, "a copy");
  return cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t *stream, unsigned flags) {
  if (flags != cudaStreamNonBlocking) std::abort();  // (others wait for the default stream: not modelled)
  *stream = static_cast<cudaStream_t>(handle());
  ++streams_made;
  return cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t stream) {
  const Seen &seen = stream_seen[stream];
  host_seen.insert(seen.begin(), seen.end());
  return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *event, unsigned) {
  *event = static_cast<cudaEvent_t>(handle());
  return cudaSuccess;
}
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t event, cudaStream_t stream) {
  event_seen[event] = stream_seen[stream];
  return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t stream, cudaEvent_t event, unsigned) {
  stream_seen[stream].insert(event_seen[event].begin(), event_seen[event].end());
  return cudaSuccess;
}
cudaError_t cudaStreamBeginCapture(cudaStream_t stream, cudaStreamCaptureMode) {
  if (!stream) return cudaErrorStreamCaptureUnsupported;
  capturing.insert(stream);
  return cudaSuccess;
}
cudaError_t cudaStreamEndCapture(cudaStream_t stream, cudaGraph_t *graph) {
  capturing.erase(stream);
  *graph = static_cast<cudaGraph_t>(handle());
  graph_bound_at[*graph] = bound;
  return cudaSuccess;
}
cudaError_t cudaGraphInstantiate(cudaGraphExec_t *exec, cudaGraph_t graph, unsigned long long) {
  *exec = static_cast<cudaGraphExec_t>(handle());
  graph_bound_at[*exec] = graph_bound_at[graph];
  return cudaSuccess;
}
cudaError_t cudaGraphDestroy(cudaGraph_t) { return cudaSuccess; }
cudaError_t cudaGraphExecDestroy(cudaGraphExec_t exec) {
  graph_bound_at.erase(exec);
  return cudaSuccess;
}
cudaError_t cudaGraphLaunch(cudaGraphExec_t exec, cudaStream_t stream) {
  if (!graph_bound_at.count(exec)) {
    std::printf("a graph is launched that is gone\n");
    ++faults;
  } else if (graph_bound_at[exec] != bound) {
    std::printf("a graph is launched that holds weights bound before the present ones\n");
    ++faults;
  }
  ++graphs_launched;
  piece(stream, "a graph");
  return cudaSuccess;
}
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes *attributes, const void *ptr) {
  std::memset(attributes, 0, sizeof *attributes);
  attributes->type = pinned ? cudaMemoryTypeHost : cudaMemoryTypeUnregistered;
  attributes->devicePointer = pinned ? const_cast<void *>(ptr) : nullptr;
  return cudaSuccess;
}

// ----------------------------------------------------------------------------- kernel library
HomUnrankedMemRef alloc3DMemRefNVGPUF16(int32_t a, int32_t b, int32_t c) { return memref({a, b, c}); }
HomUnrankedMemRef alloc3DMemRefNVGPUF32(int32_t a, int32_t b, int32_t c) { return memref({a, b, c}); }
HomUnrankedMemRef alloc1DMemRefNVGPUI32(int32_t a) { return memref({a}); }
HomUnrankedMemRef allocConstantNVGPUF16(int32_t) {
  ++bound;
  return memref({1, 64, 64});
}
void deallocNVGPUF16(int64_t, void *) {}
void deallocNVGPUI32(int64_t, void *) {}
void homDeclareWeights(const void *, int64_t) { ++bound; }
void homForgetWeights(const void *) {}
int homGetLastError(void) { return 0; }
void homSetStream(void *stream) { current = stream; }
void *homGetStream(void) { return current; }
int homSynchronize(void) { return cudaStreamSynchronize(static_cast<cudaStream_t>(current)), 0; }

#define MEMREF int64_t, void *
void cutlassGemmF16(MEMREF, bool, MEMREF, bool, MEMREF, MEMREF, int64_t, float, float, int32_t, int32_t) { piece(current, "a GEMM"); }
void nvteGemmF16(MEMREF, bool, MEMREF, bool, MEMREF, MEMREF, int64_t, float, float, int32_t, int32_t) { piece(current, "a GEMM"); }
void homBertEmbeddingF16(MEMREF, MEMREF, MEMREF, MEMREF, MEMREF, MEMREF, float) { piece(current, "an embedding"); }
void homGemmDeferredLayernormF16(MEMREF, MEMREF, MEMREF, bool, MEMREF, MEMREF, MEMREF, MEMREF, int64_t, float) { piece(current, "a GEMM"); }
void homGemmResidualLayernormF16(MEMREF, MEMREF, bool, MEMREF, MEMREF, float) { piece(current, "a GEMM"); }
void homQuantizeMxF4F16(MEMREF, bool, MEMREF, MEMREF) { piece(current, "a quantisation"); }
void homGemmMxF4F16(MEMREF, MEMREF, MEMREF, MEMREF, MEMREF, MEMREF, int64_t, float, float) { piece(current, "a product"); }
void homRotaryF16(MEMREF, MEMREF, MEMREF, MEMREF, bool, bool, float) { piece(current, "a rotation"); }
void homRotaryFrequencies(MEMREF, double, int32_t, double, double, double, double) { piece(current, "the frequencies"); }
void nvteBertAttentionF16(MEMREF, MEMREF, MEMREF, float, int64_t) { piece(current, "an attention"); }
void nvteLayernormF16(MEMREF, float) { piece(current, "a LayerNorm"); }
void thrustCuSeqLenI64(MEMREF, MEMREF) { piece(current, "the lengths"); }
void thrustElementwiseAddF16(MEMREF, MEMREF, MEMREF) { piece(current, "an addition"); }
void thrustGatherF16(MEMREF, MEMREF, MEMREF) { piece(current, "a gather"); }

}  // extern "C"

namespace {

void require(bool ok, const char *what) {
  if (ok) return;
  std::printf("%s\n", what);
  ++faults;
}

void bind(void *program, const HomBertConfig &cfg) {
  for (int i = 0; i < homBertWeightCount(&cfg); ++i) {
    HomUnrankedMemRef w = memref({1, 64, 64});
    require(homBertSetWeight(program, i, w.rank, w.descriptor) == 0, "a weight is refused");
    std::free(w.descriptor);
  }
}

}  // namespace

int main(int argc, char **argv) {
  const std::string scenario = argc > 1 ? argv[1] : "";
  HomBertConfig cfg{};
  cfg.layers = 2, cfg.hidden = 64, cfg.heads = 1, cfg.ffn = 64, cfg.vocab = 64, cfg.type_vocab = 2, cfg.batch = 1, cfg.seq = 8;
  cfg.eps = 1e-12f;
  if (scenario == "deferred_layernorm") cfg.fused_layernorm = 2;
  void *program = homBertCreate(&cfg);
  bind(program, cfg);
  HomUnrankedMemRef ids = memref({1, 8}), mask = memref({1, 8}), types = memref({1, 8}), result{};
  auto forward = [&](int use_graph) {
    require(homBertForward(program, 2, ids.descriptor, 2, mask.descriptor, 2, types.descriptor, &result, use_graph) == 0,
            "a forward is refused");
  };
  int64_t host[8] = {};
  char out[2][8 * 64 * 2];
  int steps = 0;
  auto host_step = [&](int use_graph) {
    require(homBertForwardHostAsync(program, host, host, host, out[steps++ & 1], use_graph) == 0, "a host step is refused");
  };

  if (scenario == "default_stream" || scenario == "deferred_layernorm") {
    forward(0);
    forward(0);
    for (int i = 0; i < 4; ++i) forward(1);
    require(graphs_launched == 4, "expected four graph launches");
  } else if (scenario == "options") {
    for (int i = 0; i < 3; ++i) forward(1);
    require(homBertSetRotary(program, 1e4, 0, 1, 0, 32, 1, 1) == 0, "set_rotary is refused");
    for (int i = 0; i < 3; ++i) forward(1);
    require(homBertQuantizeWeights(program) == 0, "quantize_weights is refused");
    for (int i = 0; i < 3; ++i) forward(1);
    require(graphs_launched == 6, "expected six graph launches");
  } else if (scenario == "host_buffers") {
    for (int i = 0; i < 4; ++i)
      require(homBertForwardHost(program, host, host, host, out[0], 1) == 0, "a host forward is refused");
    pinned = false;
    for (int i = 0; i < 4; ++i) host_step(1);
  } else if (scenario == "callers_stream") {
    homSetStream(handle());
    for (int i = 0; i < 4; ++i) forward(1);
    require(streams_made == 0, "a stream of the program's own where the caller's can be captured");
    require(graphs_launched == 3, "expected three graph launches");
  } else if (scenario == "new_weights" || scenario == "new_constants") {
    homSetStream(handle());
    for (int round = 0; round < 3; ++round) {
      for (int i = 0; i < 3; ++i) forward(1);
      for (int i = 0; i < 5; ++i) host_step(1);
      if (scenario == "new_weights") bind(program, cfg);
      else require(homBertLoadConstants(program, 0) == 0, "constants are refused");
    }
    require(graphs_launched > 0, "expected graph launches");
  } else {
    std::printf("no such scenario\n");
    return 2;
  }
  homBertDestroy(program);
  if (faults == 0) std::printf("ok\n");
  return faults != 0;
}
