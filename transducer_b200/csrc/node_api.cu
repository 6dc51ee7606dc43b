// C ABI of the operators on single lattice nodes (include/transducer_b200.h, last part).
#include <algorithm>
#include <cmath>

#include "api_guard.h"
#include "kernels.h"

namespace tb200 {
namespace {

NodeArgs node_args(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                   long long pStrideB, long long pStrideU, const int* frames, const int* positions, int B,
                   int maxT, int maxU, int V, int N) {
  check(B >= 0 && maxT >= 0 && maxU >= 0 && N >= 0 && V > 0,
        "negative batch/length/number of nodes or non-positive alphabet size");
  check(eStrideB >= 0 && eStrideT >= 0 && pStrideB >= 0 && pStrideU >= 0, "negative stride");
  check((long long)B * N < 0x7fffffffLL, "too many nodes (batchSize * nodes must be below 2^31 - 1)");
  check((long long)B * maxT <= 0x7fff0000LL && (long long)B * maxU <= 0x7fff0000LL,
        "too many rows (batchSize * maxInputLength and batchSize * maxLabelLength must be at most 2^31 - 2^16)");
  check(V <= 1 << 28, "the alphabet must not exceed 2^28 words");
  return NodeArgs{E, P, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT, maxU, V, N,
                  bf16 ? kDtypeBf16 : kDtypeF32};
}

void check_listed(int K) {
  check(K >= 1 && K <= kMaxListedWords, "the number of listed words must be between 1 and 256");
}
void check_temperature(double t) {
  // (it and its reciprocal are used in 32 bits)
  check(t > 0.0 && t <= 1e30 && std::isfinite((float)(1.4426950408889634 / t)),
        "temperature must be positive, at least 1e-38 and at most 1e30");
}

}  // namespace

bool node_rows_aligned(const NodeArgs& a) {
  const int size = a.dtype == kDtypeBf16 ? 2 : 4;
  const i64 bytes[] = {(i64)reinterpret_cast<uintptr_t>(a.E), (i64)reinterpret_cast<uintptr_t>(a.P),
                       a.eStrideB * size, a.eStrideT * size, a.pStrideB * size, a.pStrideU * size,
                       (i64)a.V * size};
  return std::all_of(std::begin(bytes), std::end(bytes), [](i64 x) { return x % 16 == 0; });
}

}  // namespace tb200

using namespace tb200;

extern "C" {

size_t tb200_node_summary_scratch_bytes(void) { return 64 * 3 * sizeof(int); }

int tb200_node_summary(const int* frames, const int* positions, long long nodes, const int* words,
                       long long wordCount, void* scratch, int* most) {
  return guarded([&] {
    check(nodes >= 0 && wordCount >= 0 && scratch && most, "null pointer or negative count");
    int host[64 * 3];
    const int ctas = node_summary_ctas(nodes, wordCount);
    launch_node_summary(frames, positions, nodes, words, wordCount, static_cast<int*>(scratch), api_stream());
    TB200_CUDA_CHECK(cudaMemcpyAsync(host, scratch, sizeof(int) * 3 * ctas, cudaMemcpyDeviceToHost, api_stream()));
    TB200_CUDA_CHECK(cudaStreamSynchronize(api_stream()));
    for (int k = 0; k < 3; ++k) {
      most[k] = host[k];
      for (int c = 1; c < ctas; ++c) most[k] = host[3 * c + k] > most[k] ? host[3 * c + k] : most[k];
    }
  });
}

int tb200_top_words(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                    long long pStrideB, long long pStrideU, const int* frames, const int* positions, int* words,
                    float* logits, float* rest, int B, int maxT, int maxU, int V, int N, int k,
                    double temperature) {
  return guarded([&] {
    const NodeArgs a = node_args(E, P, bf16, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT,
                                 maxU, V, N);
    check_listed(k);
    check(k <= V, "the number of listed words must not exceed the alphabet size");
    check_temperature(temperature);
    launch_top_words(a, words, logits, rest, k, temperature, api_stream());
  });
}

int tb200_sample_words(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                       long long pStrideB, long long pStrideU, const int* frames, const int* positions,
                       const float* uniforms, int* words, float* logProbs, int B, int maxT, int maxU, int V, int N,
                       double temperature, int topK, double topP, double minP) {
  return guarded([&] {
    const NodeArgs a = node_args(E, P, bf16, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT,
                                 maxU, V, N);
    if (!(temperature == 0.0)) check_temperature(temperature);
    check(topK >= 0, "top_k must not be negative");
    check(topP > 0.0 && topP <= 1.0, "top_p must be above 0 and at most 1");
    check(minP >= 0.0 && minP <= 1.0, "min_p must be between 0 and 1");
    launch_sample_words(a, uniforms, words, logProbs, SampleRule{temperature, topK, topP, minP}, api_stream());
  });
}

size_t tb200_extend_beams_workspace_bytes(int B, int V, int N) { return extend_workspace_bytes(B, V, N); }

int tb200_extend_beams(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                       long long pStrideB, long long pStrideU, const int* frames, const int* positions,
                       const float* scores, float* outScores, int* parents, int* words, int B, int maxT, int maxU,
                       int V, int N, int width, int* beyond, void* workspace, size_t workspaceBytes) {
  return guarded([&] {
    const NodeArgs a = node_args(E, P, bf16, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT,
                                 maxU, V, N);
    check(width >= 1 && width <= kMaxListedWords, "the number of extensions must be between 1 and 256");
    need(workspaceBytes, extend_workspace_bytes(B, V, N), workspace, "workspace");
    launch_extend_beams(a, scores, outScores, parents, words, width, beyond, workspace, api_stream());
  });
}

size_t tb200_distill_saved_bytes(int B, int maxT, int maxU, int N, int K) {
  return distill_saved_bytes(B, maxT, maxU, N, K);
}

int tb200_distill_forward(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                          long long pStrideB, long long pStrideU, const int* frames, const int* positions,
                          const int* words, const float* logits, const float* rest, float* costs, void* saved,
                          size_t savedBytes, int B, int maxT, int maxU, int V, int N, int K,
                          double temperature) {
  return guarded([&] {
    const NodeArgs a = node_args(E, P, bf16, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT,
                                 maxU, V, N);
    check_listed(K);
    check_temperature(temperature);
    if (saved) need(savedBytes, distill_saved_bytes(B, maxT, maxU, N, K), saved, "saved state");
    const DistillSaved state = distill_saved(B > 0 ? saved : nullptr, B, maxT, maxU, V, N, K);
    launch_distill_forward(a, words, logits, rest, costs, state, K, temperature, api_stream());
  });
}

size_t tb200_distill_backward_workspace_bytes(int B, int maxT, int maxU, int V, int N) {
  return distill_backward_workspace_bytes(B, maxT, maxU, V, N);
}

int tb200_distill_backward(const void* E, const void* P, int bf16, long long eStrideB, long long eStrideT,
                           long long pStrideB, long long pStrideU, const int* frames, const int* positions,
                           const int* words, const void* saved, size_t savedBytes, const float* weights,
                           void* egrads, void* pgrads, int B, int maxT, int maxU, int V, int N, int K,
                           double temperature, void* workspace, size_t workspaceBytes) {
  return guarded([&] {
    const NodeArgs a = node_args(E, P, bf16, eStrideB, eStrideT, pStrideB, pStrideU, frames, positions, B, maxT,
                                 maxU, V, N);
    check_listed(K);
    check_temperature(temperature);
    need(savedBytes, distill_saved_bytes(B, maxT, maxU, N, K), saved, "saved state");
    need(workspaceBytes, tb200_distill_backward_workspace_bytes(B, maxT, maxU, V, N), workspace, "workspace");
    const DistillSaved state = distill_saved(const_cast<void*>(saved), B, maxT, maxU, V, N, K);
    launch_distill_backward(a, words, state, weights, egrads, pgrads, K, temperature, workspace, api_stream());
  });
}

}  // extern "C"
