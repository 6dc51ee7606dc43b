// C ABI of the states that follow a beam search's hypotheses and of words' embeddings (include/transducer_b200.h, last
// part), and the flags that checked calls read.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "api_guard.h"
#include "kernels.h"

namespace tb200 {
namespace {

EmbedArgs embed_args(const void* table, int bf16, long long stride, const int* words, long long count, int R, int H,
                     double scale, double dropout, long long seed, const long long* seedAt) {
  check(count >= 0 && R >= 0 && H >= 0 && stride >= 0, "negative size or stride");
  check(count < 0x7fffffffLL, "too many words (there must be fewer than 2^31 - 1)");
  check(R <= 1 << 28 && H <= 1 << 23, "the table must have at most 2^28 rows of 2^23 numbers");
  check(dropout >= 0.0 && dropout < 1.0, "dropout must be at least 0 and below 1");
  const unsigned dropped = std::min(65535u, (unsigned)std::nearbyint(dropout * 65536.0));
  const double factor = scale * 65536.0 / (65536.0 - dropped);
  check(std::isfinite((float)factor), "scale must be finite");
  return EmbedArgs{table, stride, words, count, R, H, bf16 ? kDtypeBf16 : kDtypeF32, (float)factor, dropped, seed, seedAt};
}

// Flags that no call uses at present, all 0.  A call's kernels write its own in host memory, only where an index is
// beyond its tensor: to read them takes the wait for the stream and no copy.
std::mutex g_flags;
std::vector<int*> g_free;
constexpr int kFlagsAtOnce = 64, kFlagInts = 16;   // (64 bytes each)

int* take_flags() {
  std::lock_guard<std::mutex> lock(g_flags);
  if (g_free.empty()) {
    int* p = nullptr;
    const unsigned how = cudaHostAllocPortable | cudaHostAllocMapped;
    TB200_CUDA_CHECK(cudaHostAlloc(&p, kFlagsAtOnce * kFlagInts * sizeof(int), how));
    std::fill(p, p + kFlagsAtOnce * kFlagInts, 0);
    for (int i = 0; i < kFlagsAtOnce; ++i) g_free.push_back(p + i * kFlagInts);
  }
  int* flags = g_free.back();
  g_free.pop_back();
  return flags;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

int tb200_flags_take(int** flags) {
  return guarded([&] {
    check(flags != nullptr, "null pointer");
    *flags = take_flags();
  });
}

int tb200_flags_wait(int* flags, int* values) {
  return guarded([&] {
    check(flags && values, "null pointer");
    TB200_CUDA_CHECK(cudaStreamSynchronize(api_stream()));   // (where this fails the flags are not used again)
    for (int i = 0; i < 2; ++i) {
      values[i] = *static_cast<volatile int*>(flags + i);
      flags[i] = 0;
    }
    std::lock_guard<std::mutex> lock(g_flags);
    g_free.push_back(flags);
  });
}

int tb200_reorder_states(const tb200_states* states, int count, const int* parents, int B, int N, int W, int kept,
                         int* beyond) {
  return guarded([&] {
    check(count >= 0 && B >= 0 && N >= 0 && W >= 0, "negative number of states, utterances or hypotheses");
    check((long long)B * N < 0x7fffffffLL && (long long)B * W < 0x7fffffffLL,
          "too many hypotheses (batchSize * hypotheses must be below 2^31 - 1)");
    check(count == 0 || states, "null pointer");
    static_assert(sizeof(States) == sizeof(tb200_states));
    for (int i = 0; i < count; ++i) {
      const tb200_states& s = states[i];
      check(s.rowBytes >= 0 && s.fromStrideB >= 0 && s.fromStrideN >= 0 && s.toStrideB >= 0 && s.toStrideN >= 0,
            "negative size or stride");
      check(s.rowBytes <= 1ll << 40, "the states are too large");
      if (s.from == s.to && s.from) {
        check((B <= 1 || s.fromStrideB == s.toStrideB) && (std::min(N, W) <= 1 || s.fromStrideN == s.toStrideN),
              "states that are reordered in place must keep their strides");
        check(W <= kMaxReorderedWidth, "at most 4096 hypotheses are reordered in place");
      }
    }
    launch_reorder_states(reinterpret_cast<const States*>(states), count, parents, B, N, W, kept != 0, beyond,
                          api_stream());
  });
}

int tb200_embed_words(const void* table, int bf16, long long stride, const int* words, long long count, void* rows,
                      int R, int H, double scale, double dropout, long long seed, const long long* seedAt,
                      int* beyond) {
  return guarded([&] {
    launch_embed_words(embed_args(table, bf16, stride, words, count, R, H, scale, dropout, seed, seedAt), rows, beyond,
                       api_stream());
  });
}

size_t tb200_embed_backward_workspace_bytes(long long count, int R, int H) {
  return embed_backward_workspace_bytes(count, R, H);
}

int tb200_embed_backward(const void* deltas, int bf16, const int* words, long long count, void* grad, int R, int H,
                         double scale, double dropout, long long seed, const long long* seedAt, void* workspace,
                         size_t workspaceBytes) {
  return guarded([&] {
    const EmbedArgs a = embed_args(nullptr, bf16, H, words, count, R, H, scale, dropout, seed, seedAt);
    need(workspaceBytes, embed_backward_workspace_bytes(count, R, H), workspace, "workspace");
    launch_embed_backward(a, deltas, grad, workspace, api_stream());
  });
}

}  // extern "C"
