// The best words of a lattice node, and a word drawn from a node's distribution.
#include <algorithm>

#include "node_rows.cuh"
#include "profile.h"

namespace tb200 {
namespace {

// The words of one row as a group of G threads sees them: EPT of them in each thread's registers, or
// (EPT = 0, rows that no group can hold) read again for every pass.
template <typename TIn, int VEC, int G, int EPT>
struct Row {
  NodeScores<TIn> s;
  int V, tid;
  float z[EPT > 0 ? EPT : 1];

  __device__ __forceinline__ Row(const NodeScores<TIn>& scores, int V_, int tid_) : s(scores), V(V_), tid(tid_) {
    if constexpr (EPT > 0) {
#pragma unroll
      for (int j = 0; j < EPT / VEC; ++j) {
        const int v = (j * G + tid) * VEC;
        if (v < V) {
          const Words<VEC> e = load_words<VEC>(s.e + v), p = load_words<VEC>(s.p + v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) z[j * VEC + i] = e.x[i] + p.x[i];
        }
      }
    }
  }
  // f(score, word) for each of this thread's words
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (EPT > 0) {
#pragma unroll
      for (int j = 0; j < EPT / VEC; ++j) {
        const int v = (j * G + tid) * VEC;
        if (v < V)
#pragma unroll
          for (int i = 0; i < VEC; ++i) f(z[j * VEC + i], v + i);
      }
    } else {
      for (int v = tid * VEC; v < V; v += G * VEC) {
        const Words<VEC> e = load_words<VEC>(s.e + v), p = load_words<VEC>(s.p + v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f(e.x[i] + p.x[i], v + i);
      }
    }
  }
};

// Words are ordered by score, the greater first, equal ones by index, the lower first.  A cut is a
// prefix of that order: the words above `key`, and those at `key` up to `last`.
struct Cut {
  unsigned key;
  int last;
  __device__ __forceinline__ bool keeps(unsigned k, int v) const { return k > key || (k == key && v <= last); }
};

// The largest key x for which reaches(x) holds (a property that holds for 0 and for fewer and fewer
// words from there on): one pass over the row per bit.
template <typename F>
__device__ __forceinline__ unsigned largest_key(F reaches) {
  unsigned x = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned t = x | (1u << bit);
    if (reaches(t)) x = t;
  }
  return x;
}
// The smallest index y in [0, V) for which reaches(y) holds, V - 1 if it never does.
template <typename F>
__device__ __forceinline__ int smallest_index(int V, F reaches) {
  int lo = 0, hi = V - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (reaches(mid)) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The k first words of the order (0 < k <= V).
template <typename R, typename Gr>
__device__ __forceinline__ Cut first_k(const R& row, Gr& g, int k) {
  auto count = [&](auto pick) {
    int c = 0;
    row.each([&](float z, int v) { c += pick(score_key(z), v) ? 1 : 0; });
    return g.sum(c);
  };
  Cut cut;
  cut.key = largest_key([&](unsigned x) { return count([&](unsigned u, int) { return u >= x; }) >= k; });
  const int above = count([&](unsigned u, int) { return u > cut.key; });
  cut.last = smallest_index(row.V, [&](int y) {
    return count([&](unsigned u, int v) { return u == cut.key && v <= y; }) >= k - above;
  });
  return cut;
}

constexpr int kWarpRows = 8;   // rows per CTA where a warp has a row
template <int G>
constexpr int kCta = G == 32 ? 32 * kWarpRows : G;

template <typename TIn, int VEC, int G, int EPT>
__global__ void __launch_bounds__(kCta<G>) top_words_kernel(NodeArgs a, int* __restrict__ words,
                                                            float* __restrict__ logits,
                                                            float* __restrict__ rest, int k, float scale) {
  constexpr int kRows = kCta<G> / G;
  __shared__ double scratch[64];
  __shared__ unsigned long long listAll[kRows][kMaxListedWords];
  __shared__ int filled[kRows];
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kRows + sub;
  if (node >= (i64)a.B * a.N) return;
  unsigned long long* list = listAll[sub];
  words += node * k;
  logits += node * k;
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  if (!s.here) {
    for (int i = tid; i < k; i += G) words[i] = -1, logits[i] = neg_inf();
    if (rest && tid == 0) rest[node] = neg_inf();
    return;
  }
  Group<G> g(tid, scratch);
  const Row<TIn, VEC, G, EPT> row(s, a.V, tid);
  const Cut cut = first_k(row, g, k);
  if (tid == 0) filled[sub] = 0;
  g.sync();
  row.each([&](float z, int v) {
    const unsigned u = score_key(z);
    if (cut.keeps(u, v))
      list[atomicAdd(&filled[sub], 1)] = ((unsigned long long)u << 32) | (0xffffffffu - (unsigned)v);
  });
  g.sync();
  // (the list has the k words in any order: each finds its place)
  for (int i = tid; i < k; i += G) {
    const unsigned long long mine = list[i];
    int place = 0;
    for (int j = 0; j < k; ++j) place += list[j] > mine ? 1 : 0;
    words[place] = (int)(0xffffffffu - (unsigned)mine);
    logits[place] = key_score((unsigned)(mine >> 32)) * scale;
  }
  if (!rest) return;
  float m = neg_inf();
  row.each([&](float z, int v) {
    if (!cut.keeps(score_key(z), v)) m = fmaxf(m, z);
  });
  m = g.max(m);
  float sum = 0.0f;
  if (m > neg_inf())
    row.each([&](float z, int v) {
      if (!cut.keeps(score_key(z), v)) sum += expf((z - m) * scale);
    });
  sum = g.sum(sum);
  if (tid == 0) rest[node] = m > neg_inf() ? m * scale + logf(sum) : neg_inf();
}

template <typename TIn, int VEC, int G, int EPT>
__global__ void __launch_bounds__(kCta<G>) sample_words_kernel(NodeArgs a, const float* __restrict__ uniforms,
                                                               int* __restrict__ words,
                                                               float* __restrict__ logProbs, SampleRule rule) {
  constexpr int kRows = kCta<G> / G;
  __shared__ double scratch[64];
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kRows + sub;
  if (node >= (i64)a.B * a.N) return;
  auto answer = [&](int word, float logProb) {
    if (tid == 0) words[node] = word, logProbs[node] = logProb;
  };
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  if (!s.here) return answer(-1, 0.0f);
  Group<G> g(tid, scratch);
  const Row<TIn, VEC, G, EPT> row(s, a.V, tid);
  unsigned top = 0;
  row.each([&](float z, int) { top = max(top, score_key(z)); });
  top = g.max(top);
  const float m = key_score(top);
  if (!(m < pos_inf())) return answer(-1, __int_as_float(0x7fffffff));   // NaN or +inf among the scores
  if (m == neg_inf()) return answer(-1, neg_inf());                      // every word is masked
  if (rule.temperature == 0.0) {
    const int word = smallest_index(a.V, [&](int y) {
      int c = 0;
      row.each([&](float z, int v) { c |= z == m && v <= y; });
      return g.max(c) > 0;
    });
    return answer(word, 0.0f);
  }
  const double scale = 1.0 / rule.temperature;
  auto weight = [&](float z) { return exp(((double)z - (double)m) * scale); };
  auto mass = [&](auto pick) {
    double c = 0.0;
    row.each([&](float z, int v) {
      if (pick(score_key(z), z, v)) c += weight(z);
    });
    return g.sum(c);
  };
  Cut kept{0u, a.V};
  if (rule.topK > 0 && rule.topK < a.V) kept = first_k(row, g, rule.topK);
  if (rule.topP < 1.0) {
    const Cut all = kept;
    const double share = rule.topP * mass([&](unsigned u, float, int v) { return all.keeps(u, v); });
    // the word that reaches the share: its key, then, among equal ones, its index
    kept.key = largest_key([&](unsigned x) {
      return mass([&](unsigned u, float, int v) { return u >= x && all.keeps(u, v); }) >= share;
    });
    kept.key = max(kept.key, all.key);
    const double above = mass([&](unsigned u, float, int v) { return u > kept.key && all.keeps(u, v); });
    const double one = weight(key_score(kept.key));
    kept.last = smallest_index(a.V, [&](int y) {
      int c = 0;
      row.each([&](float z, int v) { c += score_key(z) == kept.key && v <= y && all.keeps(kept.key, v); });
      c = g.sum(c);
      return c > 0 && above + c * one >= share;
    });
    if (kept.key == all.key) kept.last = min(kept.last, all.last);
  }
  auto keeps = [&](unsigned u, float z, int v) { return kept.keeps(u, v) && weight(z) >= rule.minP; };
  const double total = mass(keeps);
  const float u = uniforms[node];
  const double target = (double)(u < 0.0f ? 0.0f : u) * total;
  int word = smallest_index(a.V, [&](int y) {
    return mass([&](unsigned u, float z, int v) { return v <= y && keeps(u, z, v); }) > target;
  });
  // (numbers of 1 and above, and NaN: the last word that is kept)
  int last = -1;
  row.each([&](float z, int v) {
    if (keeps(score_key(z), z, v) && weight(z) > 0.0) last = max(last, v);
  });
  last = g.max(last);
  word = min(word, last);
  double mine = 0.0;
  row.each([&](float z, int v) {
    if (v == word) mine = weight(z);
  });
  mine = g.sum(mine);
  answer(word, (float)log(mine / total));
}

// Group sizes: a warp for rows of up to 1024 words, larger groups for longer ones, 32 words a thread
// in registers; rows beyond 1024 threads' registers are read again for every pass.
template <typename TIn, int VEC, typename F>
void with_group(int V, F launch) {
  if (V <= 32 * 8) launch(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
  else if (V <= 32 * 32) launch(std::integral_constant<int, 32>{}, std::integral_constant<int, 32>{});
  else if (V <= 128 * 32) launch(std::integral_constant<int, 128>{}, std::integral_constant<int, 32>{});
  else if (V <= 512 * 32) launch(std::integral_constant<int, 512>{}, std::integral_constant<int, 32>{});
  else if (V <= 1024 * 32) launch(std::integral_constant<int, 1024>{}, std::integral_constant<int, 32>{});
  else launch(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
}

template <typename F>
void with_type(const NodeArgs& a, F launch) {
  const bool wide = node_rows_aligned(a);
  if (a.dtype == kDtypeBf16) {
    if (wide) launch(bf16{}, std::integral_constant<int, 8>{});
    else launch(bf16{}, std::integral_constant<int, 1>{});
  } else {
    if (wide) launch(float{}, std::integral_constant<int, 4>{});
    else launch(float{}, std::integral_constant<int, 1>{});
  }
}

}  // namespace

// Whether words can be moved 16 bytes at a time: every row starts on a 16-byte boundary and has whole
// vectors.
bool node_rows_aligned(const NodeArgs& a) {
  const int size = a.dtype == kDtypeBf16 ? 2 : 4;
  const i64 bytes[] = {(i64)reinterpret_cast<uintptr_t>(a.E), (i64)reinterpret_cast<uintptr_t>(a.P),
                       a.eStrideB * size, a.eStrideT * size, a.pStrideB * size, a.pStrideU * size,
                       (i64)a.V * size};
  return std::all_of(std::begin(bytes), std::end(bytes), [](i64 x) { return x % 16 == 0; });
}

void launch_top_words(const NodeArgs& a, int* words, float* logits, float* rest, int k, double temperature,
                      cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (nodes == 0) return;
  with_type(a, [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_group<TIn, vec>(a.V, [&](auto group, auto ept) {
      constexpr int G = group, rows = kCta<G> / G;
      ScopedKernel prof("top_words", stream);
      top_words_kernel<TIn, vec, G, ept><<<(unsigned)div_up64(nodes, rows), kCta<G>, 0, stream>>>(
          a, words, logits, rest, k, (float)(1.0 / temperature));
      TB200_CHECK_LAUNCH();
    });
  });
}

void launch_sample_words(const NodeArgs& a, const float* uniforms, int* words, float* logProbs,
                         SampleRule rule, cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (nodes == 0) return;
  with_type(a, [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_group<TIn, vec>(a.V, [&](auto group, auto ept) {
      constexpr int G = group, rows = kCta<G> / G;
      ScopedKernel prof("sample_words", stream);
      sample_words_kernel<TIn, vec, G, ept><<<(unsigned)div_up64(nodes, rows), kCta<G>, 0, stream>>>(
          a, uniforms, words, logProbs, rule);
      TB200_CHECK_LAUNCH();
    });
  });
}

}  // namespace tb200
