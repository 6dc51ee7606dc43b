// The best words of a lattice node.
#include "node_select.cuh"
#include "profile.h"

namespace tb200 {
namespace {

template <typename TIn, int VEC, int G>
__device__ __noinline__ void general_top_words(NodeScores<TIn> s, int V, Group<G> g, Entry* list, int* filled,
                                               int* words, float* logits, float* rest, int k, float scale,
                                               unsigned key) {
  const Cut cut = general_first_k<TIn, VEC, G>(s, V, g, k, key);
  g.sync();
  if (g.tid == 0) *filled = 0;
  g.sync();
  each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
    if (cut.keeps(z, v)) list[atomicAdd(filled, 1)] = entry_of(z, v);
  });
  g.sync();
  for (int i = g.tid; i < k; i += G) {
    const Entry mine = list[i];
    const int place = entries_before(list, k, mine);
    words[place] = entry_word(mine);
    logits[place] = key_score(entry_key(mine)) * scale;
  }
  if (!rest) return;
  float m = neg_inf();
  each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
    if (!cut.keeps(z, v)) m = fmaxf(m, z);
  });
  m = g.max(m);
  float sum = 0.0f;
  if (m > neg_inf() && m < pos_inf())
    each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
      if (!cut.keeps(z, v)) sum += expf((z - m) * scale);
    });
  sum = g.sum(sum);
  if (g.tid == 0) *rest = m > neg_inf() && m < pos_inf() ? m * scale + logf(sum) : m;
}

// The k best words.  Every thread takes the maxima of four subsets of the words that it brings; a threshold that k of
// the G * 4 maxima reach (k of the G threads' maxima where k is small) is one that k words reach, and hardly more
// than k do: 34 of 10000 words for k = 32 and 256 threads.  Three passes over the row in shared memory (maxima as it
// comes, the listing, the others' weights), bound by issue: 14900 nodes of 10000 bf16 words, k = 32, take 242 us (the
// floor of new rows is 46), 21200 of 512 words 50 us, 32 of 1025 words 12, latency.
template <typename TIn, int VEC, int G, bool RESIDENT>
__global__ void __launch_bounds__(kCta<G>, 1024 / kCta<G>) top_words_kernel(NodeArgs a, int* __restrict__ words,
                                                                            float* __restrict__ logits,
                                                                            float* __restrict__ rest, int k, int seg,
                                                                            float scale) {
  constexpr int kRows = kCta<G> / G, kListed = G == 32 ? 256 : 512, kPass = RESIDENT ? 4 : VEC;
  extern __shared__ __align__(16) float scores[];   // a warp's part of a row: seg = 128 * trips words
  __shared__ double2 scratch[64];
  __shared__ Entry listAll[kRows][kListed];
  __shared__ int filledAll[kRows];
  __shared__ Entry edgeAll[kRows][2];   // the last word of the k, and the next one (0: not in the list)
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kRows + sub;
  if (node >= (i64)a.B * a.N) return;
  Entry *list = listAll[sub], *edge = edgeAll[sub];
  int* filled = &filledAll[sub];
  words += node * k;
  logits += node * k;
  if (rest) rest += node;
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  if (!s.here) {
    for (int i = tid; i < k; i += G) words[i] = -1, logits[i] = neg_inf();
    if (rest && tid == 0) *rest = neg_inf();
    return;
  }
  Group<G> g(tid, scratch);
  const Place<TIn, VEC> at(s, a.V, seg, g.warp, g.lane);
  float* const w = scores + sub * seg * Group<G>::kWarps + at.first;   // the warp's words
  const int trips = seg / 128, own = g.lane * 4 * trips;
  // f(scores, first word) for kPass of this thread's words at a time (words beyond the row: -inf)
  auto each = [&](auto f) {
    if constexpr (RESIDENT) {
      const float4* q = reinterpret_cast<const float4*>(w + own);
#pragma unroll 4
      for (int j = 0; j < trips; ++j) {
        const float4 x = q[j];
        const float z[4] = {x.x, x.y, x.z, x.w};
        f(z, at.first + own + 4 * j);
      }
    } else {
#pragma unroll 1
      for (int v = at.first + g.lane * VEC; v < at.end; v += 32 * VEC) {
        float z[VEC];
        at.load(v, z);
        f(z, v);
      }
    }
  };
  float top[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
  bring_row<RESIDENT>(at, w, seg, [&](const float (&x)[VEC]) {
    if constexpr (VEC > 1) {   // (the i-th words of the vectors)
#pragma unroll
      for (int i = 0; i < VEC; ++i) top[i % 4] = fmaxf(top[i % 4], x[i]);
    } else {                   // (every fourth of the words)
      const float oldest = fmaxf(top[3], x[0]);
      top[3] = top[2], top[2] = top[1], top[1] = top[0], top[0] = oldest;
    }
  });
  // (a thread that has brought no words, or fewer than four without vectors, has empty subsets)
  const int mine = max(0, div_up(at.end - at.first - g.lane * VEC, 32 * VEC));
  unsigned key[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) key[q] = score_key(top[q]);
  if (VEC > 1 ? mine == 0 : mine < 4) {
    if constexpr (VEC > 1) {
      key[0] = key[1] = key[2] = key[3] = 0u;
    } else {   // (too few to tell which maxima are of words: all in one)
      key[0] = mine > 0 ? max(max(key[0], key[1]), max(key[2], key[3])) : 0u;
      key[1] = key[2] = key[3] = 0u;
    }
  }
  const unsigned best = max(max(key[0], key[1]), max(key[2], key[3]));
  unsigned lo = 1;   // no threshold
  // The least key of so many that k of them reach, and not many more than k (`reach` counts; all do from `least` on).
  auto threshold = [&](unsigned least, unsigned most, int reached, auto reach) {
    unsigned from = least, to = most + 1;
#pragma unroll 1
    while (to - from > 1 && reached > k + max(k / 8, 4)) {
      const unsigned mid = from + (to - from) / 2;
      const int n = reach(mid);
      if (n >= k) from = mid, reached = n;
      else to = mid;
    }
    return from;
  };
  constexpr int kKeys = G / 32;   // of the threads' maxima in each lane of a warp
  if (G > 32 && G <= 256 && k <= G / 4) {   // by one warp, from the threads' maxima
    unsigned* maxima = reinterpret_cast<unsigned*>(list);
    maxima[tid] = best;
    g.sync();
    if (g.warp == 0) {
      unsigned x[kKeys], least = ~0u, most = 0;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        x[i] = maxima[32 * i + g.lane];
        least = min(least, x[i] ? x[i] : ~0u), most = max(most, x[i]);
        n += x[i] ? 1 : 0;
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= k)
        lo = threshold(__reduce_min_sync(0xffffffffu, least), __reduce_max_sync(0xffffffffu, most), n, [&](unsigned t) {
          int c = 0;
#pragma unroll
          for (int i = 0; i < kKeys; ++i) c += x[i] >= t ? 1 : 0;
          return __reduce_add_sync(0xffffffffu, c);
        });
      if (g.lane == 0) *filled = (int)lo;
    }
    g.sync();
    lo = (unsigned)*filled;
    g.sync();
  } else {
    const bool threads = G > 256 && k <= G / 4;   // (their maxima, too many for one warp)
    auto reach = [&](unsigned t) {
      if (G > 256 && threads) return __syncthreads_count(best >= t);
      return g.sum((key[0] >= t) + (key[1] >= t) + (key[2] >= t) + (key[3] >= t));
    };
    auto least = [](unsigned x) { return x ? x : ~0u; };
    const int n = reach(1);
    const unsigned most = g.max(best);
    if (n >= k)
      lo = threshold(g.min(threads ? least(best)
                                   : min(min(least(key[0]), least(key[1])), min(least(key[2]), least(key[3])))),
                     most, n, reach);
  }
  const unsigned lowest = score_key(neg_inf());
  // The words that reach the threshold: how many there are, and the first kListed to come in the list.
  auto list_words = [&] {
    if (tid == 0) *filled = 0, edge[0] = edge[1] = 0;
    g.sync();
    const float bound = key_score(max(lo, lowest));
    auto append = [&](float x, int v) {
      const int i = atomicAdd(filled, 1);
      if (i < kListed) list[i] = entry_of(x, v);
    };
    each([&](const float (&z)[kPass], int v) {
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < kPass; ++i) in |= z[i] >= bound ? 1u << i : 0u;
#pragma unroll 1
      for (; in; in &= in - 1) {
        const int i = __ffs(in) - 1;
        if (v + i < a.V) append(RESIDENT ? w[v + i - at.first] : at.score(v + i), v + i);
      }
    });
    g.sync();
    return *filled;
  };
  auto general = [&](unsigned key) {
    general_top_words<TIn, VEC, G>(s, a.V, g, list, filled, words, logits, rest, k, scale, key);
  };
  int c = list_words();
  if (RESIDENT && c > min(kListed, k + k / 2 + 64)) {
    auto reach = [&](unsigned t) {   // (NaN counts as the greatest, as the order has it, and is not listed)
      int n = 0;
      each([&](const float (&z)[kPass], int v) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) n += v + i < a.V && score_key(z[i]) >= t ? 1 : 0;
      });
      return g.sum(n);
    };
    lo = max(lo, lowest);
    const int n = reach(lo + 1);
    if (n >= k) {
      lo = threshold(lo + 1, 0xfffffffeu, n, reach);
      c = list_words();
    }
    if (c > kListed) return general(lo);   // (equal scores: lo is the greatest key that k words reach)
  }
  if (c > kListed || c < k) return general(0);   // (fewer than k: some are NaN)
  constexpr int kShare = G >= 128 ? 4 : 1;   // threads per entry, each looking at its part of the others
#pragma unroll 1
  for (int i0 = 0; i0 < c; i0 += G / kShare) {
    const int i = i0 + tid / kShare;
    const Entry mine = i < c ? list[i] : 0;
    int place = 0;
#pragma unroll 4
    for (int j = tid % kShare; j < c; j += kShare) place += list[j] > mine ? 1 : 0;
#pragma unroll
    for (int o = 1; o < kShare; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    if (tid % kShare != 0 || i >= c) continue;
    if (place < k) {
      words[place] = entry_word(mine);
      logits[place] = key_score(entry_key(mine)) * scale;
    }
    if (place == k - 1) edge[0] = mine;
    if (place == k) edge[1] = mine;
  }
  g.sync();
  // the others' weights, relative to the last listed word's; of the words with its score those that are
  // left out are in the list
  const float last = key_score(entry_key(edge[0]));
  int ties = 0;
  if (edge[1] >> 32 == edge[0] >> 32) {
    for (int i = tid; i < c; i += G) ties += list[i] < edge[0] && list[i] >> 32 == edge[0] >> 32 ? 1 : 0;
    ties = g.sum(ties);
  }
  const float scale2 = scale * 1.4426950408889634f;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  each([&](const float (&z)[kPass], int) {
#pragma unroll
    for (int i = 0; i < kPass; ++i)   // (NaN comes through)
      sum[i % 4] += z[i] >= last ? 0.0f : ex2((z[i] - last) * scale2);
  });
  float all = g.sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (all != all) return general(0);
  if (!rest) return;
  all += (float)ties;
  float ref = last;
  if (!(all > 1e-25f)) {   // the others are far below: relative to their own maximum
    ref = neg_inf();
    each([&](const float (&z)[kPass], int) {
#pragma unroll
      for (int i = 0; i < kPass; ++i) ref = z[i] < last ? fmaxf(ref, z[i]) : ref;
    });
    ref = g.max(ref);
    all = 0.0f;
    if (ref > neg_inf())
      each([&](const float (&z)[kPass], int) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) all += z[i] < last ? ex2((z[i] - ref) * scale2) : 0.0f;
      });
    all = g.sum(all);
  }
  if (tid == 0) *rest = fabsf(ref) < pos_inf() ? ref * scale + logf(all) : ref;
}

}  // namespace

void launch_top_words(const NodeArgs& a, int* words, float* logits, float* rest, int k, double temperature,
                      cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (nodes == 0) return;
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    // (a warp's list holds 256 entries, and its 128 maxima tell the best 64 at most)
    with_group(a.V, k <= 64, [&](auto group, auto resident) {
      constexpr int G = decltype(group)::value, rows = kCta<G> / G;
      auto kernel = top_words_kernel<TIn, decltype(vec)::value, G, decltype(resident)::value>;
      const int seg = words_of_warp(a.V, G / 32);
      const int smem = decltype(resident)::value ? rows * seg * (G / 32) * (int)sizeof(float) : 0;
      if (smem > 24 * 1024) allow_dyn_smem(kernel, G == 32 ? 64 * 1024 : kResidentBytes);
      ScopedKernel prof("top_words", stream);
      kernel<<<(unsigned)div_up64(nodes, rows), kCta<G>, smem, stream>>>(a, words, logits, rest, k, seg,
                                                                        (float)(1.0 / temperature));
      TB200_CHECK_LAUNCH();
    });
  });
}

}  // namespace tb200
