// What node_top.cu (the best words of a lattice node) and node_sample.cu (a word drawn from a node's
// distribution) share.
//
// A row of scores is read once and stays in shared memory, seen by a group of threads (a warp for short rows, a CTA for
// long ones; rows beyond that are read again for every pass).  What both operators then need is a cut in the order
// of the words: the first k of them, or the first whose weights reach a share.  Sorting is never needed for that:
// thresholds on the scores are tried until the few words about the cut can be put in a list, where each finds its
// place by comparing itself with the others.  (In registers rows were no faster to go through, and left room for a
// quarter of the threads.)
#pragma once

#include <type_traits>

#include "node_rows.cuh"

namespace tb200 {

// Which words of a row a thread has: warp w has the words from w * seg on, as far as the next warp's,
// and its lanes take vectors of VEC words in turn.  So the warps' parts follow each other in the order
// of the alphabet, and so do the vectors of a warp.
template <typename TIn, int VEC>
struct Place {
  NodeScores<TIn> s;
  int first, end, lane;   // the warp's words
  __device__ __forceinline__ Place(const NodeScores<TIn>& scores, int V, int seg, int warp, int lane_)
      : s(scores), first(warp * seg), end(min(V, first + seg)), lane(lane_) {}
  __device__ __forceinline__ void load(int v, float (&z)[VEC]) const {
    const Words<VEC> e = load_words<VEC>(s.e + v), p = load_words<VEC>(s.p + v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) z[i] = e.x[i] + p.x[i];
  }
  __device__ __forceinline__ float score(int v) const { return to_f32(s.e[v]) + to_f32(s.p[v]); }
};

// ---- the general way, from memory: one pass over the row per bit searched --------------------
// For rows where the words about a cut are too many for a list (equal scores), and for NaN.  These
// functions have a copy of the group: the caller's next reduction comes after a barrier.

// Words are ordered by score, the greater first, equal ones by index, the lower first.  A cut is a
// prefix of that order: the words above `key`, and those at `key` up to `last`.
struct Cut {
  unsigned key;
  int last;
  __device__ __forceinline__ bool keeps(unsigned k, int v) const { return k > key || (k == key && v <= last); }
  __device__ __forceinline__ bool keeps(float z, int v) const { return keeps(score_key(z), v); }
};

template <typename TIn, int VEC, int G, typename F>
__device__ __forceinline__ void each_score(const NodeScores<TIn>& s, int V, int tid, F f) {
#pragma unroll 1
  for (int v = tid * VEC; v < V; v += G * VEC) {
    const Words<VEC> e = load_words<VEC>(s.e + v), p = load_words<VEC>(s.p + v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f(e.x[i] + p.x[i], v + i);
  }
}

// The largest key x for which reaches(x) holds (a property that holds for 0 and for fewer and fewer
// words from there on).
template <typename F>
__device__ __forceinline__ unsigned largest_key(F reaches) {
  unsigned x = 0;
#pragma unroll 1
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
#pragma unroll 1
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (reaches(mid)) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The k first words of the order (0 < k <= V).  `key`: of the k-th, if it is known.
template <typename TIn, int VEC, int G>
__device__ __noinline__ Cut general_first_k(NodeScores<TIn> s, int V, Group<G> g, int k, unsigned key = 0) {
  auto count = [&](auto pick) {
    int c = 0;
    each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) { c += pick(score_key(z), v) ? 1 : 0; });
    return g.sum(c);
  };
  Cut cut;
  cut.key = key ? key
                : largest_key([&](unsigned x) { return count([&](unsigned u, int) { return u >= x; }) >= k; });
  const int above = count([&](unsigned u, int) { return u > cut.key; });
  cut.last = smallest_index(V, [&](int y) {
    return count([&](unsigned u, int v) { return u == cut.key && v <= y; }) >= k - above;
  });
  return cut;
}

// ---- groups and lists -------------------------------------------------------------------------

constexpr int kWarpRows = 8;   // rows per CTA where a warp has a row
template <int G>
constexpr int kCta = G == 32 ? 32 * kWarpRows : G;

using Entry = unsigned long long;   // a word and its score: greater for words that come first
__device__ __forceinline__ Entry entry_of(float z, int v) {
  return ((Entry)score_key(z) << 32) | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ int entry_word(Entry e) { return (int)(0xffffffffu - (unsigned)e); }
__device__ __forceinline__ unsigned entry_key(Entry e) { return (unsigned)(e >> 32); }

// How many of the c entries of `list` come before `mine`.
__device__ __forceinline__ int entries_before(const Entry* list, int c, Entry mine) {
  int n = 0;
#pragma unroll 4
  for (int j = 0; j < c; ++j) n += list[j] > mine ? 1 : 0;
  return n;
}

// ---- rows in shared memory ---------------------------------------------------------------------

// A row's scores, fp32, in shared memory: warp w has seg words from w * seg on, and of these each lane seg / 32 that
// follow each other, so that the lanes' words are in the order of the alphabet.  seg is 128 times an odd number: lanes
// that read four of their words at a time then read from different banks.
constexpr int kResidentBytes = 220 * 1024;   // for a row, beside the lists
inline int words_of_warp(int V, int warps) { return 128 * (div_up(V, 128 * warps) | 1); }

// The warp's scores from memory to `w` (words beyond the row: -inf); f(scores) for each vector as it comes by.  Without
// RESIDENT only the latter.
template <bool RESIDENT, typename TIn, int VEC, typename F>
__device__ __forceinline__ void bring_row(const Place<TIn, VEC>& at, float* w, int seg, F f) {
  constexpr int kBatch = VEC == 1 ? 8 : VEC == 8 ? 3 : 4;   // vectors on their way at a time (more: spilled registers)
  const int words = at.end - at.first, whole = RESIDENT ? seg : words;
  for (int o = at.lane * VEC; o < whole; o += 32 * VEC * kBatch) {
    RawWords<TIn, VEC> e[kBatch], p[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int v = o + 32 * VEC * j;
      if (v < words) e[j].load(at.s.e + at.first + v), p[j].load(at.s.p + at.first + v);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int v = o + 32 * VEC * j;
      float x[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = neg_inf();
      if (v < words) {
        const Words<VEC> y = e[j].words(), z = p[j].words();
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = y.x[i] + z.x[i];
        f(x);
      }
      if constexpr (RESIDENT) {
        if (v < whole) {
          if constexpr (VEC % 4 == 0) {
#pragma unroll
            for (int i = 0; i < VEC; i += 4)
              *reinterpret_cast<float4*>(w + v + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          } else {
            w[v] = x[0];
          }
        }
      }
    }
  }
  __syncwarp();
}

// ---- launches ---------------------------------------------------------------------------------

// launch(group, resident): group sizes for rows of V words.  A warp has up to 1024, a CTA of 128 or 256 threads 32 to
// 64 words a thread; rows beyond shared memory are read again for every pass.
template <typename F>
void with_group(int V, bool warps, F launch) {
  using std::integral_constant;
  if (V <= 1024 && warps) launch(integral_constant<int, 32>{}, std::true_type{});
  else if (V <= 4096) launch(integral_constant<int, 128>{}, std::true_type{});
  else if (V <= 16384) launch(integral_constant<int, 256>{}, std::true_type{});
  else if (words_of_warp(V, 32) * 32 * 4 <= kResidentBytes) launch(integral_constant<int, 1024>{}, std::true_type{});
  else launch(integral_constant<int, 1024>{}, std::false_type{});
}

}  // namespace tb200
