// The best extensions of an utterance's hypotheses: a beam search's step.
//
// Hypothesis n of utterance b is at a lattice node; word v extends it to d(n, v) = scores[n] + z_v - log sum_w exp z_w.
// The rows are read once, by as many warps as fill the chip, which leave the greatest score and the sum of exponentials
// of every tile of 1024 words, and the greatest score of every chunk of 32 of them (one lane's).  What W extensions
// can be is then narrowed by those: W maxima that reach a threshold are W words that do, so only tiles, then
// chunks, whose maximum reaches it are looked at again, and of the words of these few chunks (read a second time)
// those that reach it are ranked by comparing them with each other.
#include <algorithm>

#include "node_select.cuh"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kTile = 1024, kChunk = 32;
constexpr int kScanWarps = 4, kPickThreads = 1024, kPickWarps = kPickThreads / 32;
constexpr int kTilesListed = 1024, kChunksListed = 8192, kWordsListed = 8192;

// A row's log-sum-exp is off by 6e-6 at most: exponents (z - m) log2(e) are rounded three times, 3 * 2^-24 |z - m|, whose
// mean under the softmax is ln V < 20 at most; ex2.approx 2^-22; sums of 32 words and 32 lanes 2^-24 (32 + 5).
constexpr float kLseError = 6e-6f;

struct ExtendScratch {
  double2* row;   // [B*N] a row's greatest score m, and scores - log sum exp(z - m); the latter -inf: it has no words
  float2* sums;   // [B*N*tiles] greatest score, sum of exponentials relative to it
  float* best;    // [B*N*tiles*32] greatest score of a chunk
};

ExtendScratch scratch_at(void* p, i64 rows, i64 tiles) {
  ExtendScratch s;
  s.row = static_cast<double2*>(p);
  s.sums = reinterpret_cast<float2*>(static_cast<char*>(p) + round_up64(rows * 16, 128));
  s.best = reinterpret_cast<float*>(reinterpret_cast<char*>(s.sums) + round_up64(rows * tiles * 8, 128));
  return s;
}

// Word i of a lane's chunk in tile `tile`: vectors of VEC words, the lanes' side by side.
template <int VEC>
__device__ __forceinline__ int chunk_word(int tile, int lane, int i) {
  return tile * kTile + i / VEC * (32 * VEC) + lane * VEC + i % VEC;
}

__device__ __forceinline__ float warp_greatest(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// A warp goes through one tile of the rows of up to 32 hypotheses that follow each other; the frame's words stay in
// registers as long as the frame is the same.
template <typename TIn, int VEC>
__global__ void __launch_bounds__(32 * kScanWarps) extend_scan_kernel(NodeArgs a, const float* __restrict__ scores,
                                                                      int tiles, int perWarp, int groups,
                                                                      ExtendScratch out) {
  constexpr int J = kChunk / VEC;
  const int lane = threadIdx.x & 31;
  const i64 id = (i64)blockIdx.x * kScanWarps + (threadIdx.x >> 5);
  const int tile = (int)(id % tiles);
  const i64 rest = id / tiles;
  const i64 b = rest / groups;
  cudaTriggerProgrammaticLaunchCompletion();
  if (b >= a.B) return;
  const int first = (int)(rest % groups) * perWarp, count = min(perWarp, a.N - first);
  int frame = -1, position = -1;
  if (lane < count) {
    const i64 node = b * a.N + first + lane;
    frame = a.frames[node], position = a.positions[node];
    if ((unsigned)frame >= (unsigned)a.T || (unsigned)position >= (unsigned)a.U || scores[node] == neg_inf())
      frame = -1;
  }
  const TIn* const E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
  const TIn* const P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
  const int at = chunk_word<VEC>(tile, lane, 0);
  RawWords<TIn, VEC> e[J], p[J];
  int held = -1;
#pragma unroll 1
  for (int n = 0; n < count; ++n) {
    const int t = __shfl_sync(0xffffffffu, frame, n), u = __shfl_sync(0xffffffffu, position, n);
    if (t < 0) continue;
    if (t != held) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (at + 32 * VEC * j < a.V) e[j].load(E + t * a.eStrideT + at + 32 * VEC * j);
      held = t;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (at + 32 * VEC * j < a.V) p[j].load(P + u * a.pStrideU + at + 32 * VEC * j);
    float z[kChunk];
    float top = neg_inf();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const Words<VEC> x = e[j].words(), y = p[j].words();
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        z[VEC * j + i] = at + 32 * VEC * j < a.V ? x.x[i] + y.x[i] : neg_inf();
        top = fmaxf(top, z[VEC * j + i]);
      }
    }
    const float most = warp_greatest(top);
    const float ref = most == neg_inf() ? 0.0f : most;   // (+inf and NaN: the sum is NaN)
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kChunk; ++i) sum[i % 4] += ex2((z[i] - ref) * 1.4426950408889634f);
    const float all = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    const i64 row = (b * a.N + first + n) * tiles + tile;
    out.best[row * 32 + lane] = top;
    if (lane == 0) out.sums[row] = make_float2(most, all);
  }
}

struct Picked {   // extensions that may be among the best
  double d[kWordsListed];
  int parent[kWordsListed], word[kWordsListed];
  int chunk[kChunksListed];
  i64 tile[kTilesListed];
  double2 scratch[64];
  int count[4], flag, close;
  unsigned char again[kWordsListed];
};

// A key that `W` of the items' greatest reach, and hardly more than W, from the threads' own (0: none); 0 if there are
// fewer.  All threads.
__device__ __forceinline__ unsigned reached_by(unsigned mine, int W, Group<kPickThreads>& g) {
  const int n = __syncthreads_count(mine != 0);
  if (n < W) return 0;
  unsigned from = g.min(mine ? mine : ~0u), to = g.max(mine) + 1;
  int reached = n;
#pragma unroll 1
  while (to - from > 1 && reached > W + W / 8) {
    const unsigned mid = from + (to - from) / 2;
    const int c = __syncthreads_count(mine >= mid);
    if (c >= W) from = mid, reached = c;
    else to = mid;
  }
  return from;
}

// The key from which on words are looked at, given one that W of them reach: as much lower as two rows' errors and the
// rounding of the keys' values to 32 bits may come to.
__device__ __forceinline__ unsigned with_slack(unsigned key) {
  const unsigned lowest = score_key(neg_inf()) + 1;
  if (key <= lowest) return lowest;
  const float x = fminf(key_score(key), 3.4028234e38f);
  return max(lowest, score_key(x - (2.5f * kLseError + fabsf(x) * 3e-7f)));
}

// Order of doubles as of whole numbers.
__device__ __forceinline__ unsigned long long wide_key(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u ^ ((unsigned long long)((long long)u >> 63) | 0x8000000000000000ull);
}

template <typename TIn, int VEC>
struct Utterance {
  const NodeArgs& a;
  const float* scores;
  const ExtendScratch& s;
  i64 first;   // node
  int tiles;

  __device__ __forceinline__ NodeScores<TIn> node(int n) const { return node_scores<TIn>(a, first + n); }
  // a hypothesis that is kept as it is
  __device__ __forceinline__ bool finished(int n) const {
    return scores[first + n] > neg_inf() && !node(n).here;
  }
  __device__ __forceinline__ double2 at_row(int n) const { return s.row[first + n]; }
  __device__ __forceinline__ bool has_words(int n) const { return at_row(n).y != -1.0 / 0.0; }
  // An extension's score: z - m loses nothing, however large the two are.
  static __device__ __forceinline__ double value(double2 row, float z) { return row.y + ((double)z - row.x); }

  // at_row(n), its sum in 64 bits, by the CTA
  __device__ __noinline__ double2 exact_row(int n, Group<kPickThreads>& g) const {
    const NodeScores<TIn> row = node(n);
    float m = neg_inf();
    each_score<TIn, VEC, kPickThreads>(row, a.V, g.tid, [&](float z, int) { m = fmaxf(m, z); });
    m = g.max(m);
    double sum = 0.0;
    if (m > neg_inf())
      each_score<TIn, VEC, kPickThreads>(row, a.V, g.tid, [&](float z, int) { sum += exp((double)z - (double)m); });
    sum = g.sum(sum);
    return make_double2(m, (double)scores[first + n] - log(sum));
  }

  // f(value, parent, word) for every extension of at least `least`, in any order, by the CTA
  template <typename F>
  __device__ __forceinline__ void each(double least, int tid, F f) const {
    const int lane = tid & 31;
    const i64 all = (i64)a.N * tiles;
#pragma unroll 1
    for (i64 t = tid >> 5; t < all; t += kPickWarps) {
      const int n = (int)(t / tiles), tile = (int)(t % tiles);
      const double2 at = at_row(n);
      if (at.y == -1.0 / 0.0) continue;
      const float top = s.best[(first * tiles + t) * 32 + lane];
      if (!(value(at, top) >= least)) continue;
      const NodeScores<TIn> row = node(n);
#pragma unroll 1
      for (int i = 0; i < kChunk; ++i) {
        const int v = chunk_word<VEC>(tile, lane, i);
        if (v >= a.V) break;
        const float z = to_f32(row.e[v]) + to_f32(row.p[v]);
        if (z > neg_inf() && value(at, z) >= least) f(value(at, z), n, v);
      }
    }
#pragma unroll 1
    for (int n = tid; n < a.N; n += kPickThreads)
      if (finished(n) && scores[first + n] >= least) f((double)scores[first + n], n, -1);
  }
};

// Where equal scores make the lists too long: the W-th value by a search over 64-bit keys, a pass over the chunks that reach
// it for each bit, then the place up to which its equals belong to the best.  Leaves the list.
template <typename TIn, int VEC>
__device__ __noinline__ int general_pick(const Utterance<TIn, VEC>& at, int W, Picked& p, Group<kPickThreads>& g) {
  const NodeArgs& a = at.a;
#pragma unroll 1
  for (int n = 0; n < a.N; ++n) {
    if (!at.has_words(n)) continue;   // (the same for all threads)
    const double2 row = at.exact_row(n, g);
    __syncthreads();
    if (g.tid == 0) at.s.row[at.first + n] = row;
    __syncthreads();
  }
  const double lowest = -1.7976931348623157e308;
  auto count = [&](double least, auto pick) {
    int c = 0;
    at.each(least, g.tid, [&](double d, int n, int v) { c += pick(d, n, v) ? 1 : 0; });
    return g.sum(min(c, 1 << 20));
  };
  auto value = [](unsigned long long k) {
    return __longlong_as_double((long long)(k ^ ((unsigned long long)((long long)~k >> 63) | 0x8000000000000000ull)));
  };
  unsigned long long key = 0;
#pragma unroll 1
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long t = key | (1ull << bit);
    if (t <= wide_key(lowest)) {   // (all reach it)
      key = t;
      continue;
    }
    if (t > wide_key(1.7976931348623157e308)) continue;
    if (count(value(t), [&](double d, int, int) { return wide_key(d) >= t; }) >= W) key = t;
  }
  key = max(key, wide_key(lowest));
  const double cut = value(key);
  const int above = count(cut, [&](double d, int, int) { return wide_key(d) > key; });
  // (the place of an extension in the order of equals)
  auto place = [&](int n, int v) { return (i64)n * (a.V + 1ll) + v + 1; };
  i64 lo = 0, hi = (i64)a.N * (a.V + 1ll) - 1;
#pragma unroll 1
  while (lo < hi) {
    const i64 mid = lo + (hi - lo) / 2;
    if (count(cut, [&](double d, int n, int v) { return wide_key(d) == key && place(n, v) <= mid; }) >= W - above)
      hi = mid;
    else lo = mid + 1;
  }
  __syncthreads();
  if (g.tid == 0) p.count[2] = 0;
  __syncthreads();
  at.each(cut, g.tid, [&](double d, int n, int v) {
    if (wide_key(d) == key && place(n, v) > lo) return;
    const int i = atomicAdd(&p.count[2], 1);
    if (i < kWordsListed) p.d[i] = d, p.parent[i] = n, p.word[i] = v;
  });
  __syncthreads();
  return min(p.count[2], W);
}

template <typename TIn, int VEC>
__global__ void __launch_bounds__(kPickThreads) extend_pick_kernel(NodeArgs a, const float* __restrict__ scores,
                                                                   float* __restrict__ outScores,
                                                                   int* __restrict__ parents, int* __restrict__ words,
                                                                   int W, int tiles, ExtendScratch s) {
  extern __shared__ __align__(16) char shared[];
  Picked& p = *reinterpret_cast<Picked*>(shared);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const i64 first = (i64)blockIdx.x * a.N;
  outScores += (i64)blockIdx.x * W;
  parents += (i64)blockIdx.x * W;
  words += (i64)blockIdx.x * W;
  Group<kPickThreads> g(tid, p.scratch);
  const Utterance<TIn, VEC> at{a, scores, s, first, tiles};
  cudaGridDependencySynchronize();

  // log-sum-exp of every row, a warp each
  bool bad = false;
#pragma unroll 1
  for (int n = warp; n < a.N; n += kPickWarps) {
    const float score = scores[first + n];
    double2 row = make_double2(0.0, -1.0 / 0.0);
    if (score != neg_inf()) {
      bad |= !(score < pos_inf());
      if (at.node(n).here) {
        const float2* t = s.sums + (first + n) * tiles;
        float m = neg_inf();
        for (int i = lane; i < tiles; i += 32) m = fmaxf(m, t[i].x);
        m = warp_greatest(m);
        double sum = 0.0;
        for (int i = lane; i < tiles; i += 32) {
          const float2 x = t[i];
          // (no word: 0, or NaN where there is one)
          sum += x.x > neg_inf() ? (double)x.y * exp((double)x.x - (double)m) : (double)x.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        bad |= !(sum < 1.0 / 0.0);
        if (m > neg_inf()) row = make_double2(m, (double)score - log(sum));
      }
    }
    if (lane == 0) s.row[first + n] = row;
  }
  if (tid < 4) p.count[tid] = 0;
  if (tid == 4) p.close = 0;
  if (__syncthreads_or(bad)) {
    for (int i = tid; i < W; i += kPickThreads)
      outScores[i] = __int_as_float(0x7fffffff), parents[i] = -1, words[i] = -1;
    return;
  }

  // tiles: [0, N * tiles), then the hypotheses that are finished
  const i64 rowTiles = (i64)a.N * tiles, allTiles = rowTiles + a.N;
  auto tile_key = [&](i64 t) {
    double d;
    if (t < rowTiles) {
      const double2 row = at.at_row((int)(t / tiles));
      if (row.y == -1.0 / 0.0) return 0u;
      d = at.value(row, s.sums[first * tiles + t].x);
    } else {
      const int n = (int)(t - rowTiles);
      if (!at.finished(n)) return 0u;
      d = scores[first + n];
    }
    const float x = (float)d;
    return x > neg_inf() ? score_key(x) : d > -1.0 / 0.0 ? score_key(neg_inf()) + 1 : 0u;
  };
  unsigned mine = 0;
#pragma unroll 1
  for (i64 t = tid; t < allTiles; t += kPickThreads) mine = max(mine, tile_key(t));
  unsigned least = with_slack(reached_by(mine, W, g));
#pragma unroll 1
  for (i64 t = tid; t < allTiles; t += kPickThreads)
    if (tile_key(t) >= least) {
      const int i = atomicAdd(&p.count[0], 1);
      if (i < kTilesListed) p.tile[i] = t;
    }
  __syncthreads();
  bool many = p.count[0] > kTilesListed;
  const int listed = min(p.count[0], kTilesListed);

  // their chunks
  auto chunk_key = [&](i64 t) {
    if (t >= rowTiles) return lane == 0 ? tile_key(t) : 0u;
    const float top = s.best[(first * tiles + t) * 32 + lane];
    if (top == neg_inf()) return 0u;
    return max(score_key((float)at.value(at.at_row((int)(t / tiles)), top)), score_key(neg_inf()) + 1);
  };
  if (!many) {
    mine = 0;
#pragma unroll 1
    for (int i = warp; i < listed; i += kPickWarps) mine = max(mine, chunk_key(p.tile[i]));
    least = max(least, with_slack(reached_by(mine, W, g)));
#pragma unroll 1
    for (int i = warp; i < listed; i += kPickWarps)
      if (chunk_key(p.tile[i]) >= least) {
        const int k = atomicAdd(&p.count[1], 1);
        if (k < kChunksListed) p.chunk[k] = i * 32 + lane;
      }
    __syncthreads();
    many = p.count[1] > kChunksListed;
  }

  // their words
  int c = 0;
  if (!many) {
    const int chunks = p.count[1];
#pragma unroll 1
    for (int k = warp; k < chunks; k += kPickWarps) {
      const i64 t = p.tile[p.chunk[k] >> 5];
      int n = (int)(t - rowTiles), v = -1;
      double d;
      bool in;
      if (t >= rowTiles) {
        d = scores[first + n];
        in = lane == 0;
      } else {
        n = (int)(t / tiles);
        v = chunk_word<VEC>((int)(t % tiles), p.chunk[k] & 31, lane);
        in = v < a.V;
        const NodeScores<TIn> row = at.node(n);
        const float z = in ? to_f32(row.e[v]) + to_f32(row.p[v]) : neg_inf();
        d = at.value(at.at_row(n), z);
        in = z > neg_inf() && max(score_key((float)d), score_key(neg_inf()) + 1) >= least;
      }
      if (in) {
        const int i = atomicAdd(&p.count[2], 1);
        if (i < kWordsListed) p.d[i] = d, p.parent[i] = n, p.word[i] = v;
      }
    }
    __syncthreads();
    c = p.count[2];
    many = c > kWordsListed;
  }
  const bool exact = many;
  if (many) c = general_pick<TIn, VEC>(at, W, p, g);

  // where each is in the order, and whether what it rests on is closer than the sums' errors
  auto before = [&](int i, int j) {   // extension j comes before i
    if (p.d[j] != p.d[i]) return p.d[j] > p.d[i];
    return p.parent[j] != p.parent[i] ? p.parent[j] < p.parent[i] : p.word[j] < p.word[i];
  };
  for (int i = tid; i < c; i += kPickThreads) p.again[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int pass = 0;; ++pass) {
#pragma unroll 1
    for (int i = tid; i < c; i += kPickThreads) {
      int rank = 0;
      bool close = false;
#pragma unroll 1
      for (int j = 0; j < c; ++j) {
        rank += before(i, j) ? 1 : 0;
        close |= p.parent[i] != p.parent[j] && fabs(p.d[i] - p.d[j]) <= 2.0 * kLseError;
      }
      if (pass == 0 && !exact && close && rank < W) {
        p.close = p.again[i] = 1;
#pragma unroll 1
        for (int j = 0; j < c; ++j)
          if (p.parent[i] != p.parent[j] && fabs(p.d[i] - p.d[j]) <= 2.0 * kLseError) p.again[j] = 1;
      }
      if (rank < W) {
        outScores[rank] = (float)p.d[i];
        parents[rank] = p.parent[i];
        words[rank] = p.word[i];
      }
    }
    __syncthreads();
    if (pass > 0 || !p.close) break;
    // 64 bits for the rows in question
#pragma unroll 1
    for (int n = 0; n < a.N; ++n) {
      bool inQuestion = false;
      for (int i = tid; i < c; i += kPickThreads)
        inQuestion |= p.again[i] && p.parent[i] == n && p.word[i] >= 0;
      if (!__syncthreads_or(inQuestion)) continue;
      const double2 exactly = at.exact_row(n, g);
      const NodeScores<TIn> row = at.node(n);
      for (int i = tid; i < c; i += kPickThreads)
        if (p.parent[i] == n && p.word[i] >= 0) {
          const int v = p.word[i];
          p.d[i] = at.value(exactly, to_f32(row.e[v]) + to_f32(row.p[v]));
        }
      __syncthreads();
    }
  }
  for (int i = c + tid; i < W; i += kPickThreads) outScores[i] = neg_inf(), parents[i] = -1, words[i] = -1;
}

}  // namespace

size_t extend_workspace_bytes(int B, int V, int N) {
  if (B <= 0 || N <= 0 || V <= 0) return 0;
  const i64 rows = (i64)B * N, tiles = div_up(V, kTile);
  return (size_t)(round_up64(rows * 16, 128) + round_up64(rows * tiles * 8, 128) + rows * tiles * 128);
}

void launch_extend_beams(const NodeArgs& a, const float* scores, float* outScores, int* parents, int* words, int W,
                         void* workspace, cudaStream_t stream) {
  if (a.B == 0) return;
  const int tiles = div_up(a.V, kTile);
  const ExtendScratch s = scratch_at(workspace, (i64)a.B * a.N, tiles);
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    if (a.N > 0) {
      // hypotheses per warp: as many as leave 20 warps per SM
      const i64 most = (i64)a.B * tiles * a.N;
      const int perWarp = (int)std::max<i64>(1, std::min<i64>(std::min(a.N, 32), most / (148 * 20)));
      const int groups = div_up(a.N, perWarp);
      const i64 ctas = div_up64((i64)a.B * tiles * groups, kScanWarps);
      if (ctas > 0x7fffffffLL) throw std::invalid_argument("too many words and hypotheses");
      ScopedKernel prof("extend_scan", stream);
      extend_scan_kernel<TIn, VEC><<<(unsigned)ctas, 32 * kScanWarps, 0, stream>>>(a, scores, tiles, perWarp, groups, s);
      TB200_CHECK_LAUNCH();
    }
    auto kernel = extend_pick_kernel<TIn, VEC>;
    allow_dyn_smem(kernel, sizeof(Picked));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(a.B), config.blockDim = dim3(kPickThreads);
    config.dynamicSmemBytes = sizeof(Picked), config.stream = stream;
    cudaLaunchAttribute early;   // (its launch overlaps the scan; it waits for the scan's end before it reads)
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early, config.numAttrs = 1;
    ScopedKernel prof("extend_pick", stream);
    TB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, scores, outScores, parents, words, W, tiles, s));
  });
}

}  // namespace tb200
