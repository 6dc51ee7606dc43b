// The best extensions of an utterance's hypotheses: a beam search's step.
//
// Hypothesis n of utterance b is at a lattice node; word v extends it to d(n, v) = scores[n] + z_v - log sum_w exp z_w.
// The rows are read once, by as many warps as fill the chip, which leave the greatest score and the sum of exponentials
// of every tile of 1024 words, and the greatest score of every chunk of 32 of them (one lane's).  What W extensions
// can be is then narrowed by those: W maxima that reach a threshold are W words that do, so only tiles, then
// chunks, whose maximum reaches it are looked at again, and of the words of these few chunks (read a second time)
// those that reach it are ranked by comparing them with each other.
//
// Large steps are bound by HBM (64 x 32 hypotheses, 32000 words, fp32: 256 MB, 39 us at the measured copy rate; the scan takes
// 45, the call 60), small ones by latency: the scan takes 3 to 4 us, picking 6 (4 x 8 hypotheses of 1025 words: 12 us).
#include <algorithm>

#include "node_select.cuh"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kTile = 1024, kChunk = 32;
constexpr int kScanWarps = 4;

// What the logarithm of a row's sum S = sum exp(z - m) is off by at most: exponents z - m times log2(e) are rounded three
// times, which is 3 * 2^-24 |z - m|, under the softmax on average at most 3 * 2^-24 (ln V - ln S) (its entropy is at most
// ln V); ex2.approx twice 2^-22; 23 additions and products one after the other 2^-24 each.
constexpr float kSumError = 1.9e-6f, kExponentError = 1.8e-7f;

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

// A warp goes through one tile of the rows of up to 32 hypotheses that follow each other, frame by frame, so that a
// frame's words stay in registers.  The rows of the hypotheses come through a ring in shared memory, as 16-byte vectors:
// where rows begin anywhere, as the aligned vectors that hold the tile's words.  Bound by HBM; 16 warps an SM without a ring,
// the next row in registers, took 67 us where this takes 58 (events around 64 x 32 rows of 32000 words), a ring of three rows
// with fewer warps 62.  fp32 rows of 31999 words take as long as those of 32000, bf16 ones 52 us instead of 32: half a word
// of shared memory per load.  bf16 rows of 32000 words take 46 us a call where their bytes take 18: the scan executes 11.7
// instructions per 32 words in fp32, by its code no fewer in bf16, 21 us of the issue slots at best.  Of the aligned vectors up to
// 15 bytes in front of and behind a row are read with it, also where those are another tensor's; they are not used.
constexpr int kScanStages = 2;
template <typename TIn, int VEC>
constexpr int kStageBytes = kTile * (int)sizeof(TIn) + (VEC == 1 ? 16 : 0);

template <typename TIn, int VEC>
__global__ void __launch_bounds__(32 * kScanWarps) extend_scan_kernel(NodeArgs a, const float* __restrict__ scores,
                                                                      int tiles, int perWarp, int groups,
                                                                      ExtendScratch out) {
  constexpr int J = kChunk / VEC;
  using Raw = RawWords<TIn, VEC>;
  extern __shared__ __align__(16) char shared[];
  __shared__ unsigned char order[kScanWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cudaTriggerProgrammaticLaunchCompletion();
  // (x: tiles, groups of hypotheses; y, z: utterances)
  const unsigned id = blockIdx.x * kScanWarps + warp;
  const int tile = id % (unsigned)tiles, group = id / (unsigned)tiles;
  const i64 b = (i64)blockIdx.z * gridDim.y + blockIdx.y;
  if (group >= groups || b >= a.B) return;
  const int first = group * perWarp, count = min(perWarp, a.N - first);
  int frame = -1, position = -1;
  if (lane < count) {
    const i64 node = b * a.N + first + lane;
    frame = a.frames[node], position = a.positions[node];
    if ((unsigned)frame >= (unsigned)a.T || (unsigned)position >= (unsigned)a.U || scores[node] == neg_inf())
      frame = -1;
  }
  // hypotheses in the order of their frames
  const int live = __popc(__ballot_sync(0xffffffffu, frame >= 0));
  int place = 0;
  for (int i = 0; i < count; ++i) {
    const int t = __shfl_sync(0xffffffffu, frame, i);
    place += t >= 0 && (t < frame || (t == frame && i < lane)) ? 1 : 0;
  }
  if (frame >= 0) order[warp][place] = lane;
  __syncwarp();
  const TIn* const E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
  const TIn* const P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
  const int at = chunk_word<VEC>(tile, lane, 0);
  constexpr int kStage = kStageBytes<TIn, VEC>;
  char* const ring = shared + warp * kScanStages * kStage;
  // the i-th hypothesis' row, to the ring
  auto row_of = [&](int i) { return P + __shfl_sync(0xffffffffu, position, order[warp][i]) * a.pStrideU; };
  auto send = [&](int i) {
    if (i < live) {
      const TIn* row = row_of(i);
      if constexpr (VEC > 1) {   // (every lane what it reads itself)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (at + 32 * VEC * j < a.V)
            copy_async<16>(ring + i % kScanStages * kStage + (32 * j + lane) * 16, row + at + 32 * VEC * j);
      } else {
        const uintptr_t from = reinterpret_cast<uintptr_t>(row + tile * kTile), begin = from & ~(uintptr_t)15;
        const uintptr_t end = from + min(kTile, a.V - tile * kTile) * sizeof(TIn);
        for (int j = lane; begin + 16 * j < end; j += 32)
          copy_async<16>(ring + i % kScanStages * kStage + 16 * j, reinterpret_cast<const char*>(begin + 16 * j));
      }
    }
    commit_copies();
  };
  if (live == 0) return;
#pragma unroll
  for (int i = 0; i < kScanStages - 1; ++i) send(i);
  Raw e[J];
  int held = -1;
#pragma unroll 1
  for (int i = 0; i < live; ++i) {
    const int n = order[warp][i], t = __shfl_sync(0xffffffffu, frame, n);
    if (t != held) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (at + 32 * VEC * j < a.V) e[j].load(E + t * a.eStrideT + at + 32 * VEC * j);
      held = t;
    }
    Raw p[J];
    if constexpr (VEC == 1) __syncwarp();   // (all have read what the next row takes the place of)
    send(i + kScanStages - 1);
    wait_copies<kScanStages - 1>();
    const char* stage = ring + i % kScanStages * kStage;
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < J; ++j) p[j].load(reinterpret_cast<const TIn*>(stage + (32 * j + lane) * 16));
    } else {
      __syncwarp();
      const TIn* words = reinterpret_cast<const TIn*>(stage + (reinterpret_cast<uintptr_t>(row_of(i) + tile * kTile) & 15));
#pragma unroll
      for (int j = 0; j < J; ++j) p[j].load(words + 32 * j + lane);   // (beyond the row: anything)
    }
    float z[kChunk];
    float top = neg_inf();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const Words<VEC> x = e[j].words(), y = p[j].words();
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        z[VEC * j + k] = at + 32 * VEC * j < a.V ? x.x[k] + y.x[k] : neg_inf();
        top = fmaxf(top, z[VEC * j + k]);
      }
    }
    const float most = warp_greatest(top);
    const float ref = most == neg_inf() ? 0.0f : most;   // (+inf and NaN: the sum is NaN)
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kChunk; ++k) sum[k % 4] += ex2((z[k] - ref) * 1.4426950408889634f);
    const float all = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    const i64 row = (b * a.N + first + n) * tiles + tile;
    out.best[row * 32 + lane] = top;
    if (lane == 0) out.sums[row] = make_float2(most, all);
  }
}

// ---- what is picked of them ---------------------------------------------------------------------
// A CTA per utterance: of kSmall threads where up to 64 extensions are wanted of so many rows and tiles as shared memory
// holds, else of kLarge, whose own maxima tell 256 extensions, and which read what is not held from memory again.  It is a
// chain of loads and barriers: with 512 threads small steps take 14.5 us instead of 12.4, 64 x 32 hypotheses of 32000 words
// the same.

constexpr int kRowsHeld = 256, kTilesHeld = 4096;
constexpr int kSmall = 256, kLarge = 1024;   // threads
constexpr int kRoots = 32;   // of 2, for exp64
inline bool all_held(int W, i64 N, i64 tiles) { return W <= 64 && N <= kRowsHeld && N * tiles + N <= kTilesHeld; }
enum Kind : unsigned char { kNotThere, kFinished, kExtended };

// An extension's parent and word: of equal extensions the lower one comes first.
using Place = unsigned long long;
__device__ __forceinline__ Place place_of(int parent, int word) { return (Place)parent << 32 | (unsigned)(word + 1); }
__device__ __forceinline__ int parent_of(Place x) { return (int)(x >> 32); }
__device__ __forceinline__ int word_of(Place x) { return (int)(unsigned)x - 1; }

// A tile that is looked at again: its hypothesis, which tile of its row (-1: the hypothesis is finished, its score is row.y),
// its row (see ExtendScratch), and where the rows of the frame and of the position begin.
struct ListedTile {
  int n, tile;
  double2 row;
  i64 e, p;
};

template <int T>
struct PickRoom {
  static constexpr int kTiles = T == kSmall ? 128 : 384;       // listed; where there are more: general_pick
  static constexpr int kChunks = 4096;
  static constexpr int kWords = T == kSmall ? 4096 : 9216;
  double2 row[kRowsHeld];
  i64 e[kRowsHeld], p[kRowsHeld];   // where the rows begin
  union {
    unsigned chunkKey[kTiles * 32];
    struct {   // extensions that may be among the best
      double d[kWords];
      Place place[kWords];
    };
  };
  double2 scratch[64];
  ListedTile tile[kTiles];
  unsigned key[T];
  union {
    float top[kTilesHeld];          // of tiles
    unsigned tileKey[kTilesHeld];   // of their greatest extensions
  };
  union {
    int chunk[kChunks];
    float z[kChunks];   // exact_row: words that are added up next
  };
  float score[kRowsHeld];
  int count[4];
  unsigned reached;
  int close;
  unsigned spread;   // the greatest ln V - ln S of the rows
  double root[kRoots];   // kRoot
  double cutValue;   // general_pick: extensions that come before this one may be among the best
  Place cutPlace;
  Kind kind[kRowsHeld];
  unsigned char again[kWords];
};

// A key that `W` of the threads' keys reach (0: none), the W-th of them or a little less; 0 if there are fewer.
template <int T>
__device__ __forceinline__ unsigned reached_by(unsigned mine, int W, PickRoom<T>& r, Group<T>& g) {
  if constexpr (T == kSmall) {   // (by one warp: no barriers in between)
    r.key[g.tid] = mine;
    if (__syncthreads_count(mine != 0) < W) return 0;
    if (g.warp == 0) {
      constexpr int kKeys = T / 32;
      unsigned k[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; ++i) k[i] = r.key[32 * i + g.lane];
      unsigned least = ~0u, most = 0;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) least = min(least, k[i] ? k[i] : ~0u), most = max(most, k[i]);
      unsigned from = __reduce_min_sync(0xffffffffu, least), to = __reduce_max_sync(0xffffffffu, most) + 1;
      int reached = T;
#pragma unroll 1
      while (to - from > 1 && reached > W + W / 8) {
        const unsigned mid = from + (to - from) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < kKeys; ++i) c += k[i] >= mid ? 1 : 0;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= W) from = mid, reached = c;
        else to = mid;
      }
      if (g.lane == 0) r.reached = from;
    }
    __syncthreads();
    return r.reached;
  } else {
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
}

// The key from which on words are looked at, given one that W of them reach: as much lower as two rows' errors and the
// rounding of the keys' values to 32 bits may come to.
__device__ __forceinline__ unsigned with_slack(unsigned key, float error) {
  const unsigned lowest = score_key(neg_inf()) + 1;
  if (key <= lowest) return lowest;
  const float x = fminf(key_score(key), 3.4028234e38f);
  return max(lowest, score_key(x - (2.5f * error + fabsf(x) * 3e-7f)));
}

// The key of an extension's score; above 0 for all that are extensions.
__device__ __forceinline__ unsigned extension_key(double d) {
  const unsigned lowest = score_key(neg_inf());
  return d > -1.0 / 0.0 ? max(score_key((float)d), lowest + 1) : 0u;
}

// exp(z - m) for z <= m in 64 bits, 2^(n + j/32) times the Taylor series of exp(r), |r| <= log(2) / 64, whose seventh power
// weighs less than 2^-57 (P. T. P. Tang: Table-driven implementation of the exponential function in IEEE floating-point
// arithmetic, 1989).  Below exp(-100) it is that: next to the row's greatest weight, 1, nothing.
__device__ const double kRoot[kRoots] = {   // 2^(j/32)
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};
__device__ __forceinline__ double exp64(const double* roots, float z, float m) {
  const float about = fmaxf(z - m, -100.0f);
  const double x = fmax((double)z - (double)m, -100.0);
  const float shifted = fmaf(about, 46.166241f, 12582912.0f);   // 32 / log(2); 3 * 2^22: the sum is rounded to a whole number
  const int n = __float_as_int(shifted) - __float_as_int(12582912.0f);
  const double k = (double)(shifted - 12582912.0f);
  constexpr double high = 0x1.62e42fefa39efp-6, low = 0x1.abc9e3b39803fp-61;   // log(2) / 32
  const double r = fma(k, -low, fma(k, -high, x)), r2 = r * r;
  const double p = fma(fma(fma(r, 1.0 / 720, 1.0 / 120), r2, fma(r, 1.0 / 24, 1.0 / 6)), r2 * r, fma(r2, 1.0 / 2, r));
  const double root = roots[n & (kRoots - 1)], y = fma(root, p, root);
  return __hiloint2double(__double2hiint(y) + (n >> 5 << 20), __double2loint(y));
}

template <typename TIn, int VEC, int T>
struct Utterance {
  const NodeArgs& a;
  const float* scores;   // of the utterance
  const ExtendScratch& s;
  i64 first;   // node
  int tiles;
  PickRoom<T>& room;

  __device__ __forceinline__ i64 all_tiles() const { return (i64)a.N * tiles; }
  // A hypothesis, from memory: what it is, and its rows.
  __device__ __forceinline__ Kind look(int n, float& score, i64& e, i64& p) const {
    const int t = a.frames[first + n], u = a.positions[first + n];
    score = scores[n];
    const bool here = (unsigned)t < (unsigned)a.T && (unsigned)u < (unsigned)a.U;
    e = here ? t * a.eStrideT : 0, p = here ? u * a.pStrideU : 0;
    return score == neg_inf() ? kNotThere : here ? kExtended : kFinished;
  }
  __device__ __forceinline__ void hold(int n) const {
    room.kind[n] = look(n, room.score[n], room.e[n], room.p[n]);
  }
  static __device__ __forceinline__ bool held(int n) { return T == kSmall || n < kRowsHeld; }
  __device__ __forceinline__ Kind kind(int n) const {
    if (held(n)) return room.kind[n];
    float score;
    i64 e, p;
    return look(n, score, e, p);
  }
  __device__ __forceinline__ float score(int n) const { return held(n) ? room.score[n] : scores[n]; }
  __device__ __forceinline__ void begins(int n, i64& e, i64& p) const {
    float score;
    if (held(n)) e = room.e[n], p = room.p[n];
    else look(n, score, e, p);
  }
  __device__ __forceinline__ const TIn* frame_at(i64 e) const {
    return static_cast<const TIn*>(a.E) + blockIdx.x * a.eStrideB + e;
  }
  __device__ __forceinline__ const TIn* position_at(i64 p) const {
    return static_cast<const TIn*>(a.P) + blockIdx.x * a.pStrideB + p;
  }
  __device__ __forceinline__ NodeScores<TIn> rows(int n) const {
    i64 e, p;
    begins(n, e, p);
    return {frame_at(e), position_at(p), 0, 0, true};
  }
  // Its greatest score m and score - log sum exp(z - m); the latter -inf if it has no words.
  __device__ __forceinline__ double2 row(int n) const { return held(n) ? room.row[n] : s.row[first + n]; }
  __device__ __forceinline__ void set_row(int n, double2 x) const {
    if (held(n)) room.row[n] = x;
    else s.row[first + n] = x;
  }
  // An extension's score: z - m loses nothing, however large the two are.
  static __device__ __forceinline__ double value(double2 row, float z) { return row.y + ((double)z - row.x); }
  __device__ __forceinline__ float tile_top(i64 t) const {
    return T == kSmall || t < kTilesHeld ? room.top[t] : s.sums[first * tiles + t].x;
  }
  // the key of a tile's greatest extension; tiles from all_tiles() on: hypotheses that are finished
  __device__ __forceinline__ unsigned tile_key(i64 t) const {
    if (t >= all_tiles()) {
      const int n = (int)(t - all_tiles());
      return kind(n) == kFinished ? extension_key(score(n)) : 0u;
    }
    const int n = tiles == 1 ? (int)t : (int)((unsigned)t / (unsigned)tiles);
    const double2 x = row(n);
    return x.y > -1.0 / 0.0 ? extension_key(value(x, tile_top(t))) : 0u;
  }
  __device__ __forceinline__ ListedTile listed(i64 t) const {
    ListedTile x;
    if (t >= all_tiles()) {
      x.n = (int)(t - all_tiles()), x.tile = -1;
      x.row = make_double2(0.0, score(x.n));
      x.e = x.p = 0;
    } else {
      x.n = (int)((unsigned)t / (unsigned)tiles), x.tile = (int)((unsigned)t % (unsigned)tiles);
      x.row = row(x.n);
      begins(x.n, x.e, x.p);
    }
    return x;
  }

  // Its sum in 64 bits, by the CTA.  (Little code: where it is needed it has to be brought first.)  One CTA's loads and sums, 1
  // word a cycle: 32000 words take 17 us.  Of 240 inputs of 64 x 32 hypotheses of N(0, 1.5) scores a tenth needs two rows' (60 ->
  // 98 us).  Exponentials in two 32-bit terms, and 64 bits only where those are too close as well, took 13 us a row and
  // 97 a call; clusters of four CTAs that share a row 12 us more in every call.
  __device__ __noinline__ double2 exact_row(int n, Group<T>& g) const {
    constexpr int kWords = PickRoom<T>::kChunks / T, kBatch = kWords > VEC ? kWords / VEC : 1;   // of a thread at a time
    static_assert(VEC <= kWords || T == kLarge);
    const NodeScores<TIn> r = rows(n);
    const float m = (float)row(n).x;
    double part[4] = {0.0, 0.0, 0.0, 0.0};
    if (g.tid < kRoots) room.root[g.tid] = kRoot[g.tid];
    __syncthreads();
    constexpr int kStep = VEC < kWords ? VEC : kWords;   // words of a vector that are added at once
    RawWords<TIn, VEC> x[kBatch], y[kBatch];
    auto bring = [&](int v) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (v + j * T * VEC < a.V) x[j].load(r.e + v + j * T * VEC), y[j].load(r.p + v + j * T * VEC);
    };
    bring(g.tid * VEC);
#pragma unroll 1
    for (int v = g.tid * VEC; v < a.V; v += T * VEC * kBatch) {
      Words<VEC> xs[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const Words<VEC> es = x[j].words(), ps = y[j].words();
#pragma unroll
        for (int i = 0; i < VEC; ++i) xs[j].x[i] = v + j * T * VEC < a.V ? es.x[i] + ps.x[i] : neg_inf();
      }
      bring(v + T * VEC * kBatch);
#pragma unroll
      for (int h = 0; h < VEC / kStep; ++h) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
          for (int i = 0; i < kStep; ++i) room.z[(kStep * j + i) * T + g.tid] = xs[j].x[kStep * h + i];
#pragma unroll 1
        for (int i = 0; i < kBatch * kStep; i += 4)
#pragma unroll
          for (int k = 0; k < 4; ++k) part[k] += exp64(room.root, room.z[(i + k) * T + g.tid], m);
      }
    }
    const double sum = g.sum((part[0] + part[1]) + (part[2] + part[3]));
    return make_double2(m, (double)score(n) - log(sum));
  }
};

// Where equal scores make the lists too long, as in the first steps of an untrained model: all rows' sums in 64 bits, one after
// the other by the utterance's CTA (64 x 64 rows of 10000 words: 700 us), then one way through everything that may be among
// the best, the best W so far in a list that is put in order and cut whenever it is full.  Leaves the list.
template <typename TIn, int VEC, int T>
__device__ __noinline__ int general_pick(const Utterance<TIn, VEC, T>& at, int W, unsigned least, float error, Group<T>& g) {
  constexpr int kRoom = 2 * T;   // of the list
  const NodeArgs& a = at.a;
  PickRoom<T>& p = at.room;
  static_assert(kRoom <= PickRoom<T>::kWords);
  int& count = p.count[2];
  __syncthreads();
  if (g.tid == 0) {
    count = 0;
    p.cutValue = least <= score_key(neg_inf()) + 1 ? -1.0 / 0.0 : (double)key_score(with_slack(least, error));
    p.cutPlace = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int n = 0; n < a.N; ++n) {
    if (at.row(n).y == -1.0 / 0.0) continue;   // (the same for all threads)
    const double2 row = at.exact_row(n, g);
    __syncthreads();
    if (g.tid == 0) at.set_row(n, row);
    __syncthreads();
  }
  auto cut = [&] {   // the first W of the list, in order
    double d[2];
    Place place[2];
    int rank[2];
    const int c = count;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = g.tid + k * T;
      d[k] = i < c ? p.d[i] : 0.0, place[k] = i < c ? p.place[i] : 0, rank[k] = i < c ? 0 : W;
    }
#pragma unroll 4
    for (int j = 0; j < c; ++j) {
      const double other = p.d[j];
      const Place from = p.place[j];
#pragma unroll
      for (int k = 0; k < 2; ++k) rank[k] += (other > d[k]) | ((other == d[k]) & (from < place[k]));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (rank[k] >= W) continue;
      p.d[rank[k]] = d[k], p.place[rank[k]] = place[k];
      if (rank[k] == W - 1) p.cutValue = d[k], p.cutPlace = place[k];
    }
    if (g.tid == 0) count = min(c, W);
    __syncthreads();
  };
  auto better = [&](double d, Place place) {
    return d > p.cutValue || (d == p.cutValue && place < p.cutPlace);
  };
  auto push = [&](bool has, double d, Place place) {   // by all threads; between two of these the cut does not change
    if (has) {
      const int i = atomicAdd(&count, 1);
      p.d[i] = d, p.place[i] = place;
    }
    __syncthreads();
    const int c = count;
    __syncthreads();
    if (c > kRoom - T) cut();
  };
#pragma unroll 1
  for (int n0 = 0; n0 < a.N; n0 += T) {
    const int n = n0 + g.tid;
    const bool has = n < a.N && at.kind(n) == kFinished;
    const double d = has ? (double)at.score(n) : 0.0;
    push(has && better(d, place_of(n, -1)), d, place_of(n, -1));
  }
#pragma unroll 1
  for (i64 t0 = 0; t0 < at.all_tiles(); t0 += T / 32) {   // a warp a tile, a lane a chunk
    const i64 t = t0 + g.warp;
    unsigned left = 0;   // of its words
    double2 row = make_double2(0.0, -1.0 / 0.0);
    NodeScores<TIn> r{};
    int n = 0, tile = 0;
    if (t < at.all_tiles()) {
      n = (int)((unsigned)t / (unsigned)at.tiles), tile = (int)((unsigned)t % (unsigned)at.tiles);
      row = at.row(n);
    }
    auto value = [&](int i) {
      const int v = chunk_word<VEC>(tile, g.lane, i);
      return v < a.V ? at.value(row, to_f32(r.e[v]) + to_f32(r.p[v])) : -1.0 / 0.0;
    };
    auto place = [&](int i) { return place_of(n, chunk_word<VEC>(tile, g.lane, i)); };
    auto counts = [&](int i, double d) { return d > -1.0 / 0.0 && better(d, place(i)); };
    // (the chunk's first word is the first of equals)
    if (row.y > -1.0 / 0.0 && counts(0, at.value(row, at.s.best[(at.first * at.tiles + t) * 32 + g.lane]))) {
      r = at.rows(n);
#pragma unroll 8
      for (int i = 0; i < kChunk; ++i) left |= counts(i, value(i)) ? 1u << i : 0u;
    }
    while (__syncthreads_or(left != 0)) {   // (one word of every lane at a time)
      const int i = __ffs(left) - 1;
      const double d = i >= 0 ? value(i) : 0.0;
      const bool has = i >= 0 && counts(i, d);
      left &= left - 1;
      push(has, d, i >= 0 ? place(i) : 0);
    }
  }
  cut();
  return count;
}

template <typename TIn, int VEC, int T>
__global__ void __launch_bounds__(T) extend_pick_kernel(NodeArgs a, const float* __restrict__ scores,
                                                        float* __restrict__ outScores, int* __restrict__ parents,
                                                        int* __restrict__ words, int W, int tiles, ExtendScratch s,
                                                        int* beyond) {
  constexpr int kWarps = T / 32;
  extern __shared__ __align__(16) char shared[];
  PickRoom<T>& r = *reinterpret_cast<PickRoom<T>*>(shared);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const i64 first = (i64)blockIdx.x * a.N;
  outScores += (i64)blockIdx.x * W;
  parents += (i64)blockIdx.x * W;
  words += (i64)blockIdx.x * W;
  Group<T> g(tid, r.scratch);
  const Utterance<TIn, VEC, T> at{a, scores + first, s, first, tiles, r};
  // (what the scan does not write may be read before it ends)
  for (int n = tid; n < (beyond ? a.N : min(a.N, kRowsHeld)); n += T) {
    if (n < kRowsHeld) at.hold(n);
    if (beyond && scores[first + n] != neg_inf()) {
      if (a.frames[first + n] >= a.T) beyond[0] = 1;
      if (a.positions[first + n] >= a.U) beyond[1] = 1;
    }
  }
  if (tid < 4) r.count[tid] = 0;
  if (tid == 4) r.close = 0, r.spread = 0;
  __syncthreads();
  cudaGridDependencySynchronize();

  // every row's greatest score and sum, a warp each, four rows at a time
  constexpr int kRows = 4;
#pragma unroll 1
  for (int n0 = warp; n0 < a.N; n0 += kRows * kWarps) {
    float2 x[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int n = n0 + k * kWarps;
      x[k] = s.sums[(first + min(n, a.N - 1)) * tiles + min(lane, tiles - 1)];   // (whether or not it was written)
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int n = n0 + k * kWarps;
      if (!(n < a.N && lane < tiles && at.kind(n) == kExtended)) x[k] = make_float2(neg_inf(), 0.0f);
    }
    float m[kRows], sum[kRows];
    // (no word: 0, or NaN where there is one)
    auto weight = [](float2 y, float most) {
      return y.x > neg_inf() ? y.y * ex2((y.x - most) * 1.4426950408889634f) : y.y;
    };
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      m[k] = x[k].x;
      if (tiles > 32) {
        const int n = min(n0 + k * kWarps, a.N - 1);
        const float2* t = s.sums + (first + n) * tiles;
        double all = 0.0;
        if (n == n0 + k * kWarps && at.kind(n) == kExtended) {
          for (int i = lane + 32; i < tiles; i += 32) m[k] = fmaxf(m[k], t[i].x);
          m[k] = warp_greatest(m[k]);
          for (int i = lane; i < tiles; i += 32) {
            all += weight(t[i], m[k]);
            if (T == kSmall || (i64)n * tiles + i < kTilesHeld) r.top[n * tiles + i] = t[i].x;
          }
        }
        sum[k] = (float)all;
      } else {
        m[k] = warp_greatest(m[k]);
        sum[k] = weight(x[k], m[k]);
        const i64 t = (i64)(n0 + k * kWarps) * tiles + lane;
        if (n0 + k * kWarps < a.N && lane < tiles && (T == kSmall || t < kTilesHeld)) r.top[t] = x[k].x;
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      sum[k] = warp_sum(sum[k]);
      if (lane == 0 && n0 + k * kWarps < a.N) at.set_row(n0 + k * kWarps, make_double2(m[k], sum[k]));
    }
  }
  __syncthreads();
  bool bad = false;
#pragma unroll 1
  for (int n = tid; n < a.N; n += T) {
    const Kind kind = at.kind(n);
    double2 row = at.row(n);
    if (kind != kNotThere) bad |= !(at.score(n) < pos_inf());
    if (kind == kExtended) bad |= !(row.y < 1.0 / 0.0);
    const bool extends = kind == kExtended && row.x > -1.0 / 0.0;
    const double log_sum = extends ? log(row.y) : 0.0;
    if (extends) atomicMax(&r.spread, __float_as_uint(fmaxf(0.0f, logf((float)a.V) - (float)log_sum)));
    row.y = extends ? (double)at.score(n) - log_sum : -1.0 / 0.0;
    at.set_row(n, row);
  }
  if (__syncthreads_or(bad)) {
    for (int i = tid; i < W; i += T) outScores[i] = __int_as_float(0x7fffffff), parents[i] = -1, words[i] = -1;
    return;
  }

  // tiles, and the hypotheses that are finished; all of them where they are few
  const i64 rowTiles = at.all_tiles(), allTiles = rowTiles + a.N;
  const float error = kSumError + kExponentError * __uint_as_float(r.spread);
  unsigned least = with_slack(0, error), mine = 0;
  // A key that W of `count` items reach, as they do `from`, and hardly more than W: the threads' own maxima have told one that
  // too many do.
  auto exactly = [&](auto key_of, i64 count, unsigned from) {
    unsigned to = 0;
    for (i64 i = tid; i < count; i += T) to = max(to, key_of(i));
    to = g.max(to) + 1;
    int reached = 0x7fffffff;
#pragma unroll 1
    while (to - from > 1 && reached > W + W / 8) {
      const unsigned mid = from + (to - from) / 2;
      int c = 0;
#pragma unroll 4
      for (i64 i = tid; i < count; i += T) c += key_of(i) >= mid ? 1 : 0;
      c = g.sum(c);
      if (c >= W) from = mid, reached = c;
      else to = mid;
    }
    return from;
  };
  if (allTiles > r.kTiles) {
    auto take = [&](i64 t) {
      const unsigned key = at.tile_key(t);
      if (T == kSmall || t < kTilesHeld) r.tileKey[t] = key;   // (in the place of what it comes from)
      mine = max(mine, key);
    };
    if constexpr (T == kSmall) {   // (t / tiles: fewer than 2^12 tiles, off by less than half of one)
      const float per = 1.0f / (float)tiles;
      for (int t = tid; t < rowTiles; t += T) {
        const double2 row = at.row((int)(((float)t + 0.5f) * per));
        const unsigned key = row.y > -1.0 / 0.0 ? extension_key(at.value(row, r.top[t])) : 0u;
        r.tileKey[t] = key;
        mine = max(mine, key);
      }
      for (i64 t = rowTiles + tid; t < allTiles; t += T) take(t);
    } else {
#pragma unroll 1
      for (i64 t = tid; t < allTiles; t += T) take(t);
    }
    least = with_slack(reached_by<T>(mine, W, r, g), error);
  }
  auto listed_key = [&](i64 t) {
    return allTiles > r.kTiles && (T == kSmall || t < kTilesHeld) ? r.tileKey[t] : at.tile_key(t);
  };
  auto list_tiles = [&] {
#pragma unroll 1
    for (i64 t = tid; t < allTiles; t += T)
      if (listed_key(t) >= least) {
        const int i = atomicAdd(&r.count[0], 1);
        if (i < r.kTiles) r.tile[i] = at.listed(t);
      }
    __syncthreads();
  };
  list_tiles();
  if (r.count[0] > r.kTiles) {
    least = with_slack(exactly(listed_key, allTiles, least), error);
    __syncthreads();
    if (tid == 0) r.count[0] = 0;
    __syncthreads();
    list_tiles();
  }
  bool many = r.count[0] > r.kTiles;

  // their chunks
  if (!many) {
    const int listed = r.count[0];
    mine = 0;
    constexpr int kBatch = 8;
#pragma unroll 1
    for (int i0 = warp; i0 < listed; i0 += kBatch * kWarps) {
      float top[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const ListedTile& t = r.tile[min(i0 + j * kWarps, listed - 1)];
        const i64 place = ((first + t.n) * tiles + max(t.tile, 0)) * 32 + lane;
        top[j] = s.best[place];   // (whether or not it was written)
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kWarps;
        if (i >= listed) break;
        const bool extends = r.tile[i].tile >= 0;
        const unsigned key = extension_key(at.value(r.tile[i].row, extends ? top[j] : lane == 0 ? 0.0f : neg_inf()));
        r.chunkKey[i * 32 + lane] = key;
        mine = max(mine, key);
      }
    }
    least = max(least, with_slack(reached_by<T>(mine, W, r, g), error));
    auto list_chunks = [&] {
#pragma unroll 1
      for (int i = tid; i < 32 * listed; i += T)
        if (r.chunkKey[i] >= least) {
          const int k = atomicAdd(&r.count[1], 1);
          if (k < r.kChunks) r.chunk[k] = i;
        }
      __syncthreads();
    };
    list_chunks();
    if (r.count[1] > r.kWords / 32) {   // (more words than there is room for)
      least = max(least, with_slack(exactly([&](i64 i) { return r.chunkKey[i]; }, 32 * listed, least), error));
      __syncthreads();
      if (tid == 0) r.count[1] = 0;
      __syncthreads();
      list_chunks();
    }
    many = r.count[1] > r.kChunks;
  }

  // their words
  int c = 0;
  if (!many) {
    const int chunks = r.count[1];
    constexpr int kBatch = 8;   // chunks on their way at a time
#pragma unroll 1
    for (int k0 = warp; k0 < chunks; k0 += kBatch * kWarps) {
      float z[kBatch];
      TIn e[kBatch], p[kBatch];
      unsigned words = 0;   // bit j: this lane has a word of the j-th chunk
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = min(k0 + j * kWarps, chunks - 1), chunk = r.chunk[k];
        const ListedTile& t = r.tile[chunk >> 5];
        const int v = chunk_word<VEC>(t.tile, chunk & 31, lane);
        const bool in = t.tile >= 0 && v < a.V;
        words |= in ? 1u << j : 0u;
        if (in) e[j] = at.frame_at(t.e)[v];
        if (in) p[j] = at.position_at(t.p)[v];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) z[j] = words >> j & 1 ? to_f32(e[j]) + to_f32(p[j]) : neg_inf();
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = k0 + j * kWarps;
        if (k >= chunks) break;
        const ListedTile& t = r.tile[r.chunk[k] >> 5];
        if (t.tile < 0 && lane == 0) z[j] = 0.0f;
        const double d = at.value(t.row, z[j]);
        if (extension_key(d) < least) continue;
        const int v = t.tile < 0 ? -1 : chunk_word<VEC>(t.tile, r.chunk[k] & 31, lane);
        const int i = atomicAdd(&r.count[2], 1);
        if (i < r.kWords) r.d[i] = d, r.place[i] = place_of(t.n, v);
      }
    }
    __syncthreads();
    c = r.count[2];
    many = c > r.kWords;
  }

  // of many words those that can be among the best
  if (!many && c > 2 * W + 64) {
    mine = 0;
    for (int i = tid; i < c; i += T) mine = max(mine, extension_key(r.d[i]));
    least = with_slack(reached_by<T>(mine, W, r, g), error);
#pragma unroll 1
    for (int i0 = 0; i0 < c; i0 += T) {   // (in place: what is written lies before what is read)
      const int i = i0 + tid;
      const bool in = i < c && extension_key(r.d[i]) >= least;
      const double d = in ? r.d[i] : 0.0;
      const Place place = in ? r.place[i] : 0;
      __syncthreads();
      if (in) {
        const int k = atomicAdd(&r.count[3], 1);
        r.d[k] = d, r.place[k] = place;
      }
      __syncthreads();
    }
    c = r.count[3];
    many = c > 2 * T;   // (to compare each with all others takes as long as the way through the rows)
  }
  const bool exact = many;
  if (many) c = general_pick<TIn, VEC, T>(at, W, least, error, g);

  // where each is in the order, and whether what it rests on is closer than the sums' errors
  for (int i = tid; i < c; i += T) r.again[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    constexpr int kShare = 4;   // threads that look at a quarter of the others each
#pragma unroll 1
    for (int i0 = 0; i0 < c; i0 += T / kShare) {
      const int i = i0 + tid / kShare;
      const double d = r.d[min(i, c - 1)];
      const Place place = r.place[min(i, c - 1)];
      const int parent = parent_of(place);
      int rank = 0;
      bool close = false;
#pragma unroll 4
      for (int j = tid % kShare; j < c; j += kShare) {
        const double other = r.d[j];
        const Place at = r.place[j];
        rank += (other > d) | ((other == d) & (at < place));
        close |= (parent_of(at) != parent) & (fabs(d - other) <= 2.0f * error);
      }
      rank += close ? 1 << 20 : 0;
#pragma unroll
      for (int o = 1; o < kShare; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      close = rank >= 1 << 20;
      rank &= (1 << 20) - 1;
      if (i >= c || tid % kShare != 0) continue;
      if (pass == 0 && !exact && close && rank < W) {
        r.close = r.again[i] = 1;
#pragma unroll 1
        for (int j = 0; j < c; ++j)
          if (parent_of(r.place[j]) != parent && fabs(d - r.d[j]) <= 2.0f * error) r.again[j] = 1;
      }
      if (rank < W) outScores[rank] = (float)d, parents[rank] = parent, words[rank] = word_of(place);
    }
    __syncthreads();
    if (pass > 0 || !r.close) break;
    // 64 bits for the rows in question
#pragma unroll 1
    for (int k = 0; k < c; ++k) {
      if (!r.again[k] || word_of(r.place[k]) < 0) continue;   // (the same for all threads)
      const int n = parent_of(r.place[k]);
      const double2 exactly = at.exact_row(n, g);
      const NodeScores<TIn> rows = at.rows(n);
      __syncthreads();
      for (int i = tid; i < c; i += T)
        if (parent_of(r.place[i]) == n && word_of(r.place[i]) >= 0) {
          const int v = word_of(r.place[i]);
          r.d[i] = at.value(exactly, to_f32(rows.e[v]) + to_f32(rows.p[v]));
          r.again[i] = 0;
        }
      __syncthreads();
    }
  }
  for (int i = c + tid; i < W; i += T) outScores[i] = neg_inf(), parents[i] = -1, words[i] = -1;
}

}  // namespace

size_t extend_workspace_bytes(int B, int V, int N) {
  if (B <= 0 || N <= 0 || V <= 0) return 0;
  const i64 rows = (i64)B * N, tiles = div_up(V, kTile);
  return (size_t)(round_up64(rows * 16, 128) + round_up64(rows * tiles * 8, 128) + rows * tiles * 128);
}

void launch_extend_beams(const NodeArgs& a, const float* scores, float* outScores, int* parents, int* words, int W,
                         int* beyond, void* workspace, cudaStream_t stream) {
  if (a.B == 0) return;
  const int tiles = div_up(a.V, kTile);
  if ((i64)a.N * tiles >= 0x7fff0000LL) throw std::invalid_argument("too many words and hypotheses");
  const ExtendScratch s = scratch_at(workspace, (i64)a.B * a.N, tiles);
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    if (a.N > 0) {
      // hypotheses per warp: as many as leave 64 warps per SM (with 12 the scan of 64 x 32 rows of 32000 words takes 61 us, not 58)
      const i64 most = (i64)a.B * tiles * a.N;
      const int fewest = (int)std::max<i64>(1, std::min<i64>(std::min(a.N, 32), most / (148 * 64)));
      const int groups = div_up(a.N, fewest), perWarp = div_up(a.N, groups);
      const i64 warps = (i64)tiles * groups;
      const int rows = std::min(a.B, 65535), layers = div_up(a.B, rows);
      if (warps > 0x7fff0000LL || layers > 65535) throw std::invalid_argument("too many words and hypotheses");
      ScopedKernel prof("extend_scan", stream);
      auto kernel = extend_scan_kernel<TIn, VEC>;
      constexpr int smem = kScanWarps * kScanStages * kStageBytes<TIn, VEC>;
      if (smem > 40 * 1024) allow_dyn_smem(kernel, smem);
      kernel<<<dim3((unsigned)div_up64(warps, kScanWarps), rows, layers), 32 * kScanWarps, smem, stream>>>(
          a, scores, tiles, perWarp, groups, s);
      TB200_CHECK_LAUNCH();
    }
    auto pick = [&](auto threads) {
      constexpr int T = decltype(threads)::value;
      auto kernel = extend_pick_kernel<TIn, VEC, T>;
      allow_dyn_smem(kernel, sizeof(PickRoom<T>));
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(a.B), config.blockDim = dim3(T);
      config.dynamicSmemBytes = sizeof(PickRoom<T>), config.stream = stream;
      cudaLaunchAttribute early;   // (its launch overlaps the scan; it waits for the scan's end before it reads its results)
      early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      early.val.programmaticStreamSerializationAllowed = a.N > 0;
      config.attrs = &early, config.numAttrs = 1;
      ScopedKernel prof("extend_pick", stream);
      TB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, scores, outScores, parents, words, W, tiles, s, beyond));
    };
    if (all_held(W, a.N, tiles)) pick(std::integral_constant<int, kSmall>{});
    else pick(std::integral_constant<int, kLarge>{});
  });
}

}  // namespace tb200
