// A word drawn from a lattice node's distribution.
//
// Weights are 2^x in 32 bits, x = (z - m) log2(e) / temperature.  They decide where they are sure to:
// the difference from the maximum m is rounded, the factor is, their product is (2^-24 of x each), and
// ex2 is good to 2^-22, so that a weight is off by at most 2^-24 * 2.1 |x| + 2^-22 of itself, and any sum
// of weights by 2^-24 * 2.1 sum w |x| + 2^-22 sum w, both sums over the row (the former is log2 of the number of
// words times the latter at most: the difference of the logarithm of the sum and the entropy).  With twenty roundings
// of the sum itself (a thread has eight sums of up to nine weights, then come eleven steps; the row's whole and the
// draw's sums are of fours in 32 bits and 64 bits from there) that is `unsure` below.  Where a comparison is closer
// than that the sums are formed anew from memory with exponentials in 64 bits.
#include <cfloat>

#include "node_select.cuh"
#include "profile.h"

namespace tb200 {
namespace {

// exp(x) for x <= 0 in 64 bits: 2^n times the Taylor series of exp(f) for |f| <= log(2) / 2, whose twelfth power
// is below 2^-46 of it and whose 13th of 1e-15; down to the least of the 64-bit numbers, by way of 2^(n + 100).  The
// library's own takes about twice the instructions, and a row's 64-bit sums are nothing but these.
__device__ __forceinline__ double exp64(double x) {
  if (!(x > -746.0)) return x != x ? x : 0.0;
  const double n = rint(x * 1.4426950408889634074);
  // log(2) as its 32-bit rounding, n times which is exact, and the rest
  const double f = fma(-n, -1.904654299957767878541823e-9, fma(-n, (double)0.69314718246459960937f, x));
  constexpr double inverse[13] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                                  1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
  double y = inverse[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) y = fma(y, f, inverse[i]);
  const bool low = x < -700.0;
  y = __hiloint2double(__double2hiint(y) + (((int)n + (low ? 100 : 0)) << 20), __double2loint(y));
  return low ? y * 0x1p-100 : y;
}

// exp((z - m) scale) in 64 bits.
struct ExactWeight {
  float m;
  double scale;
  __device__ __forceinline__ double exponent(float z) const { return ((double)z - (double)m) * scale; }
  __device__ __forceinline__ double operator()(float z) const { return exp64(exponent(z)); }
};

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The first words of the order, among those that `all` keeps, that have the share topP of their weight.
template <typename TIn, int VEC, int G>
__device__ __noinline__ Cut general_share(NodeScores<TIn> s, int V, Group<G> g, Cut all, ExactWeight weight,
                                          double topP) {
  auto mass = [&](auto pick) {
    double c = 0.0;
    each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
      const unsigned u = score_key(z);
      if (all.keeps(u, v) && pick(u)) c += weight(z);
    });
    return g.sum(c);
  };
  const double share = topP * mass([](unsigned) { return true; });
  Cut cut;
  // the word that reaches the share: its key, then, among equal ones, its index
  cut.key = max(all.key, largest_key([&](unsigned x) { return mass([&](unsigned u) { return u >= x; }) >= share; }));
  const double above = mass([&](unsigned u) { return u > cut.key; }), one = weight(key_score(cut.key));
  cut.last = smallest_index(V, [&](int y) {
    int c = 0;
    each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
      c += score_key(z) == cut.key && v <= y && all.keeps(cut.key, v) ? 1 : 0;
    });
    c = g.sum(c);
    return c > 0 && above + c * one >= share;
  });
  if (cut.key == all.key) cut.last = min(cut.last, all.last);
  return cut;
}

constexpr double kUnsureSlope = 2.1 * 0x1p-24, kUnsureSum = 0x1p-22 + 20 * 0x1p-24;
constexpr int kNear = 64;          // words about a cut that are listed
constexpr float kAbove = 2.0f;     // above every weight

struct Weight {
  float m, c;
  __device__ __forceinline__ float exponent(float z) const { return __fmul_rn(__fsub_rn(z, m), c); }
  __device__ __forceinline__ float operator()(float z) const { return ex2(exponent(z)); }
};

// Which words stay: those of weight hi and above, and of those between lo and hi the ones before the cut;
// in any case those of minP and above (`exact` decides where that is close).  In 32 bits weights below FLT_MIN are 0:
// a row's words with such add up to less than 2^-98 of its weight, which is below what is unsure of any sum, so that
// it is for the 64-bit draw to have them.
struct Keep {
  float lo = FLT_MIN, hi = FLT_MIN;
  Cut cut{0u, 0x7fffffff};
  double minP = 0.0;
  ExactWeight exact;
  __device__ __forceinline__ bool operator()(float w, float z, int v) const {
    if (w < lo || (w < hi && !cut.keeps(z, v))) return false;
    if (w >= sure()) return true;
    return w >= (float)minP * 0.9999f && exact(z) >= minP;
  }
  // The 64-bit weight of a word that stays, however small, or 0.  (lo = FLT_MIN: no word is out for its weight.)
  __device__ __forceinline__ double exactly(float w, float z, int v) const {
    if ((w < lo && lo > FLT_MIN) || (w < hi && !cut.keeps(z, v))) return 0.0;
    const double x = exact(z);
    return x >= minP ? x : 0.0;
  }
  __device__ __forceinline__ float sure() const { return (float)minP * 1.0001f; }   // of minP, whatever the rounding
};

// Sums over the words that stay, in 64 bits from memory: of all of them, and of those of weight `from` and above.
struct ExactSums {
  double all, above;
};
template <typename TIn, int VEC, int G>
__device__ __noinline__ ExactSums exact_sums(NodeScores<TIn> s, int V, Group<G> g, Keep keep, Weight weight,
                                             float from) {
  double all = 0.0, above = 0.0;
  each_score<TIn, VEC, G>(s, V, g.tid, [&](float z, int v) {
    const float w = weight(z);
    if (!keep(w, z, v)) return;
    const double x = keep.exact(z);
    all += x;
    if (w >= from) above += x;
  });
  return {g.sum(all), g.sum(above)};
}

// The word that `u` picks among those that stay, in 64 bits from memory.
template <typename TIn, int VEC, int G>
__device__ __noinline__ void exact_draw(NodeScores<TIn> s, int V, int seg, Group<G> g, Keep keep,
                                        Weight weight, float u, int* word, float* logProb) {
  const Place<TIn, VEC> at(s, V, seg, g.warp, g.lane);
  auto kept = [&](float z, int v) { return keep.exactly(weight(z), z, v); };
  double part = 0.0;
#pragma unroll 1
  for (int v = at.first + g.lane * VEC; v < at.end; v += 32 * VEC) {
    float z[VEC];
    at.load(v, z);
#pragma unroll
    for (int i = 0; i < VEC; ++i) part += kept(z[i], v + i);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  part = g.exchange(part);
  double upto = part;
#pragma unroll
  for (int o = 1; o < Group<G>::kWarps; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, upto, o);
    if (g.lane >= o) upto += x;
  }
  const double total = __shfl_sync(0xffffffffu, upto, Group<G>::kWarps - 1);
  const double target = (double)u * total;
  const unsigned past = __ballot_sync(0xffffffffu, upto > target && g.lane < Group<G>::kWarps);
  // (the last warp with words that stay, should rounding let none pass)
  const unsigned some = __ballot_sync(0xffffffffu, part > 0.0 && g.lane < Group<G>::kWarps);
  const int pick = past ? __ffs(past) - 1 : 31 - __clz(some);
  if (g.warp != pick) return;
  double before = __shfl_sync(0xffffffffu, upto - part, pick);
  int found = -1;   // the first word past the target, or (rounding) the last one that stays
#pragma unroll 1
  for (int j = 0; at.first + j * 32 * VEC < at.end; ++j) {
    const int v = at.first + (j * 32 + g.lane) * VEC;
    float z[VEC];
    double w[VEC], sum = 0.0;
    if (v < at.end) at.load(v, z);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[i] = v < at.end ? kept(z[i], v + i) : 0.0;
      sum += w[i];
    }
    double scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, scan, o);
      if (g.lane >= o) scan += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, sum > 0.0 && before + scan > target);
    const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
    if (any) {
      int word = -1;
      double c = before + (scan - sum);
      bool over = false;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        c += w[i];
        if (w[i] > 0.0 && !over) word = v + i, over = c > target;
      }
      const int owner = hit ? __ffs(hit) - 1 : 31 - __clz(any);
      found = __shfl_sync(0xffffffffu, word, owner);
    }
    if (hit) break;
    before += __shfl_sync(0xffffffffu, scan, 31);
  }
  if (g.lane == 0) *word = found, *logProb = (float)(keep.exact.exponent(at.score(found)) - log(total));
}

// One group of threads per node; the row's weights take the scores' place in shared memory.  Each threshold tried is a
// pass over them, and there the time goes (issue and barriers): 14900 nodes of 10000 fp32 words take 250 us without a
// rule (2.3 TB/s of new rows) and 587 with topP = 0.9, four to five thresholds and the list; one row of 32000 words 27,
// latency.  Sums of the weights in 32 bits throughout left more draws to the 64-bit pass and were slower.  The 64
// registers that 1024 threads an SM leave are not enough: 8 to 104 bytes a thread are spilled, most by a warp per row.
template <typename TIn, int VEC, int G, bool RESIDENT>
__global__ void __launch_bounds__(kCta<G>, 1024 / kCta<G>) sample_words_kernel(
    NodeArgs a, const float* __restrict__ uniforms, int* __restrict__ words, float* __restrict__ logProbs,
    SampleRule rule, int seg) {
  constexpr int kRows = kCta<G> / G, kPass = RESIDENT ? 4 : VEC;   // words a thread takes at a time
  extern __shared__ __align__(16) float weights[];   // a warp's part of a row: seg = 128 * trips words
  __shared__ double2 scratch[64];
  __shared__ Entry listAll[kRows][kNear], sortedAll[kRows][kNear];
  __shared__ int nearAll[kRows][kNear];
  __shared__ int filledAll[kRows];
  __shared__ int sureAll[kRows];
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kRows + sub;
  if (node >= (i64)a.B * a.N) return;
  Entry *list = listAll[sub], *sorted = sortedAll[sub];
  int *near = nearAll[sub], *filled = &filledAll[sub], *sure = &sureAll[sub];
  auto answer = [&](int word, float logProb) {
    if (tid == 0) words[node] = word, logProbs[node] = logProb;
  };
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  if (!s.here) return answer(-1, 0.0f);
  float u = uniforms[node];
  u = u < 0.0f ? 0.0f : u < 1.0f ? u : 0.99999994f;
  Group<G> g(tid, scratch);
  const Place<TIn, VEC> at(s, a.V, seg, g.warp, g.lane);
  float* const row = weights + sub * seg * Group<G>::kWarps;   // (scores at first)
  float* const w = row + at.first;                             // the warp's words
  const int trips = seg / 128, own = g.lane * 4 * trips;   // a lane's words follow each other
  const float nan = __int_as_float(0x7fffffff);
  float m = neg_inf();
  bring_row<RESIDENT>(at, w, seg, [&](const float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = fmaxf(m, x[i]);
  });
  m = g.max(m);
  if (m == neg_inf() || rule.temperature == 0.0) {
    // every word is masked, or the first of the greatest scores is asked for
    int broken = 0, firstBest = 0x7fffffff;
    each_score<TIn, VEC, G>(s, a.V, tid, [&](float z, int v) {
      if (z != z) broken = 1;
      if (z == m && v < firstBest) firstBest = v;
    });
    broken = g.max(broken);
    firstBest = (int)g.min((unsigned)firstBest);
    if (broken || m == pos_inf()) return answer(-1, nan);
    return m == neg_inf() ? answer(-1, neg_inf()) : answer(firstBest, 0.0f);
  }
  const Weight weight{m, (float)(1.4426950408889634 / rule.temperature)};
  Keep keep;
  keep.exact = ExactWeight{m, 1.0 / rule.temperature};
  // f(weights, first word) for kPass words at a time: weights of 0 for those that do not stay, as far as
  // `keep` says it so far
  auto each = [&](auto f) {
    if constexpr (RESIDENT) {
      const float4* q = reinterpret_cast<const float4*>(w + own);
#pragma unroll 4
      for (int j = 0; j < trips; ++j) {
        const float4 x = q[j];
        const float y[4] = {x.x, x.y, x.z, x.w};
        f(y, at.first + own + 4 * j);
      }
    } else {
#pragma unroll 1
      for (int o = g.lane * VEC; at.first + o < at.end; o += 32 * VEC) {
        float x[VEC], y[VEC];
        at.load(at.first + o, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[i] = weight(x[i]);
          if (!(keep(y[i], x[i], at.first + o + i) || y[i] != y[i])) y[i] = 0.0f;
        }
        f(y, at.first + o);
      }
    }
  };
  // f(word) for those of this thread's words whose weight is in [from, below): few of them
  auto each_between = [&](float from, float below, auto f) {
    each([&](const float (&y)[kPass], int v) {
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < kPass; ++i) in |= y[i] >= from && y[i] < below ? 1u << i : 0u;
#pragma unroll 1
      for (; in; in &= in - 1) f(v + __ffs(in) - 1);
    });
  };
  // The sum of this thread's words that stay, a few weights at a time in 32 bits; those below keep.lo become 0 (what
  // else does not stay has been made 0), and those below keep.minP, of which a few are close to it.
  auto apply = [&] {
    double sum = 0.0;
    if constexpr (RESIDENT) {
      const float lo = keep.lo, tested = keep.sure();
      float4* q = reinterpret_cast<float4*>(w + own);
#pragma unroll 2
      for (int j = 0; j < trips; ++j) {
        const float4 x = q[j];
        float y[4] = {x.x, x.y, x.z, x.w};
        bool test = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = y[i] < lo ? 0.0f : y[i];
          test |= y[i] > 0.0f && y[i] < tested;
        }
        if (test) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (y[i] > 0.0f && y[i] < tested && keep.exact(at.score(at.first + own + 4 * j + i)) < keep.minP)
              y[i] = 0.0f;
        }
        q[j] = make_float4(y[0], y[1], y[2], y[3]);
        sum += (double)((y[0] + y[1]) + (y[2] + y[3]));
      }
    } else {
      each([&](const float (&y)[kPass], int) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) sum += (double)y[i];
      });
    }
    return sum;
  };
  // The weights, and where a share of them is looked for their moments: of |x| for the bound on what is unsure,
  // of x^2 for a first guess.
  double part = 0.0;
  float slope = 0.0f, square = 0.0f;
  auto form = [&](auto guessed) {
    auto moments = [&](float x, float y) {
      if (!decltype(guessed)::value) return;
      const float b = fmaxf(x, -200.0f);
      slope = fmaf(-b, y, slope);
      square = fmaf(b * b, y, square);
    };
    if constexpr (RESIDENT) {
      float4* q = reinterpret_cast<float4*>(w + own);
#pragma unroll 2
      for (int j = 0; j < trips; ++j) {
        const float4 x = q[j];
        const float z[4] = {x.x, x.y, x.z, x.w};
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = weight.exponent(z[i]);
          y[i] = ex2(e);
          moments(e, y[i]);
        }
        q[j] = make_float4(y[0], y[1], y[2], y[3]);
        part += (double)((y[0] + y[1]) + (y[2] + y[3]));
      }
    } else {
#pragma unroll 1
      for (int o = g.lane * VEC; at.first + o < at.end; o += 32 * VEC) {
        float x[VEC];
        at.load(at.first + o, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float e = weight.exponent(x[i]), y = ex2(e);
          moments(e, y);
          part += (double)y;
        }
      }
    }
  };
  if (rule.topP < 1.0) form(std::true_type{});
  else form(std::false_type{});
  double total = part;
  if (rule.topP < 1.0) g.sum(total, slope);
  else total = g.sum(total), slope = (float)total * lg2((float)a.V);   // (its bound)
  if (total != total) return answer(-1, nan);
  const double unsure = 1.01 * kUnsureSlope * slope + kUnsureSum * total;

  // The first words of the order with a count of k, or a weight of topP * total.  False: that is all.
  // A threshold that fewer reach and one that enough reach are brought together until at most kNear words
  // lie between them.  Weights add up to about a logistic function of the exponent (log-counts are about
  // linear): that gives the next threshold, a little past the target towards the farther end, so that
  // the two close in from both sides; the first is that of a normal distribution.  4 to 5 rounds for
  // topP = 0.9 and 10000 words, 11 with the weights themselves taken for linear.
  auto find_cut = [&](auto by_weight, int k, float guess) {
    constexpr bool kByWeight = decltype(by_weight)::value;
    double target = kByWeight ? rule.topP * total : (double)k;
    // (counts decide as whole numbers: 32-bit floats have all of them up to 2^24 only)
    int count = 0, countHi = 0;   // measured last, and at `hi`
    auto measure = [&](float t) -> float {
      if constexpr (!kByWeight) {
        int c = 0;
        each([&](const float (&y)[kPass], int) {
#pragma unroll
          for (int i = 0; i < kPass; ++i) c += y[i] >= t ? 1 : 0;
        });
        count = g.sum(c);
        return (float)count;
      } else if constexpr (RESIDENT) {
        float sum[8] = {};
        const float4* q = reinterpret_cast<const float4*>(w + own);
        auto add = [&](const float4& x, int i) {
          if (x.x >= t) sum[i] += x.x;
          if (x.y >= t) sum[i + 1] += x.y;
          if (x.z >= t) sum[i + 2] += x.z;
          if (x.w >= t) sum[i + 3] += x.w;
        };
        int j = 0;
#pragma unroll 2
        for (; j + 1 < trips; j += 2) {
          const float4 x = q[j], y = q[j + 1];
          add(x, 0);
          add(y, 4);
        }
        if (j < trips) add(q[j], 0);
        return g.sum(((sum[0] + sum[4]) + (sum[1] + sum[5])) + ((sum[2] + sum[6]) + (sum[3] + sum[7])));
      } else {
        double sum = 0.0;
        each([&](const float (&y)[kPass], int) {
#pragma unroll
          for (int i = 0; i < kPass; ++i)
            if (y[i] >= t) sum += (double)y[i];
        });
        return (float)g.sum(sum);
      }
    };
    const float floor = (float)(1e-5 * total), all = (float)total;
    float want = (float)target;
    auto level = [&](float v) {
      return kByWeight ? lg2(fmaxf(v, 0.25f)) - lg2(fmaxf(all - v, floor)) : -lg2(fmaxf(v, 0.5f));
    };
    // thresholds, what has been measured there, their exponents and levels
    float lo = FLT_MIN, hi = kAbove, vLo = 0.0f, vHi = 0.0f, xLo = -126.0f, xHi = 0.1f, lLo = 0.0f, lHi = level(0.0f);
    if (kByWeight) {
      // (the words below a quarter of (1 - topP) / V cannot be needed for the share)
      lo = fmaxf(0.25f * (1.0f - (float)rule.topP) / (float)a.V, FLT_MIN), xLo = lg2(lo);
      vLo = all * (1.0f - 0.25f * (1.0f - (float)rule.topP)), lLo = level(vLo);
    }
    float t = guess, x = lg2(guess), had = 3e38f;
    const float lWant = level(want);
    int stuck = 0, wrong = 0;
    bool done = false;
    Cut cut;
#pragma unroll 1
    for (int round = 0; round < 64 && !done; ++round) {
      const float v = measure(t), l = level(v);
      if (kByWeight ? v >= want : count >= k) lo = t, vLo = v, xLo = x, lLo = l;
      else hi = t, vHi = v, xHi = x, lHi = l, countHi = count;
      if (vLo == 0.0f) {   // nothing is known from below yet
        if (t == FLT_MIN) return false;   // there are no more words than that
        t = round == 0 && t > 1e-9f ? t * 1e-3f : FLT_MIN;
        x = lg2(t);
        continue;
      }
      // how many words lie between: known, or at most the weight over the lesser threshold
      const float between = kByWeight ? __fdividef(vLo - vHi, lo) : vLo - vHi;
      bool listed = between <= (kByWeight ? 1.25f * kNear : (float)kNear);
      int c = 0;
      if (listed) {
        g.sync();
        if (tid == 0) *filled = 0;
        g.sync();
        each_between(lo, hi, [&](int v) {
          const int i = atomicAdd(filled, 1);
          if (i < kNear) near[i] = v;
        });
        g.sync();
        c = *filled;
        listed = c <= kNear;   // (weights next to nothing may be more)
        if (listed) {
          for (int i = tid; i < c; i += G) list[i] = entry_of(at.score(near[i]), near[i]);
          g.sync();
        }
      }
      if (!listed) {
        stuck = between > 0.5f * had ? stuck + 1 : 0;
        had = between;
        float f = __fdividef(lLo - lWant, lLo - lHi);
        const float past = __fdividef(0.3f * kNear, fmaxf(between, (float)kNear));
        f = stuck >= 2 ? 0.5f : f < 0.5f ? f + past : f - past;
        f = fminf(fmaxf(f, 0.01f), 0.99f);
        x = xLo + f * (xHi - xLo);
        t = ex2(x);
        if (!(t > lo && t < hi)) {
          t = __uint_as_float((__float_as_uint(lo) + __float_as_uint(hi)) / 2);
          x = lg2(t);
        }
        if (!(t > lo && t < hi)) break;
        continue;
      }
      if constexpr (G >= 4 * kNear) {   // four threads per entry, each looking at every fourth of the others
        const Entry mine = tid / 4 < c ? list[tid / 4] : ~0ull;
        int place = 0;
#pragma unroll 4
        for (int i = tid % 4; i < c; i += 4) place += list[i] > mine ? 1 : 0;
        place += __shfl_xor_sync(0xffffffffu, place, 1);
        place += __shfl_xor_sync(0xffffffffu, place, 2);
        if (tid % 4 == 0 && tid / 4 < c) sorted[place] = mine;
      } else {
        for (int i = tid; i < c; i += G) {
          const Entry mine = list[i];
          sorted[entries_before(list, c, mine)] = mine;
        }
      }
      g.sync();
      int kept = k - countHi;
      bool enough = true;
      if (kByWeight) {
        // by one warp: lane i has entries 2 i and 2 i + 1.  In 32 bits, or, where the sum up to a word is too close
        // to the target to tell, in 64 bits from memory.
        const int i0 = 2 * g.lane, i1 = i0 + 1;
        auto settle = [&](double above, double share, double w0, double w1, double margin) {
          double upto = w0 + w1;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, upto, o);
            if (g.lane >= o) upto += x;
          }
          // the words whose predecessors have not reached the target
          const double d0 = above + (upto - w1 - w0) - share, d1 = above + (upto - w1) - share;
          const double end = above + __shfl_sync(0xffffffffu, upto, 31) - share;
          const bool close = (i0 < c && fabs(d0) <= margin) || (i1 < c && fabs(d1) <= margin) || fabs(end) <= margin;
          const unsigned b0 = __ballot_sync(0xffffffffu, i0 < c && d0 < 0.0);
          const unsigned b1 = __ballot_sync(0xffffffffu, i1 < c && d1 < 0.0);
          const bool any = __any_sync(0xffffffffu, close);
          if (g.lane == 0) *filled = 4 * (__popc(b0) + __popc(b1)) + (end >= 0.0 ? 2 : 0) + (any ? 1 : 0);
        };
        auto score = [&](int i) { return i < c ? key_score(entry_key(sorted[i])) : neg_inf(); };
        if (g.warp == 0) settle((double)vHi, target, (double)weight(score(i0)), (double)weight(score(i1)), unsure);
        g.sync();
        if (*filled & 1) {
          const ExactSums sums = exact_sums<TIn, VEC, G>(s, a.V, g, keep, weight, hi);
          target = rule.topP * sums.all;
          g.sync();
          if (g.warp == 0) settle(sums.above, target, keep.exact(score(i0)), keep.exact(score(i1)), -1.0);
          g.sync();
        }
        kept = *filled >> 2;
        enough = *filled & 2;
      }
      // A threshold whose side 32 bits have taken wrongly, the target being closer to the sum there than they can tell:
      // the next one is beyond it, farther and farther off until a word has been passed (in steps of a rounding that
      // took up to 54 rounds), and what is wanted is moved past the sum so that none on the way is taken wrongly again.
      if (kByWeight && (!enough || kept == 0)) {
        const float step = ex2((float)(4 * wrong++ - 14));
        want = enough ? vHi : __uint_as_float(__float_as_uint(vLo) + 1);
        x = enough ? xHi + step : xLo - step;
        t = fminf(fmaxf(ex2(x), FLT_MIN), kAbove);
        continue;
      }
      // (32-bit weights of different scores may come out in the wrong order by a rounding: not so the
      // cut's and those beyond the thresholds)
      const Entry last = sorted[kept - 1];
      cut = Cut{entry_key(last), entry_word(last)};
      const float y = weight(key_score(cut.key));
      if (hi < kAbove && y * 1.000004f >= hi) t = hi * 1.00003f, x = xHi;
      else if (!(y * 0.999996f < lo)) done = true;
      else if (lo > FLT_MIN) t = fmaxf(lo * 0.99997f, FLT_MIN), x = xLo;
      else break;   // (beside weights that are 0 here)
      if constexpr (RESIDENT)   // what lies between and does not stay
        if (done)
          for (int i = kept + tid; i < c; i += G) row[entry_word(sorted[i])] = 0.0f;
    }
    if (!done) {
      cut = kByWeight ? general_share<TIn, VEC, G>(s, a.V, g, keep.cut, keep.exact, rule.topP)
                      : general_first_k<TIn, VEC, G>(s, a.V, g, k);
      g.sync();
      lo = FLT_MIN;
      hi = kAbove;
      if constexpr (RESIDENT)
        each([&](const float (&)[kPass], int v) {
          for (int i = 0; i < kPass; ++i)
            if (v + i < a.V && !cut.keeps(at.score(v + i), v + i)) row[v + i] = 0.0f;
        });
    }
    g.sync();
    keep.lo = lo;
    keep.hi = hi;
    keep.cut = cut;
    return true;
  };
  bool cutAny = false;   // `keep` says something that has not been applied
  bool open = false;     // the cut lies among weights that are 0 in 32 bits
  if (rule.topK > 0 && rule.topK < a.V) {
    cutAny = find_cut(std::false_type{}, rule.topK, 0x1p-8f);
    open = !cutAny && rule.topP == 1.0;
    if (cutAny && rule.topP < 1.0) total = g.sum(apply());
  }
  if (rule.topP < 1.0) {
    const float mean = __fdividef(-slope, (float)total);
    const float spread2 = __fdividef(g.sum(square), (float)total) - mean * mean;
    const float p = (float)rule.topP, odds = 0.55f * 0.6931472f * (lg2(p) - lg2(1.0f - p));
    float deviation;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(deviation) : "f"(fmaxf(spread2, 0.0f)));
    find_cut(std::true_type{}, 0, fmaxf(ex2(fminf(mean - odds * deviation, -0.05f)), 0.5f * (1.0f - p) / (float)a.V));
    cutAny = true;
  }
  if (rule.minP > 0.0) {
    keep.minP = rule.minP;
    keep.lo = fmaxf(keep.lo, (float)rule.minP * 0.9999f);
    cutAny = true;
  }

  // the draw: the warp, its vectors, the word
  if (cutAny) part = apply();
  // sums up to and with each lane's words, then each warp's
  double scan = part;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, scan, d);
    if (g.lane >= d) scan += x;
  }
  const double whole = g.exchange(__shfl_sync(0xffffffffu, scan, 31));
  double upto = whole;
#pragma unroll
  for (int d = 1; d < Group<G>::kWarps; d <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, upto, d);
    if (g.lane >= d) upto += x;
  }
  total = __shfl_sync(0xffffffffu, upto, Group<G>::kWarps - 1);
  const double target = (double)u * total;
  const unsigned past = __ballot_sync(0xffffffffu, upto > target && g.lane < Group<G>::kWarps);
  const int pick = past ? __ffs(past) - 1 : Group<G>::kWarps - 1;
  if (g.warp == pick) {
    double before = __shfl_sync(0xffffffffu, upto - whole, pick);
    int found = -1;
    bool certain = false;
    float mine = 0.0f;
    if constexpr (RESIDENT) {
      const unsigned hit = __ballot_sync(0xffffffffu, before + scan > target);
      if (hit && g.lane == __ffs(hit) - 1) {   // one of this lane's words
        before += scan - part;
        const float4* q = reinterpret_cast<const float4*>(w + own);
#pragma unroll 2
        for (int j = 0; j < trips && found < 0; ++j) {
          const float4 x = q[j];
          const float y[4] = {x.x, x.y, x.z, x.w};
          float few = 0.0f;
          double b = before;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            few += y[i];
            const double after = before + (double)few;
            if (found < 0 && after > target) {
              found = at.first + own + 4 * j + i;
              mine = y[i];
              certain = y[i] > 0.0f && target - b > unsure && after - target > unsure;
            }
            b = after;
          }
          before = b;
        }
      }
      const int owner = hit ? __ffs(hit) - 1 : 0;
      found = __shfl_sync(0xffffffffu, found, owner);
      mine = __shfl_sync(0xffffffffu, mine, owner);
      certain = __shfl_sync(0xffffffffu, certain ? 1 : 0, owner);
    } else {
#pragma unroll 1
      for (int o = 0; found < 0 && at.first + o < at.end; o += 32 * VEC) {
        const int v = at.first + o + g.lane * VEC;
        float x[VEC], y[VEC];
        double sum = 0.0;
        if (v < at.end) at.load(v, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[i] = v < at.end ? weight(x[i]) : 0.0f;
          if (v < at.end && !keep(y[i], x[i], v + i)) y[i] = 0.0f;
          sum += (double)y[i];
        }
        double upTo = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double z = __shfl_up_sync(0xffffffffu, upTo, d);
          if (g.lane >= d) upTo += z;
        }
        if (const unsigned hit = __ballot_sync(0xffffffffu, before + upTo > target)) {
          double b = before + (upTo - sum);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const double after = b + (double)y[i];
            if (found < 0 && after > target) {
              found = v + i;
              mine = y[i];
              certain = y[i] > 0.0f && target - b > unsure && after - target > unsure;
            }
            b = after;
          }
          const int owner = __ffs(hit) - 1;
          found = __shfl_sync(0xffffffffu, found, owner);
          mine = __shfl_sync(0xffffffffu, mine, owner);
          certain = __shfl_sync(0xffffffffu, certain ? 1 : 0, owner);
          break;
        }
        before += __shfl_sync(0xffffffffu, upTo, 31);
      }
    }
    if (g.lane == 0) {
      *sure = certain;
      if (certain) words[node] = found, logProbs[node] = logf(mine / (float)total);
    }
  }
  g.sync();
  if (*sure) return;
  if (open) {
    keep.cut = general_first_k<TIn, VEC, G>(s, a.V, g, rule.topK);
    keep.hi = kAbove;
    g.sync();
  }
  exact_draw<TIn, VEC, G>(s, a.V, seg, g, keep, weight, u, words + node, logProbs + node);
}

}  // namespace

void launch_sample_words(const NodeArgs& a, const float* uniforms, int* words, float* logProbs,
                         SampleRule rule, cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (nodes == 0) return;
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_group(a.V, true, [&](auto group, auto resident) {
      constexpr int G = decltype(group)::value, rows = kCta<G> / G;
      auto kernel = sample_words_kernel<TIn, decltype(vec)::value, G, decltype(resident)::value>;
      const int seg = words_of_warp(a.V, G / 32);
      const int smem = decltype(resident)::value ? rows * seg * (G / 32) * (int)sizeof(float) : 0;
      if (smem > 32 * 1024) allow_dyn_smem(kernel, G == 32 ? 64 * 1024 : kResidentBytes);
      ScopedKernel prof("sample_words", stream);
      kernel<<<(unsigned)div_up64(nodes, rows), kCta<G>, smem, stream>>>(a, uniforms, words, logProbs, rule, seg);
      TB200_CHECK_LAUNCH();
    });
  });
}

}  // namespace tb200
