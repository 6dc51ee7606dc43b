// Distillation at single lattice nodes from a teacher's recorded best words.
//
// The teacher's record of a node is K words with logits l_k, and optionally l_r, the log-sum-exp of all
// its other words: q = softmax over these bins (r: the last one's share).  With the student's scores
// z = (E[t,:] + P[u,:]) / temperature, p = softmax(z) and R = log-sum-exp of z over the words that
// are not listed,
//   cost    = sum_k q_k (log q_k - log p_k) + r (log r - (R - L)),   L = log-sum-exp of all z,
//   dc/dz_v = p_v - q_v for listed words, p_v - r exp(z_v - R) for the others,
// times 1 / temperature for the gradients with respect to E[t,:] and P[u,:], which are sums over the
// nodes on frame t resp. position u.  For the others the gradient is exp(z_v - L) (1 - r/rho), rho =
// exp(R - L): one exponential, exp(z_v - A) with A = L - log|1 - r/rho| and the sign of 1 - r/rho.
#include <algorithm>

#include "node_rows.cuh"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kForwardBytes = 64 * 1024;   // of shared memory, at most
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Running maximum of the scores and sum of 2^((score - maximum) scale2).  The maximum is subtracted
// before the scaling, so that scores as low as the type's lowest number still have a softmax.
struct RunningSum {
  float m = -3.402823466e38f, s = 0.0f;   // (a finite start: the difference from it is never NaN)
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N], float scale2) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) {
      s *= ex2((m - top) * scale2);
      m = top;
    }
    float sum[2] = {s, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i % 2] += ex2((z[i] - m) * scale2);
    s = sum[0] + sum[1];
  }
  __device__ __forceinline__ void add(RunningSum o, float scale2) {
    const float top = fmaxf(m, o.m);
    s = s * ex2((m - top) * scale2) + o.s * ex2((o.m - top) * scale2);
    m = top;
  }
  template <typename Gr>
  __device__ __forceinline__ void join(Gr& g, float scale2) {
    const float top = g.max(m);
    s = g.sum(s * ex2((m - top) * scale2));
    m = top;
  }
  // log2 of the sum, relative to a maximum `ref` that is no smaller; -inf where there is no word
  __device__ __forceinline__ float log2sum(float ref, float scale2) const {
    return s == 0.0f ? neg_inf() : (m - ref) * scale2 + log2f(s);
  }
};

// The same with two operations less per word: sum of 2^(z scale2 - r) for a whole number r, one fused operation for
// the exponent, whatever the words' maximum: r follows when the sum gets large.  Scores whose multiples by scale2 lie
// beyond +-2^20 are left to RunningSum, as are sums that are not finite.
struct QuickSum {
  static constexpr float kRange = 0x1p20f;
  float r = -kRange, s = 0.0f;
  template <int N>
  __device__ __forceinline__ float weights(const float (&z)[N], float scale2) const {
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i % 2] += ex2(fmaf(z[i], scale2, -r));
    return sum[0] + sum[1];
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N], float scale2) {
    float sum = weights(z, scale2);
    if (!(sum < 0x1p60f)) {
      float top = z[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
      const float to = fminf(rintf(top * scale2), kRange);
      s *= ex2(r - to);
      r = to;
      sum = weights(z, scale2);
    }
    s += sum;
  }
  // s in [1, 2) relative to a score; NaN where RunningSum has to do it
  __device__ __forceinline__ RunningSum sum(float scale2) const {
    RunningSum x;
    if (s == 0.0f) return x;
    if (!(s >= 0.5f && s < pos_inf())) {   // (below 0.5: no word has come near r)
      x.s = __int_as_float(0x7fffffff);
      return x;
    }
    const int exponent = (int)(__float_as_uint(s) >> 23) - 127;
    const float whole = r + (float)exponent;
    x.m = __fdividef(whole, scale2);
    x.s = __uint_as_float(__float_as_uint(s) - ((unsigned)exponent << 23)) * ex2(-fmaf(x.m, scale2, -whole));
    return x;
  }
};

constexpr int kLookBack = 64;   // places without a node that a path may have between two nodes

// Where a node lies: of consecutive nodes on the same frame, or position, the first and the last one speak for all.
__device__ __forceinline__ void mark_spans(const NodeArgs& a, const DistillSaved& k, i64 node, int n, int t, int u,
                                           int tBefore, int uBefore, int tAfter, int uAfter) {
  auto valid = [&](int t, int u) { return (unsigned)t < (unsigned)a.T && (unsigned)u < (unsigned)a.U; };
  const i64 b = (unsigned)(node - n) / (unsigned)a.N;
  const bool before = valid(tBefore, uBefore), after = valid(tAfter, uAfter);
  int2* frame = k.spans + b * a.T + t;
  int2* position = k.spans + (i64)a.B * a.T + b * a.U + u;
  if (!before || tBefore != t) {
    atomicMax(&frame->x, a.N - n);
    k.segUsed[b * k.segs + t / k.segFrames] = 1;
  }
  if (!after || tAfter != t) atomicMax(&frame->y, n + 1);
  if (!before || uBefore != u) atomicMax(&position->x, a.N - n);
  if (!after || uAfter != u) atomicMax(&position->y, n + 1);
  if (!before) {
    int back = 2;
    while (back <= n && back <= kLookBack && !valid(a.frames[node - back], a.positions[node - back])) ++back;
    if (back > n) return;   // (the first node)
    tBefore = back > kLookBack ? a.T : a.frames[node - back], uBefore = a.positions[node - back];
  }
  if (tBefore > t || uBefore > u) k.offPath[b] = 1;
}

// A word of the teacher's record.
struct Listed {
  int word;      // -1: outside the vocabulary
  float share;   // of the teacher's distribution; kNoShare: the word is ignored, or an earlier place has its share
  float z;       // the student's score
};

constexpr int kWarpNodes = 8;   // nodes per CTA where a warp has a node
template <int G>
constexpr int kCta = G == 32 ? 32 * kWarpNodes : G;

// The row of E comes through a ring in shared memory, a turn of kTurn vectors of each lane at a time, and the listed
// words are masked there by the lanes that have their places.  (With a bit per word, looked up for each vector, every
// second turn of a warp went through the masking code: 371 us against 331 for 58800 nodes of 10000 bf16 words.)
template <int VEC>
constexpr int kTurn = VEC == 1 ? 8 : 2;
constexpr int kTurns = 4;   // in the ring
template <typename TIn, int VEC>
constexpr int kRingWords = kTurns * kTurn<VEC> * 32 * VEC;   // of a warp

// One group of G threads per node: one pass over the row with a running reference and sum.  Bound by the issue of
// instructions (75 % of the slots): about 1200 for a node whatever its size, the teacher's softmax, the logarithms
// and the gradients of the listed words, and eight for each of a lane's words.  58800 nodes: 331 us with 10000 bf16
// words (3.6 TB/s of E), 98 us with 512.  A warp per node needs no barriers; a CTA of 256 per node is for few long
// rows only. Dynamic shared memory: the warps' rings, and per node its record, K Listed.
template <typename TIn, int VEC, int G, bool REST>
__global__ void __launch_bounds__(kCta<G>, (VEC == 1 && sizeof(TIn) == 4 ? 768 : 1024) / kCta<G>)
    distill_forward_kernel(
    NodeArgs a, const int* __restrict__ words, const float* __restrict__ logits,
    const float* __restrict__ rest, float* __restrict__ costs, DistillSaved saved, int K, float scale2) {
  constexpr int kNodes = kCta<G> / G;
  extern __shared__ __align__(16) unsigned char memory[];
  __shared__ double2 scratch[64];
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kNodes + sub;
  if (node >= (i64)a.B * a.N) return;
  TIn* const ring = reinterpret_cast<TIn*>(memory) + threadIdx.x / 32 * kRingWords<TIn, VEC>;
  constexpr int kRings = kCta<G> / 32 * kRingWords<TIn, VEC> * (int)sizeof(TIn);
  Listed* const record = reinterpret_cast<Listed*>(memory + kRings) + sub * K;
  float2* const savedListed = saved.listed ? saved.listed + node * K : nullptr;
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  if (!s.here) {
    if (tid == 0) costs[node] = 0.0f;
    if (savedListed) {
      for (int k = tid; k < K; k += G) savedListed[k] = make_float2(kNoShare, 0.0f);
      if (tid == 0) saved.node[node] = make_float4(0.0f, pos_inf(), 1.0f, 0.0f);
    }
    return;
  }
  // (the nodes before and after: their frames and positions, wanted at the end)
  const i64 beside = node + (tid < 2 ? -1 : 1);
  const int n = (int)((unsigned)node % (unsigned)a.N);
  int around = -1;
  if (savedListed && tid < 4 && (tid < 2 ? n > 0 : n + 1 < a.N)) around = (tid & 1 ? a.positions : a.frames)[beside];
  Group<G> g(tid, scratch);
  // vectors c = 0, 1, ... of this thread, the words (c * G + tid) * VEC and on, are in turn c / kTurn; place(c): in
  // the ring
  const int turns = div_up(a.V, G * VEC * kTurn<VEC>);
  auto place = [&](int c) { return c % (kTurns * kTurn<VEC>) * 32 * VEC; };
  auto fetch = [&](int turn) {
    if (turn < turns) {
#pragma unroll
      for (int j = 0; j < kTurn<VEC>; ++j) {
        const int c = turn * kTurn<VEC> + j, v = (c * G + tid) * VEC;
        TIn* const slot = ring + place(c) + g.lane * VEC;
        if (v >= a.V) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) from_f32(slot[i], neg_inf());
        } else if constexpr (VEC * sizeof(TIn) >= 4) {
          copy_async<VEC * sizeof(TIn)>(slot, s.e + v);
        } else {
          *slot = s.e[v];   // (too small for an asynchronous copy)
        }
      }
    }
    commit_copies();
  };
  // the student's sum over the words that are not listed (all words, without REST)
  auto begin = [&] {
#pragma unroll 1
    for (int i = 0; i < kTurns - 1; ++i) fetch(i);
  };
  auto add_row = [&](auto& sum) {
    // the listed words of this lane: the turn, and the place in the ring (-1: another warp's)
    auto find = [&](int k, int& turn, int& at) {
      const int v = k < K ? record[k].word : -1;
      const int q = v / VEC, c = q / G, owner = q % G;
      turn = v >= 0 && owner / 32 == g.warp ? c / kTurn<VEC> : -1;
      at = place(c) + owner % 32 * VEC + v % VEC;
    };
    [[maybe_unused]] int hit = -1, at = 0;
    if constexpr (REST) find(g.lane, hit, at);
#pragma unroll 1
    for (int turn = 0; turn < turns; ++turn) {
      RawWords<TIn, VEC> p[kTurn<VEC>];
#pragma unroll
      for (int j = 0; j < kTurn<VEC>; ++j) {
        const int v = ((turn * kTurn<VEC> + j) * G + tid) * VEC;
        p[j].load(s.p + (v < a.V ? v : 0));
      }
      fetch(turn + kTurns - 1);
      wait_copies<kTurns - 1>();
      if constexpr (REST) {
        __syncwarp();
        if (turn == hit) from_f32(ring[at], neg_inf());
        if (K > 32) {
#pragma unroll 1
          for (int k = g.lane + 32; k < K; k += 32) {
            int turnOf, there;
            find(k, turnOf, there);
            if (turn == turnOf) from_f32(ring[there], neg_inf());
          }
        }
        __syncwarp();
      }
      float z[VEC * kTurn<VEC>];
#pragma unroll
      for (int j = 0; j < kTurn<VEC>; ++j) {
        RawWords<TIn, VEC> e;
        e.load(ring + place(turn * kTurn<VEC> + j) + g.lane * VEC);
        const Words<VEC> x = e.words(), y = p[j].words();
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[j * VEC + i] = x.x[i] + y.x[i];
      }
      sum.add(z, scale2);
    }
  };
  begin();
  // the teacher's shares
  const float lRest = REST ? rest[node] : neg_inf();
  float top = lRest;
  for (int k = tid; k < K; k += G) {
    Listed x{words[node * K + k], logits[node * K + k], neg_inf()};
    if ((unsigned)x.word >= (unsigned)a.V) x.word = -1, x.share = neg_inf();
    else x.z = to_f32(s.e[x.word]) + to_f32(s.p[x.word]);
    record[k] = x;
    top = fmaxf(top, x.share);
  }
  top = g.max(top);
  float sum = 0.0f;
  for (int k = tid; k < K; k += G) {
    const float l = record[k].share, x = l == neg_inf() ? 0.0f : expf(l - top);
    record[k].share = x;
    sum += x;
  }
  float r = REST && lRest != neg_inf() ? expf(lRest - top) : 0.0f;
  sum = g.sum(sum) + r;
  g.sync();
  const bool empty = top == neg_inf();   // the record has no weight: cost and gradient are 0
  const float one = empty ? 0.0f : 1.0f / sum;
  r *= one;
  // A word that is listed more than once: its first place has all its shares.
  bool twice = false;
  if (G == 32 && K <= 32) {
    const int v = tid < K ? record[tid].word : -1 - tid;
    twice = (__match_any_sync(0xffffffffu, v) & ~(1u << tid)) != 0 && v >= 0;
  } else {
    for (int k = tid; k < K; k += G) {
      const int v = record[k].word;
      for (int j = 0; j < K; ++j) twice |= v >= 0 && j != k && record[j].word == v;
    }
  }
  const bool repeated = g.max(twice ? 1 : 0) != 0;
  float all[kMaxListedWords / G > 0 ? kMaxListedWords / G : 1];   // of this thread's words
#pragma unroll
  for (int i = 0; i < (int)(sizeof(all) / sizeof(float)); ++i) {
    const int k = tid + i * G;
    if (k >= K) break;
    const int v = record[k].word;
    all[i] = v < 0 ? kNoShare : record[k].share * one;
    if (repeated && v >= 0) {
      float x = 0.0f;
      bool first = true;
      for (int j = 0; j < K; ++j)
        if (record[j].word == v) {
          first = first && j >= k;
          x += record[j].share;
        }
      all[i] = first ? x * one : kNoShare;
    }
  }
  if (repeated) g.sync();   // (everybody has read the record)
#pragma unroll
  for (int i = 0; i < (int)(sizeof(all) / sizeof(float)); ++i) {
    const int k = tid + i * G;
    if (k < K) record[k].share = all[i];
  }
  g.sync();
  QuickSum quick;
  add_row(quick);
  RunningSum others = quick.sum(scale2);
  others.join(g, scale2);
  if (!(others.s > 0.0f && others.s < pos_inf())) {   // (the same for the whole group)
    others = RunningSum();
    begin();
    add_row(others);
    others.join(g, scale2);
  }
  RunningSum full = others;
  if constexpr (REST) {
    RunningSum mine;
    for (int k = tid; k < K; k += G) {
      const float z[1] = {record[k].share != kNoShare ? record[k].z : neg_inf()};
      mine.add(z, scale2);
    }
    mine.join(g, scale2);
    full.add(mine, scale2);
  }
  const float all2 = full.log2sum(full.m, scale2), other2 = others.log2sum(full.m, scale2);
  // what of the gradient a listed word shares with the others
  float logRatio = neg_inf();   // of r to the student's weight of the others
  if (REST && r > 0.0f && other2 != neg_inf()) logRatio = logf(r) - (other2 - all2) * kLn2;
  const bool apart = logRatio > kLn2;   // (more than 2: listed words would be differences of large numbers)
  const float ratio = apart ? 1.0f : expf(logRatio);
  float cost = 0.0f;
  for (int k = tid; k < K; k += G) {
    const float q = record[k].share, z = record[k].z;
    const float logP = z == neg_inf() ? z : ((z - full.m) * scale2 - all2) * kLn2;
    if (q != kNoShare && q != 0.0f) cost += q * (logf(q) - logP);
    if (savedListed) {
      const float p = z == neg_inf() || empty ? 0.0f : expf(logP);
      savedListed[k] = q == kNoShare ? make_float2(q, 0.0f) : make_float2(q - ratio * p, p - q);
    }
  }
  cost = g.sum(cost);
  if (tid >= 32) return;
  const int tBefore = __shfl_sync(0xffffffffu, around, 0), uBefore = __shfl_sync(0xffffffffu, around, 1);
  const int tAfter = __shfl_sync(0xffffffffu, around, 2), uAfter = __shfl_sync(0xffffffffu, around, 3);
  if (tid != 0) return;
  if (REST && r != 0.0f) cost += r * (logf(r) - (other2 == neg_inf() ? other2 : (other2 - all2) * kLn2));
  costs[node] = cost;
  if (!savedListed) return;
  // (an empty record has no gradient, and a student without any word left has p = 0)
  const float L = empty || all2 == neg_inf() ? pos_inf() : all2;
  float m = full.m, A = L, sign = 1.0f;
  if (apart && !empty) {   // (r - rho times the others' own softmax, however far they are below the listed words)
    sign = -2.0f;
    m = others.m;
    A = log2f(others.s) - log2f(r - ex2(other2 - all2));
  } else if (logRatio != neg_inf()) {
    sign = logRatio > 0.0f ? -1.0f : 1.0f;
    A = L - (fmaxf(logRatio, 0.0f) + log1pf(-expf(-fabsf(logRatio)))) * kLog2e;
  }
  saved.node[node] = make_float4(m, A, sign, 0.0f);
  mark_spans(a, saved, node, n, s.t, s.u, tBefore, uBefore, tAfter, uAfter);
}

// The greatest indices of a call, so that it can be refused: one CTA per 16384 of them, up to 64.
__global__ void __launch_bounds__(512) node_summary_kernel(const int* __restrict__ frames,
                                                           const int* __restrict__ positions, i64 nodes,
                                                           const int* __restrict__ words, i64 wordCount,
                                                           int* __restrict__ most) {
  __shared__ double2 scratch[64];
  Group<512> g(threadIdx.x, scratch);
  const i64 first = (i64)blockIdx.x * 512 + threadIdx.x, step = (i64)gridDim.x * 512;
  int frame = -1, position = -1, word = -1;
  for (i64 i = first; i < nodes; i += step) frame = max(frame, frames[i]), position = max(position, positions[i]);
#pragma unroll 8
  for (i64 i = first; i < wordCount; i += step) word = max(word, words[i]);
  frame = g.max(frame);
  position = g.max(position);
  word = g.max(word);
  if (threadIdx.x == 0) {
    int* mine = most + 3 * blockIdx.x;
    mine[0] = frame, mine[1] = position, mine[2] = word;
  }
}

template <typename F>
void with_flag(bool on, F launch) {
  if (on) launch(std::true_type{});
  else launch(std::false_type{});
}

}  // namespace

int node_summary_ctas(i64 nodes, i64 wordCount) {
  return (int)std::min<i64>(64, std::max<i64>(1, (nodes + wordCount) / 16384));
}

void launch_node_summary(const int* frames, const int* positions, i64 nodes, const int* words, i64 wordCount,
                         int* most, cudaStream_t stream) {
  ScopedKernel prof("node_summary", stream);
  node_summary_kernel<<<node_summary_ctas(nodes, wordCount), 512, 0, stream>>>(frames, positions, nodes, words,
                                                                              words ? wordCount : 0, most);
  TB200_CHECK_LAUNCH();
}

void launch_distill_forward(const NodeArgs& a, const int* words, const float* logits, const float* rest,
                            float* costs, DistillSaved saved, int K, double temperature,
                            cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (saved.spans)
    TB200_CUDA_CHECK(cudaMemsetAsync(saved.spans, 0, sizeof(int) * a.B * (2 * ((size_t)a.T + a.U) + 1 + saved.segs),
                                     stream));
  if (nodes == 0) return;
  const float scale2 = (float)(1.4426950408889634 / temperature);
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_flag(rest != nullptr, [&](auto has_rest) {
      auto launch = [&](auto group) {
        constexpr int G = group, rows = kCta<G> / G;
        auto kernel = distill_forward_kernel<TIn, vec, G, has_rest>;
        const int smem = kCta<G> / 32 * kRingWords<TIn, vec> * (int)sizeof(TIn) + rows * K * (int)sizeof(Listed);
        if (smem > 40 * 1024) allow_dyn_smem(kernel, kForwardBytes);
        ScopedKernel prof("distill_forward", stream);
        kernel<<<(unsigned)div_up64(nodes, rows), kCta<G>, smem, stream>>>(a, words, logits, rest, costs, saved,
                                                                         K, scale2);
        TB200_CHECK_LAUNCH();
      };
      // a warp per node where there are warps enough to fill the chip
      if (a.V <= 1024 || nodes >= 148 * 16) launch(std::integral_constant<int, 32>{});
      else launch(std::integral_constant<int, 256>{});
    });
  });
}

}  // namespace tb200
