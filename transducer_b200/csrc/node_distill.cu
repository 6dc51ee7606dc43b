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

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
#pragma unroll
    for (int i = 0; i < N; ++i) s += ex2((z[i] - m) * scale2);
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

constexpr int kWarpRows = 8;
template <int G>
constexpr int kCta = G == 32 ? 32 * kWarpRows : G;

// One group of G threads per node.  Dynamic shared memory: a bit per word and node, set for listed ones.
template <typename TIn, int VEC, int G, bool REST>
__global__ void __launch_bounds__(kCta<G>) distill_forward_kernel(
    NodeArgs a, const int* __restrict__ words, const float* __restrict__ logits,
    const float* __restrict__ rest, float* __restrict__ costs, DistillSaved saved, int K, float scale2) {
  constexpr int kRows = kCta<G> / G;
  extern __shared__ unsigned bits_all[];
  __shared__ double scratch[64];
  __shared__ int wordAll[kRows][kMaxListedWords];
  __shared__ float shareAll[kRows][kMaxListedWords];
  const int sub = threadIdx.x / G, tid = threadIdx.x % G;
  const i64 node = (i64)blockIdx.x * kRows + sub;
  if (node >= (i64)a.B * a.N) return;
  const NodeScores<TIn> s = node_scores<TIn>(a, node);
  int* word = wordAll[sub];
  float* share = shareAll[sub];
  words += node * K;
  logits += node * K;
  float* q = saved.q ? saved.q + node * K : nullptr;
  if (!s.here) {
    if (tid == 0) costs[node] = 0.0f;
    if (q) {
      for (int k = tid; k < K; k += G) q[k] = -1.0f;
      if (tid == 0) saved.node[node] = make_float4(0.0f, pos_inf(), pos_inf(), 1.0f);
    }
    return;
  }
  Group<G> g(tid, scratch);
  // the teacher's shares
  const float l_rest = REST ? rest[node] : neg_inf();
  float top = l_rest;
  for (int k = tid; k < K; k += G) {
    const int v = words[k];
    const bool there = (unsigned)v < (unsigned)a.V;
    const float l = there ? logits[k] : neg_inf();
    word[k] = there ? v : -1;
    share[k] = l;
    top = fmaxf(top, l);
  }
  unsigned* bits = bits_all;
  if constexpr (REST) {
    const int n = (a.V + 31) / 32;
    bits += sub * n;
    for (int i = tid; i < n; i += G) bits[i] = 0;
  }
  top = g.max(top);
  float sum = 0.0f;
  for (int k = tid; k < K; k += G) {
    share[k] = share[k] == neg_inf() ? 0.0f : expf(share[k] - top);
    sum += share[k];
  }
  float r = REST && l_rest != neg_inf() ? expf(l_rest - top) : 0.0f;
  sum = g.sum(sum) + r;
  g.sync();
  const bool empty = top == neg_inf();   // the record lists nothing: cost and gradient are 0
  const float one = empty ? 0.0f : 1.0f / sum;
  r *= one;
  // a word that is listed more than once: the first place has all its shares
  for (int k = tid; k < K; k += G) {
    const int v = word[k];
    float all = 0.0f;
    bool first = v >= 0;
    if (first)
      for (int j = 0; j < K; ++j)
        if (word[j] == v) {
          first = first && j >= k;
          all += share[j];
        }
    if (q) q[k] = first ? all * one : -1.0f;
    if constexpr (REST)
      if (first) atomicOr(&bits[v >> 5], 1u << (v & 31));
  }
  if constexpr (REST) g.sync();
  // the student's sums: of the words that are not listed (all words, without REST), and of all
  RunningSum others;
  for (int v = tid * VEC; v < a.V; v += G * VEC) {
    const Words<VEC> e = load_words<VEC>(s.e + v), p = load_words<VEC>(s.p + v);
    unsigned listed = 0;
    if constexpr (REST) listed = bits[v >> 5] >> (v & 31);
    float z[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      z[i] = e.x[i] + p.x[i];
      if constexpr (REST) z[i] = listed >> i & 1 ? neg_inf() : z[i];
    }
    others.add(z, scale2);
  }
  others.join(g, scale2);
  RunningSum all = others;
  if constexpr (REST) {
    RunningSum mine;
    for (int k = tid; k < K; k += G) {
      const int v = word[k];
      bool first = v >= 0;
      for (int j = 0; first && j < k; ++j) first = word[j] != v;
      const float z[1] = {first ? to_f32(s.e[v]) + to_f32(s.p[v]) : neg_inf()};
      mine.add(z, scale2);
    }
    mine.join(g, scale2);
    all.add(mine, scale2);
  }
  const float all2 = all.log2sum(all.m, scale2), other2 = others.log2sum(all.m, scale2);
  float cost = 0.0f;
  for (int k = tid; k < K; k += G) {
    const int v = word[k];
    float mass = 0.0f;
    bool first = v >= 0;
    if (first)
      for (int j = 0; j < K; ++j)
        if (word[j] == v) {
          first = first && j >= k;
          mass += share[j];
        }
    const float qk = mass * one;
    if (!first || qk == 0.0f) continue;
    const float z = to_f32(s.e[v]) + to_f32(s.p[v]);
    cost += qk * (logf(qk) - (z == neg_inf() ? z : ((z - all.m) * scale2 - all2) * kLn2));
  }
  cost = g.sum(cost);
  if (tid != 0) return;
  if (REST && r != 0.0f) cost += r * (logf(r) - (other2 == neg_inf() ? other2 : (other2 - all2) * kLn2));
  costs[node] = cost;
  if (!q) return;
  // (an empty record has no gradient, and a student without any word left has p = 0)
  const float L = empty || all2 == neg_inf() ? pos_inf() : all2;
  float A = L, sign = 1.0f;
  if (REST && r > 0.0f && other2 != neg_inf()) {
    const float d = logf(r) - (other2 - all2) * kLn2;   // log(r / rho)
    sign = d > 0.0f ? -1.0f : 1.0f;
    A = L - (fmaxf(d, 0.0f) + log1pf(-expf(-fabsf(d)))) * kLog2e;
  }
  saved.node[node] = make_float4(all.m, L, A, sign);
}

template <typename F>
void with_type(int dtype, bool wide, F launch) {
  if (dtype == kDtypeBf16) {
    if (wide) launch(bf16{}, std::integral_constant<int, 8>{});
    else launch(bf16{}, std::integral_constant<int, 1>{});
  } else {
    if (wide) launch(float{}, std::integral_constant<int, 4>{});
    else launch(float{}, std::integral_constant<int, 1>{});
  }
}
template <typename F>
void with_flag(bool on, F launch) {
  if (on) launch(std::true_type{});
  else launch(std::false_type{});
}

}  // namespace

void launch_distill_forward(const NodeArgs& a, const int* words, const float* logits, const float* rest,
                            float* costs, DistillSaved saved, int K, double temperature,
                            cudaStream_t stream) {
  const i64 nodes = (i64)a.B * a.N;
  if (nodes == 0) return;
  const float scale2 = (float)(1.4426950408889634 / temperature);
  with_type(a.dtype, node_rows_aligned(a), [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_flag(rest != nullptr, [&](auto has_rest) {
      auto launch = [&](auto group) {
        constexpr int G = group, rows = kCta<G> / G;
        auto kernel = distill_forward_kernel<TIn, vec, G, has_rest>;
        const int smem = has_rest ? rows * div_up(a.V, 32) * 4 : 0;
        if (smem > 48 * 1024) allow_dyn_smem(kernel, kDistillMaxBits / 8);
        ScopedKernel prof("distill_forward", stream);
        kernel<<<(unsigned)div_up64(nodes, rows), kCta<G>, smem, stream>>>(a, words, logits, rest, costs, saved,
                                                                         K, scale2);
        TB200_CHECK_LAUNCH();
      };
      if (a.V <= 1024) launch(std::integral_constant<int, 32>{});
      else if (a.V <= 4096) launch(std::integral_constant<int, 128>{});
      else launch(std::integral_constant<int, 256>{});
    });
  });
}

}  // namespace tb200
