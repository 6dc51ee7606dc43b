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

// Where the nodes of each frame and each position lie among the N of their utterance: spans[row] =
// (N - first, last + 1) for the B*T frames, then the B*U positions; zeros where there is none.
__global__ void __launch_bounds__(256) node_spans_kernel(NodeArgs a, int2* __restrict__ spans) {
  const i64 node = (i64)blockIdx.x * 256 + threadIdx.x;
  if (node >= (i64)a.B * a.N) return;
  const int t = a.frames[node], u = a.positions[node];
  if ((unsigned)t >= (unsigned)a.T || (unsigned)u >= (unsigned)a.U) return;
  const i64 b = node / a.N;
  const int n = (int)(node - b * a.N);
  int2* f = spans + b * a.T + t;
  int2* p = spans + (i64)a.B * a.T + b * a.U + u;
  atomicMax(&f->x, a.N - n);
  atomicMax(&f->y, n + 1);
  atomicMax(&p->x, a.N - n);
  atomicMax(&p->y, n + 1);
}

// Gradients of the rows of E (FRAMES) or P: one warp per row and tile of 32 * VEC * NV words, which
// goes through the row's nodes in their order.
template <typename TIn, int VEC, int NV, bool REST, bool FRAMES>
__global__ void __launch_bounds__(256) distill_rows_kernel(NodeArgs a, const int* __restrict__ words,
                                                           DistillSaved saved,
                                                           const float* __restrict__ weights,
                                                           TIn* __restrict__ grads,
                                                           const int2* __restrict__ spans, int K, int tiles,
                                                           float scale, float scale2) {
  constexpr int kTile = 32 * VEC * NV, kOwn = VEC * NV;
  const int lane = threadIdx.x & 31;
  const i64 task = (i64)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int perUtt = FRAMES ? a.T : a.U;
  const i64 row = task / tiles;
  if (row >= (i64)a.B * perUtt) return;
  const int tile0 = (int)(task - row * tiles) * kTile;
  const i64 b = row / perUtt;
  const int own = (int)(row - b * perUtt);
  const TIn* E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
  const TIn* P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
  const TIn* mine = FRAMES ? E + own * a.eStrideT : P + own * a.pStrideU;
  float acc[kOwn], own_x[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) acc[i] = 0.0f, own_x[i] = 0.0f;
  const int2 span = spans[(FRAMES ? 0 : (i64)a.B * a.T) + row];
  const int* ownIdx = (FRAMES ? a.frames : a.positions) + b * a.N;
  const int* otherIdx = (FRAMES ? a.positions : a.frames) + b * a.N;
  const int others = FRAMES ? a.U : a.T;
  if (span.y > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = tile0 + (j * 32 + lane) * VEC;
      if (v < a.V) {
        const Words<VEC> x = load_words<VEC>(mine + v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) own_x[j * VEC + i] = x.x[i];
      }
    }
    for (int n0 = a.N - span.x; n0 < span.y; n0 += 32) {
      const int nl = n0 + lane;
      int other = -1;
      if (nl < span.y && ownIdx[nl] == own) other = otherIdx[nl];
      unsigned todo = __ballot_sync(0xffffffffu, (unsigned)other < (unsigned)others);
      while (todo) {
        const int bit = __ffs(todo) - 1;
        todo &= todo - 1;
        const i64 node = b * a.N + n0 + bit;
        const i64 o = __shfl_sync(0xffffffffu, other, bit);
        const TIn* theirs = FRAMES ? P + o * a.pStrideU : E + o * a.eStrideT;
        const float4 of = saved.node[node];
        const float w = weights[node] * scale;
        // the listed words of this tile: the teacher's shares are subtracted by the lanes that have them
        unsigned listed = 0;
        for (int k0 = 0; k0 < K; k0 += 32) {
          int v = -1;
          float q = -1.0f;
          if (k0 + lane < K) {
            v = words[node * K + k0 + lane] - tile0;
            q = saved.q[node * K + k0 + lane];
          }
          unsigned hits = __ballot_sync(0xffffffffu, (unsigned)v < (unsigned)kTile && !(q < 0.0f));
          while (hits) {
            const int k = __ffs(hits) - 1;
            hits &= hits - 1;
            const int at = __shfl_sync(0xffffffffu, v, k);
            const float share = w * __shfl_sync(0xffffffffu, q, k);
            if (at / VEC % 32 == lane) {
              const int slot = at / (32 * VEC) * VEC + at % VEC;
              listed |= 1u << slot;
#pragma unroll
              for (int i = 0; i < kOwn; ++i)
                if (i == slot) acc[i] -= share;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int v = tile0 + (j * 32 + lane) * VEC;
          if (v < a.V) {
            const Words<VEC> x = load_words<VEC>(theirs + v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float z = own_x[j * VEC + i] + x.x[i] - of.x;
              if constexpr (REST) {
                const bool in = listed >> (j * VEC + i) & 1;
                acc[j * VEC + i] += w * (in ? 1.0f : of.w) * ex2(fmaf(z, scale2, in ? -of.y : -of.z));
              } else {
                acc[j * VEC + i] += w * ex2(fmaf(z, scale2, -of.y));
              }
            }
          }
        }
      }
    }
  }
  grads += row * a.V;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = tile0 + (j * 32 + lane) * VEC;
    if (v < a.V) store_words<VEC>(grads + v, acc + j * VEC);
  }
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

void launch_distill_backward(const NodeArgs& a, const int* words, DistillSaved saved, const float* weights,
                             void* egrads, void* pgrads, int K, bool hasRest, double temperature, int* spans,
                             cudaStream_t stream) {
  const i64 frameRows = (i64)a.B * a.T, posRows = (i64)a.B * a.U, nodes = (i64)a.B * a.N;
  if (frameRows + posRows == 0) return;
  TB200_CUDA_CHECK(cudaMemsetAsync(spans, 0, sizeof(int2) * (frameRows + posRows), stream));
  int2* sp = reinterpret_cast<int2*>(spans);
  if (nodes > 0) {
    ScopedKernel prof("node_spans", stream);
    node_spans_kernel<<<(unsigned)div_up64(nodes, 256), 256, 0, stream>>>(a, sp);
    TB200_CHECK_LAUNCH();
  }
  const float scale = (float)(1.0 / temperature), scale2 = (float)(1.4426950408889634 / temperature);
  const bool wide = node_rows_aligned(a) && reinterpret_cast<uintptr_t>(egrads) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(pgrads) % 16 == 0;
  with_type(a.dtype, wide, [&](auto type, auto vec) {
    using TIn = decltype(type);
    with_flag(hasRest, [&](auto has_rest) {
      constexpr int VEC = vec, NV = 16 / VEC;
      const int tiles = div_up(a.V, 32 * VEC * NV);
      auto rows = [&](auto frames, i64 n, void* grads, const char* name) {
        if (n == 0 || grads == nullptr) return;
        ScopedKernel prof(name, stream);
        distill_rows_kernel<TIn, VEC, NV, has_rest, frames><<<(unsigned)div_up64(n * tiles, 8), 256, 0, stream>>>(
            a, words, saved, weights, static_cast<TIn*>(grads), sp, K, tiles, scale, scale2);
        TB200_CHECK_LAUNCH();
      };
      rows(std::true_type{}, frameRows, egrads, "distill_egrads");
      rows(std::false_type{}, posRows, pgrads, "distill_pgrads");
    });
  });
}

}  // namespace tb200
