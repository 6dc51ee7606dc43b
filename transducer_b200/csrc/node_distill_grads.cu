// Gradients of the distillation costs (node_distill.cu has the formulas): sums over the nodes on each
// frame, and on each position, of w (p_v - q_v) for listed words and w sign 2^(x - A) for the others.
//
// A warp has a tile of 32 * COLS words and goes through nodes in their order, so that sums have the same
// bits from run to run.  Two ways:
// Where an utterance's nodes are a path (neither frames nor positions go back from one to the next; a
// device flag says so) the rows of E and P that are in use, and the sums for both, stay in registers:
// everything is read once and written once.  The frames are cut into segments to fill the chip; a
// position whose nodes lie in several segments is added up from partial rows by a second kernel.
// Otherwise each row of either gradient has a warp per tile that looks for its nodes between the first
// and the last one, and reads the other side's rows again for each; where there are few rows, their nodes
// are shared out to several warps, and joined in the same way.
#include <algorithm>

#include "node_rows.cuh"
#include "profile.h"

namespace tb200 {
namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kWarps = 8;         // per CTA
constexpr int kTarget = 148 * 24;  // warps that fill the chip
constexpr int kLookBack = 64;      // places without a node that a path may have between two nodes

struct GradArgs {
  const int* words;
  DistillSaved saved;
  const float* weights;
  void *egrads, *pgrads;   // either may be null
  int K;
  float scale, scale2;
  int2* spans;        // of the B * T frames, then the B * U positions: (N - first node, last node + 1), or 0
  int* offPath;       // [B] 1: the nodes are not a path
  int* segUsed;       // [B, segs] 1: a segment has nodes
  float* partial;     // of paths [B, segs, 2, V], or of other nodes [splits, rows, V] of E, then of P
  int segFrames, segs, tiles, eSplits, pSplits;
};

__global__ void __launch_bounds__(256) node_spans_kernel(NodeArgs a, GradArgs k) {
  const i64 node = (i64)blockIdx.x * 256 + threadIdx.x;
  if (node >= (i64)a.B * a.N) return;
  auto valid = [&](i64 i) {
    return (unsigned)a.frames[i] < (unsigned)a.T && (unsigned)a.positions[i] < (unsigned)a.U;
  };
  if (!valid(node)) return;
  const int t = a.frames[node], u = a.positions[node];
  const i64 b = node / a.N;
  const int n = (int)(node - b * a.N);
  int2* f = k.spans + b * a.T + t;
  int2* p = k.spans + (i64)a.B * a.T + b * a.U + u;
  atomicMax(&f->x, a.N - n);
  atomicMax(&f->y, n + 1);
  atomicMax(&p->x, a.N - n);
  atomicMax(&p->y, n + 1);
  k.segUsed[b * k.segs + t / k.segFrames] = 1;
  int back = 1;
  while (back <= n && back <= kLookBack && !valid(node - back)) ++back;
  if (back > n) return;
  if (back > kLookBack || a.frames[node - back] > t || a.positions[node - back] > u) k.offPath[b] = 1;
}

// A warp's tile: 32 * COLS words in vectors of VEC, lane by lane.
template <typename TIn, int VEC, int COLS>
struct Tile {
  static constexpr int NV = COLS / VEC;
  int first, V, lane;
  __device__ __forceinline__ int word(int j) const { return first + (j * 32 + lane) * VEC; }
  __device__ __forceinline__ void load(const TIn* row, float (&x)[COLS]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Words<VEC> q;
#pragma unroll
      for (int i = 0; i < VEC; ++i) q.x[i] = 0.0f;
      if (word(j) < V) q = load_words<VEC>(row + word(j));
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[j * VEC + i] = q.x[i];
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&x)[COLS]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (word(j) < V) {
        if constexpr (std::is_same<T, TIn>::value) {
          store_words<VEC>(row + word(j), x + j * VEC);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) row[word(j) + i] = x[j * VEC + i];
        }
      }
  }
};

// The listed words' shares are subtracted in shared memory (`sub`, a number per word of the tile in the order
// of memory), by the lanes that read the record, and join the sums when a row is finished.
template <int VEC, int COLS>
__device__ __forceinline__ void take_shares(float* sub, int lane, float (&acc)[COLS]) {
#pragma unroll
  for (int j = 0; j < COLS / VEC; ++j) {
    float* p = sub + (j * 32 + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      acc[j * VEC + i] += p[i];
      p[i] = 0.0f;
    }
  }
  __syncwarp();
}

// sums += the node's gradients, for one or both sides.
template <int VEC, int COLS, bool REST, bool BOTH>
__device__ __forceinline__ void add_node(const float (&e)[COLS], const float (&p)[COLS], float4 of, float w,
                                         float scale2, unsigned listed, float (&accA)[COLS], float (&accB)[COLS]) {
  const float ws = w * of.w;
#pragma unroll
  for (int i = 0; i < COLS; ++i) {
    const float z = e[i] + p[i] - of.x;
    float g;
    if constexpr (REST) {
      const bool in = listed >> i & 1;
      g = (in ? w : ws) * ex2(fmaf(z, scale2, in ? -of.y : -of.z));
    } else {
      g = w * ex2(fmaf(z, scale2, -of.y));
    }
    accA[i] += g;
    if constexpr (BOTH) accB[i] += g;
  }
}

// The listed words of a node that lie in the tile: subtracted from subA (and subB), marked in `marks`.
template <int VEC, int COLS, bool REST, bool BOTH>
__device__ __forceinline__ unsigned add_record(const GradArgs& k, i64 node, float w, int tileFirst, int lane,
                                               float* subA, float* subB, unsigned* marks) {
  bool any = false;
  for (int k0 = 0; k0 < k.K; k0 += 32) {
    int v = -1;
    float q = -1.0f;
    if (k0 + lane < k.K) {
      v = k.words[node * k.K + k0 + lane] - tileFirst;
      q = k.saved.q[node * k.K + k0 + lane];
    }
    const bool hit = (unsigned)v < (unsigned)(32 * COLS) && !(q < 0.0f);
    if (hit) {
      subA[v] -= w * q;
      if (BOTH) subB[v] -= w * q;
      if (REST) atomicOr(&marks[v / VEC % 32], 1u << (v / (32 * VEC) * VEC + v % VEC));
    }
    any |= hit;
  }
  unsigned mine = 0;
  if (REST && __any_sync(0xffffffffu, any)) {
    __syncwarp();
    mine = marks[lane];
    marks[lane] = 0;
  }
  __syncwarp();
  return mine;
}

template <typename TIn, int VEC, int COLS, bool REST>
__global__ void __launch_bounds__(kWarps * 32) distill_path_kernel(NodeArgs a, GradArgs k) {
  __shared__ __align__(16) float subAll[kWarps][2][32 * COLS];
  __shared__ unsigned marksAll[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float *subE = subAll[warp][0], *subP = subAll[warp][1];
  unsigned* marks = marksAll[warp];
  const i64 task = (i64)blockIdx.x * kWarps + warp;
  const i64 bs = task / k.tiles;
  const int b = (int)(bs / k.segs), seg = (int)(bs - (i64)b * k.segs);
  if (b >= a.B || k.offPath[b]) return;
  for (int i = lane; i < 32 * COLS; i += 32) subE[i] = subP[i] = 0.0f;
  marks[lane] = 0;
  __syncwarp();
  const Tile<TIn, VEC, COLS> tile{(int)(task - bs * k.tiles) * 32 * COLS, a.V, lane};
  const int t0 = seg * k.segFrames, t1 = min(t0 + k.segFrames, a.T);
  const TIn* E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
  const TIn* P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
  TIn* dE = k.egrads ? static_cast<TIn*>(k.egrads) + (i64)b * a.T * a.V : nullptr;
  TIn* dP = k.pgrads ? static_cast<TIn*>(k.pgrads) + (i64)b * a.U * a.V : nullptr;
  const int2* frameSpans = k.spans + (i64)b * a.T;
  const int2* posSpans = k.spans + (i64)a.B * a.T + (i64)b * a.U;
  const int* frames = a.frames + (i64)b * a.N;
  const int* positions = a.positions + (i64)b * a.N;
  // the segment's nodes
  int n0 = 0x7fffffff, n1 = 0;
  for (int t = t0 + lane; t < t1; t += 32) {
    const int2 s = frameSpans[t];
    if (s.y > 0) n0 = min(n0, a.N - s.x), n1 = max(n1, s.y);
  }
  n0 = __reduce_min_sync(0xffffffffu, n0);
  n1 = __reduce_max_sync(0xffffffffu, n1);
  float e[COLS], p[COLS], accE[COLS], accP[COLS];
#pragma unroll
  for (int i = 0; i < COLS; ++i) accE[i] = accP[i] = 0.0f;
  int curT = -1, curU = -1, nextRow = t0;   // frames below nextRow are written
  auto finish_frame = [&] {   // writes the current frame, and zeros for those before it that have no nodes
    take_shares<VEC>(subE, lane, accE);
    if (dE) tile.store(dE + (i64)curT * a.V, accE);
#pragma unroll
    for (int i = 0; i < COLS; ++i) accE[i] = 0.0f;
    nextRow = curT + 1;
  };
  auto zeros_to = [&](int t) {
    float zero[COLS];
#pragma unroll
    for (int i = 0; i < COLS; ++i) zero[i] = 0.0f;
    for (; nextRow < t; ++nextRow)
      if (dE) tile.store(dE + (i64)nextRow * a.V, zero);
  };
  auto finish_position = [&] {
    take_shares<VEC>(subP, lane, accP);
    if (dP) {
      const int2 s = posSpans[curU];
      const int from = frames[a.N - s.x] / k.segFrames, to = frames[s.y - 1] / k.segFrames;
      if (from == to) tile.store(dP + (i64)curU * a.V, accP);
      else tile.store(k.partial + (((i64)b * k.segs + seg) * 2 + (from == seg ? 1 : 0)) * a.V, accP);
    }
#pragma unroll
    for (int i = 0; i < COLS; ++i) accP[i] = 0.0f;
  };
  for (int nb = n0; nb < n1; nb += 32) {
    const int n = nb + lane;
    int t = -1, u = -1;
    float4 of = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float w = 0.0f;
    if (n < n1) {
      t = frames[n], u = positions[n];
      if ((unsigned)t >= (unsigned)a.T || (unsigned)u >= (unsigned)a.U) t = -1;
      of = k.saved.node[(i64)b * a.N + n];
      w = k.weights[(i64)b * a.N + n] * k.scale;
    }
    unsigned todo = __ballot_sync(0xffffffffu, t >= 0);
    while (todo) {
      const int bit = __ffs(todo) - 1;
      todo &= todo - 1;
      const int nt = __shfl_sync(0xffffffffu, t, bit), nu = __shfl_sync(0xffffffffu, u, bit);
      if (nt != curT) {
        if (curT >= 0) finish_frame();
        zeros_to(nt);
        curT = nt;
        tile.load(E + nt * a.eStrideT, e);
      }
      if (nu != curU) {
        if (curU >= 0) finish_position();
        curU = nu;
        tile.load(P + nu * a.pStrideU, p);
      }
      float4 f;
      f.x = __shfl_sync(0xffffffffu, of.x, bit);
      f.y = __shfl_sync(0xffffffffu, of.y, bit);
      f.z = __shfl_sync(0xffffffffu, of.z, bit);
      f.w = __shfl_sync(0xffffffffu, of.w, bit);
      const float fw = __shfl_sync(0xffffffffu, w, bit);
      const unsigned listed =
          add_record<VEC, COLS, REST, true>(k, (i64)b * a.N + nb + bit, fw, tile.first, lane, subE, subP, marks);
      add_node<VEC, COLS, REST, true>(e, p, f, fw, k.scale2, listed, accE, accP);
    }
  }
  if (curT >= 0) finish_frame();
  zeros_to(t1);
  if (curU >= 0) finish_position();
}

// Rows of either gradient of utterances whose nodes are not a path.  Tasks: (row, split, tile) of E, then of P.
template <typename TIn, int VEC, int COLS, bool REST>
__global__ void __launch_bounds__(kWarps * 32) distill_rows_kernel(NodeArgs a, GradArgs k) {
  __shared__ __align__(16) float subAll[kWarps][32 * COLS];
  __shared__ unsigned marksAll[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* sub = subAll[warp];
  unsigned* marks = marksAll[warp];
  for (int i = lane; i < 32 * COLS; i += 32) sub[i] = 0.0f;
  marks[lane] = 0;
  __syncwarp();
  const i64 ePer = (i64)a.T * k.eSplits * k.tiles, pPer = (i64)a.U * k.pSplits * k.tiles;   // tasks of an utterance
  const i64 step = (i64)gridDim.x * kWarps;
  for (int b = 0; b < a.B; ++b) {
    if (!k.offPath[b]) continue;
    for (i64 task = (i64)blockIdx.x * kWarps + warp; task < ePer + pPer; task += step) {
      const bool ofFrames = task < ePer;
      if ((ofFrames ? k.egrads : k.pgrads) == nullptr) continue;
      const i64 r = ofFrames ? task : task - ePer;
      const int splits = ofFrames ? k.eSplits : k.pSplits;
      const int own = (int)(r / (splits * k.tiles)), rem = (int)(r - (i64)own * splits * k.tiles);
      const int split = rem / k.tiles;
      const Tile<TIn, VEC, COLS> tile{(rem - split * k.tiles) * 32 * COLS, a.V, lane};
      const TIn* E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
      const TIn* P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
      const int2 span = k.spans[ofFrames ? (i64)b * a.T + own : (i64)a.B * a.T + (i64)b * a.U + own];
      const int* ownIdx = (ofFrames ? a.frames : a.positions) + (i64)b * a.N;
      const int* otherIdx = (ofFrames ? a.positions : a.frames) + (i64)b * a.N;
      const unsigned others = ofFrames ? a.U : a.T;
      const TIn* otherRows = ofFrames ? P : E;
      const i64 otherStride = ofFrames ? a.pStrideU : a.eStrideT;
      float mine[COLS], acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
      const int first = a.N - span.x, count = span.y > 0 ? span.y - first : 0;
      const int n0 = first + (int)((i64)count * split / splits), n1 = first + (int)((i64)count * (split + 1) / splits);
      if (n0 < n1) tile.load(ofFrames ? E + own * a.eStrideT : P + own * a.pStrideU, mine);
      for (int nb = n0; nb < n1; nb += 32) {
        const int n = nb + lane;
        int o = -1;
        float4 of = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float w = 0.0f;
        if (n < n1 && ownIdx[n] == own) {
          o = otherIdx[n];
          of = k.saved.node[(i64)b * a.N + n];
          w = k.weights[(i64)b * a.N + n] * k.scale;
        }
        unsigned todo = __ballot_sync(0xffffffffu, (unsigned)o < others);
        while (todo) {
          const int bit = __ffs(todo) - 1;
          todo &= todo - 1;
          float theirs[COLS];
          tile.load(otherRows + __shfl_sync(0xffffffffu, o, bit) * otherStride, theirs);
          float4 f;
          f.x = __shfl_sync(0xffffffffu, of.x, bit);
          f.y = __shfl_sync(0xffffffffu, of.y, bit);
          f.z = __shfl_sync(0xffffffffu, of.z, bit);
          f.w = __shfl_sync(0xffffffffu, of.w, bit);
          const float fw = __shfl_sync(0xffffffffu, w, bit);
          const unsigned listed =
              add_record<VEC, COLS, REST, false>(k, (i64)b * a.N + nb + bit, fw, tile.first, lane, sub, sub, marks);
          add_node<VEC, COLS, REST, false>(mine, theirs, f, fw, k.scale2, listed, acc, acc);
        }
      }
      take_shares<VEC>(sub, lane, acc);
      const i64 row = ofFrames ? (i64)b * a.T + own : (i64)b * a.U + own;
      if (splits == 1) {
        tile.store(static_cast<TIn*>(ofFrames ? k.egrads : k.pgrads) + row * a.V, acc);
      } else {
        const i64 rows = (i64)a.B * (ofFrames ? a.T : a.U);
        float* part = k.partial + (ofFrames || k.eSplits == 1 ? 0 : (i64)k.eSplits * a.B * a.T * a.V);
        tile.store(part + (split * rows + row) * a.V, acc);
      }
    }
  }
}

// Rows that are added up from partial ones, and rows of P without nodes on a path.  One CTA per row.
template <typename TIn>
__global__ void __launch_bounds__(256) distill_join_kernel(NodeArgs a, GradArgs k, int eRows) {
  i64 row = blockIdx.x;
  const bool ofFrames = row < eRows;
  if (!ofFrames) row -= eRows;
  const int per = ofFrames ? a.T : a.U;
  const int b = (int)(row / per);
  const float* part = k.partial;
  i64 stride = a.V;
  int count = 0;
  const int* used = nullptr;
  if (k.offPath[b]) {
    count = ofFrames ? k.eSplits : k.pSplits;
    if (count == 1) return;
    const i64 rows = (i64)a.B * per;
    if (!ofFrames && k.eSplits > 1) part += (i64)k.eSplits * a.B * a.T * a.V;
    part += row * a.V;
    stride = rows * a.V;
  } else {
    if (ofFrames) return;
    const int2 s = k.spans[(i64)a.B * a.T + row];
    if (s.y > 0) {
      const int* frames = a.frames + (i64)b * a.N;
      const int from = frames[a.N - s.x] / k.segFrames, to = frames[s.y - 1] / k.segFrames;
      if (from == to) return;
      // the part of the first segment is in its second place, the others' in their first
      part += (((i64)b * k.segs + from) * 2 + 1) * a.V;
      count = to - from + 1;
      used = k.segUsed + (i64)b * k.segs + from;
    }
  }
  TIn* out = static_cast<TIn*>(ofFrames ? k.egrads : k.pgrads) + row * a.V;
  for (int v = threadIdx.x; v < a.V; v += 256) {
    float sum = 0.0f;
    for (int c = 0; c < count; ++c) {
      if (used) {
        if (used[c]) sum += part[c == 0 ? v : (2 * c - 1) * stride + v];
      } else {
        sum += part[c * stride + v];
      }
    }
    from_f32(out[v], sum);
  }
}

constexpr int kCols = 16, kLeastFrames = 16, kLeastNodes = 8;

struct Plan {
  int tiles, segFrames, segs, eSplits, pSplits;
  size_t spanBytes;
};
Plan plan_of(int B, int T, int U, int V, int N) {
  Plan p{};
  p.tiles = div_up(V, 32 * kCols);
  // segments of at least 16 frames, as many as fill the chip
  const i64 want = std::max<i64>(1, kTarget / std::max<i64>(1, (i64)B * p.tiles));
  p.segFrames = (int)std::max<i64>(kLeastFrames, div_up64(std::max(T, 1), want));
  p.segs = div_up(std::max(T, 1), p.segFrames);
  auto splits = [&](int rows) {   // with 8 nodes of a row in the mean at least
    const i64 fill = kTarget / std::max<i64>(1, (i64)B * rows * p.tiles);
    return (int)std::max<i64>(1, std::min<i64>(fill, N / (kLeastNodes * std::max<i64>(1, rows))));
  };
  p.eSplits = splits(T);
  p.pSplits = splits(U);
  p.spanBytes = sizeof(int) * ((size_t)B * (2 * ((size_t)T + U) + 1 + p.segs));
  return p;
}
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

size_t distill_backward_workspace_bytes(int B, int T, int U, int V, int N) {
  if (B <= 0 || T < 0 || U < 0 || V <= 0 || N < 0) return 0;
  // Bounds on what the plan takes, so that no smaller call needs more than a larger one: the segments of all
  // utterances are max(B, kTarget / tiles) at most and a tile is 32 * kCols words; the splits of a side
  // fill kTarget tiles at most.
  const size_t leastSegs = div_up(std::max(T, 1), kLeastFrames), full = (size_t)kTarget * 32 * kCols;
  const size_t path = 2 * std::min(B * leastSegs * V, std::max((size_t)B * V, full));
  const size_t rows = 2 * std::min((size_t)N / kLeastNodes * B * V, full);
  return round256(sizeof(int) * ((size_t)B * (2 * ((size_t)T + U) + 1 + leastSegs))) +
         round256(sizeof(float) * std::max(path, rows));
}

void launch_distill_backward(const NodeArgs& a, const int* words, DistillSaved saved, const float* weights,
                             void* egrads, void* pgrads, int K, bool hasRest, double temperature,
                             void* workspace, cudaStream_t stream) {
  const i64 frameRows = egrads ? (i64)a.B * a.T : 0, posRows = pgrads ? (i64)a.B * a.U : 0, nodes = (i64)a.B * a.N;
  if (frameRows + posRows == 0) return;
  const Plan p = plan_of(a.B, a.T, a.U, a.V, a.N);
  GradArgs k{};
  k.words = words;
  k.saved = saved;
  k.weights = weights;
  k.egrads = frameRows ? egrads : nullptr;
  k.pgrads = posRows ? pgrads : nullptr;
  k.K = K;
  k.scale = (float)(1.0 / temperature);
  k.scale2 = (float)(1.4426950408889634 / temperature);
  k.spans = static_cast<int2*>(workspace);
  k.offPath = reinterpret_cast<int*>(k.spans + (i64)a.B * ((i64)a.T + a.U));
  k.segUsed = k.offPath + a.B;
  k.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(p.spanBytes));
  k.segFrames = p.segFrames;
  k.segs = p.segs;
  k.tiles = p.tiles;
  k.eSplits = p.eSplits;
  k.pSplits = p.pSplits;
  TB200_CUDA_CHECK(cudaMemsetAsync(workspace, 0, p.spanBytes, stream));
  if (nodes > 0) {
    ScopedKernel prof("node_spans", stream);
    node_spans_kernel<<<(unsigned)div_up64(nodes, 256), 256, 0, stream>>>(a, k);
    TB200_CHECK_LAUNCH();
  }
  const bool wide = node_rows_aligned(a) && reinterpret_cast<uintptr_t>(egrads) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(pgrads) % 16 == 0;
  auto run = [&](auto type, auto vec, auto rest) {
    using TIn = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool REST = decltype(rest)::value;
    {
      ScopedKernel prof("distill_path", stream);
      const i64 tasks = (i64)a.B * p.segs * p.tiles;
      distill_path_kernel<TIn, VEC, kCols, REST><<<(unsigned)div_up64(tasks, kWarps), kWarps * 32, 0, stream>>>(a, k);
      TB200_CHECK_LAUNCH();
    }
    if (nodes > 1) {   // (a single node is a path)
      ScopedKernel prof("distill_rows", stream);
      const i64 tasks = ((i64)a.T * p.eSplits + (i64)a.U * p.pSplits) * p.tiles;
      const i64 ctas = std::min<i64>(div_up64(tasks, kWarps), 148 * 6);
      distill_rows_kernel<TIn, VEC, kCols, REST><<<(unsigned)ctas, kWarps * 32, 0, stream>>>(a, k);
      TB200_CHECK_LAUNCH();
    }
    const i64 eRows = p.eSplits > 1 ? frameRows : 0;
    if (eRows + posRows > 0) {
      ScopedKernel prof("distill_join", stream);
      distill_join_kernel<TIn><<<(unsigned)(eRows + posRows), 256, 0, stream>>>(a, k, (int)eRows);
      TB200_CHECK_LAUNCH();
    }
  };
  auto with_rest = [&](auto type, auto vec) {
    if (hasRest) run(type, vec, std::true_type{});
    else run(type, vec, std::false_type{});
  };
  using std::integral_constant;
  if (a.dtype == kDtypeBf16) {
    if (wide) with_rest(bf16{}, integral_constant<int, 8>{});
    else with_rest(bf16{}, integral_constant<int, 1>{});
  } else {
    if (wide) with_rest(float{}, integral_constant<int, 4>{});
    else with_rest(float{}, integral_constant<int, 1>{});
  }
}

}  // namespace tb200
