// Gradients of the distillation costs (node_distill.cu has the formulas): sums over the nodes on each
// frame, and on each position, of w sign 2^(x - A), x = (z - m) log2e / temperature, less w share for
// listed words (DistillSaved).
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

constexpr int kWarps = 4;       // per CTA
constexpr int kPathWarps = 4;   // of the path kernel, at most
// Warps that a launch is cut into where it can be: six times the 16 that an SM holds, so that the last ones to
// finish leave little of the chip idle.
constexpr int kTarget = 148 * 96;

struct GradArgs {
  const int* words;
  DistillSaved saved;
  const float* weights;
  void *egrads, *pgrads;   // either may be null
  int K;
  float scale, scale2;
  float* partial;     // of paths [B, segs, 2, V]
  float* rowPartial;  // of other nodes [splits, rows, V] of E, then of P
  int tiles, eSplits, pSplits;
};

// A warp's tile: 32 * COLS words, vector j of a lane being the words (j * 32 + lane) * VEC and on.
template <typename TIn, int VEC, int COLS>
struct Tile {
  static constexpr int NV = COLS / VEC;
  using Row = RawWords<TIn, VEC>[NV];
  int first, V, lane;
  __device__ __forceinline__ int place(int j) const { return (j * 32 + lane) * VEC; }   // in the tile
  __device__ __forceinline__ bool in(int j) const { return first + place(j) < V; }
  __device__ __forceinline__ void load(const TIn* row, Row& x) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j].clear();
      if (in(j)) x[j].load(row + first + place(j));
    }
  }
  // to shared memory: each lane its own words
  __device__ __forceinline__ void fetch(const TIn* row, TIn* slot) const {
    if constexpr (VEC * sizeof(TIn) >= 4) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in(j)) copy_async<VEC * sizeof(TIn)>(slot + place(j), row + first + place(j));
    } else {   // (too small for an asynchronous copy: all on their way before the first is stored)
      Row x;
      load(row, x);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in(j)) slot[place(j)] = x[j].bits;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int j, const float* x) const {   // vector j
    if (!in(j)) return;
    row += first + place(j);
    if constexpr (std::is_same<T, TIn>::value) {
      store_words<VEC>(row, x);
    } else {   // fp32 sums of bf16 gradients
#pragma unroll
      for (int i = 0; i < VEC; i += VEC > 1 ? 4 : 1) store_words<(VEC > 1 ? 4 : 1)>(row + i, x + i);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&x)[COLS]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) store(row, j, x + j * VEC);
  }
};

// VEC floats of shared memory.
template <int VEC>
__device__ __forceinline__ void read_floats(const float* p, float (&x)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += VEC > 1 ? 4 : 1) {
    if constexpr (VEC > 1) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      x[i] = q.x, x[i + 1] = q.y, x[i + 2] = q.z, x[i + 3] = q.w;
    } else {
      x[i] = p[i];
    }
  }
}
template <int VEC>
__device__ __forceinline__ void write_floats(float* p, const float (&x)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += VEC > 1 ? 4 : 1) {
    if constexpr (VEC > 1) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    else p[i] = x[i];
  }
}

// What is saved of a node, made ready for its words' gradients.
struct Terms {
  float m, A, w, ws;   // ws: w with the others' sign
  bool apart;          // the listed words' gradients are their shares alone
  __device__ __forceinline__ static Terms of(float4 saved, float w) {
    return Terms{saved.x, saved.y, w, saved.z > 0.0f ? w : -w, fabsf(saved.z) > 1.5f};
  }
  // gradients of a vector but for the shares; bit i of `listed`: whether word i is
  template <int VEC>
  __device__ __forceinline__ void vector(Words<VEC> e, const Words<VEC>& p, unsigned listed, float scale2,
                                         float (&g)[VEC]) const {
    if (apart && listed) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (listed >> i & 1) e.x[i] = neg_inf();
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = ws * ex2(fmaf(e.x[i] + p.x[i] - m, scale2, -A));
  }
};

// The same for whole vectors with fewer operations: `weight` 2^(z scale2 - r), r next to m scale2 + A and the weight
// what is left of it, or, where gradients are rounded to 8 bits anyway, the weight in r too, and in `weight` its sign
// and what the rounding of r has left, 2^-15 at most (not where r is larger).  The sums take that with them: beside
// listed words they are differences, p - q, whose terms have to be good to 32 bits.  A gradient that is stored for
// itself goes without, its own rounding being 2^-9 to 2^-8 (where it belongs to a listed word it is replaced).
template <int VEC>
struct QuickTerms {
  static constexpr bool kFolded = VEC == 8;
  float r, weight;
  bool fits;
  __device__ __forceinline__ static QuickTerms of(const Terms& x, float scale2) {
    QuickTerms q;   // (apart: the listed words' gradients must not come by with the others')
    if constexpr (kFolded) {
      const double r = fma((double)x.m, (double)scale2, (double)x.A) - (double)log2f(fabsf(x.ws));
      q.r = (float)r;
      q.weight = copysignf(fabsf(q.r) < pos_inf() ? ex2((float)((double)q.r - r)) : 1.0f, x.ws);
      // (r = +inf: A says that there is no gradient, or the weight is 0)
      q.fits = fabsf(x.m * scale2) < 0x1p10f && (fabsf(q.r) < 0x1p10f || q.r == pos_inf());
    } else {
      q.r = rintf(fmaf(x.m, scale2, x.A));
      q.weight = x.ws * ex2(-(fmaf(x.m, scale2, -q.r) + x.A));
      q.fits = fabsf(q.r) < 0x1p24f;
    }
    q.fits = q.fits && !x.apart;
    return q;
  }
  // acc += gradients, and these in storage form to `row`
  template <typename T>
  __device__ __forceinline__ void vector(const Words<VEC>& e, const Words<VEC>& p, float scale2, float* acc,
                                         T* row) const {
    float g[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = ex2(fmaf(e.x[i] + p.x[i], scale2, -r));
      if constexpr (kFolded) {
        g[i] = x;
        acc[i] = fmaf(weight, x, acc[i]);
      } else {
        g[i] = weight * x;
        acc[i] += g[i];
      }
    }
    if (!row) return;
    if constexpr (kFolded) {
      unsigned u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(g[2 * i + 1]), "f"(g[2 * i]));
        u[i] ^= weight < 0.0f ? 0x80008000u : 0u;
      }
      *reinterpret_cast<uint4*>(row) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      store_words<VEC>(row, g);
    }
  }
};

// A node's number, and 32 words of its record, one in each lane.
struct Record {
  i64 at;   // of the record's first word among all
  int v;
  float2 listed;   // share, gradient
  __device__ __forceinline__ void load(const GradArgs& k, i64 at_, int from, int lane) {
    at = at_;
    v = -1;
    listed = make_float2(kNoShare, 0.0f);
    if (from + lane < k.K) {
      v = k.words[at + from + lane];
      listed = k.saved.listed[at + from + lane];
    }
  }
  // whether the lane's word is one of the tile's, and its place there
  template <int WORDS>
  __device__ __forceinline__ bool hits(int tileFirst, int& place) const {
    place = v - tileFirst;
    return v >= 0 && (unsigned)place < (unsigned)WORDS && listed.x != kNoShare;
  }
};

// The listed words of a node that lie in the tile: their shares are subtracted in shared memory, `subA` (and `subB`
// if there is one), by the lanes that read the record, and `marks` gets a bit for each word of a lane.
template <int VEC, int COLS>
__device__ __forceinline__ void add_record(const GradArgs& k, Record r, float w, int tileFirst, float* subA,
                                           float* subB, unsigned* marks, int lane) {
  for (int k0 = 0;;) {
    int at;
    if (r.hits<32 * COLS>(tileFirst, at)) {
      const float x = w * r.listed.x;
      subA[at] -= x;
      if (subB) subB[at] -= x;
      atomicOr(&marks[at / VEC % 32], 1u << (at / (32 * VEC) * VEC + at % VEC));
    }
    k0 += 32;
    if (k0 >= k.K) break;
    r.load(k, r.at, k0, lane);
  }
}

// A node as its CTA comes to it: all that can be known beforehand, made for 32 nodes at a time by a lane each.
template <int VEC>
struct Step {
  Terms terms;
  QuickTerms<VEC> quick;
  int flags, n, t, u;
  i64 target;   // of a new position: its row of dP, or -1 less its place among the partial rows
};
constexpr int kNewFrame = 1, kMoreOfFrame = 2, kNewPosition = 4;   // another than the node's before; not the last node
constexpr int kSteps = 64;    // in shared memory
constexpr int kCols = 16;     // words per lane
template <typename TIn>
constexpr int kAhead = sizeof(TIn) == 2 ? 3 : 2;   // rows of E that are on their way
template <typename TIn>
struct __align__(16) PathWarp {
  static constexpr int kRecords = kAhead<TIn> + 1;
  TIn rows[kAhead<TIn> + 1][32 * kCols];
  TIn nextP[32 * kCols];   // the row of P of the next new position
  float subE[32 * kCols], subP[32 * kCols];
  unsigned marks[32];
  int words[kRecords][32];   // of the records on their way, up to 32 words
  float2 listed[kRecords][32];
};
template <int VEC>
struct __align__(16) PathCta {
  Step<VEC> steps[kSteps];
  int appended, base, lastT, lastU;
};

// A warp's tile: rows of E and the nodes' records come through rings in shared memory, the row of P in use and the sums
// for it are in registers, a frame's gradients are written when its last node comes by and wait in `subE` until then.
// The warps of a CTA go along the same nodes.  Bound by latencies and issue: 16 warps an SM, 63 % of the issue slots, 360
// instructions for a node and tile, of which 8 for each of a lane's 16 words.  More warps spill registers, and next to
// this much shared memory the L1 does not hold them.  Records loaded one node ahead, into registers, were waited for at
// every node: 774 us against 571 for 58800 nodes of 10000 bf16 words (now 576, 4.2 TB/s of E and its gradients; at the copy
// rate 365); 8 utterances in fp32 224 us (5.2 TB/s).
template <typename TIn, int VEC>
__global__ void __launch_bounds__(kPathWarps * 32, 16 / kPathWarps)
    distill_path_kernel(NodeArgs a, GradArgs k) {
  constexpr int COLS = kCols, NV = COLS / VEC, kA = kAhead<TIn>;
  extern __shared__ __align__(16) unsigned char memory[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  PathCta<VEC>& cta = *reinterpret_cast<PathCta<VEC>*>(memory);
  PathWarp<TIn>& mem = reinterpret_cast<PathWarp<TIn>*>(memory + sizeof(PathCta<VEC>))[warp];
  const int groups = (k.tiles + warps - 1) / warps;   // of tiles
  const i64 bs = blockIdx.x / groups;
  const int b = (int)(bs / k.saved.segs), seg = (int)(bs - (i64)b * k.saved.segs);
  if (k.saved.offPath[b]) return;
  using T = Tile<TIn, VEC, COLS>;
  const T tile{((int)(blockIdx.x - bs * groups) * warps + warp) * 32 * COLS, a.V, lane};
  const int t0 = seg * k.saved.segFrames, t1 = min(t0 + k.saved.segFrames, a.T);
  const TIn* E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
  TIn* dE = k.egrads ? static_cast<TIn*>(k.egrads) + (i64)b * a.T * a.V : nullptr;
  // the segment's nodes
  int n0 = 0x7fffffff, n1 = 0;
  for (int tb = t0; tb < t1; tb += 32) {
    const int t = tb + lane;
    const int2 s = t < t1 ? k.saved.spans[(i64)b * a.T + t] : make_int2(0, 1);
    if (t < t1 && s.y > 0) n0 = min(n0, a.N - s.x), n1 = max(n1, s.y);
    const float zero[VEC] = {};   // for frames without nodes
    for (unsigned none = __ballot_sync(0xffffffffu, s.y == 0); dE && none; none &= none - 1)
#pragma unroll
      for (int j = 0; j < NV; ++j) tile.store(dE + (i64)(tb + __ffs(none) - 1) * a.V, j, zero);
  }
  n0 = __reduce_min_sync(0xffffffffu, n0);
  n1 = __reduce_max_sync(0xffffffffu, n1);
  if (n1 == 0) return;   // (the same for all warps)
  for (int i = lane; i < 32 * COLS; i += 32) mem.subE[i] = mem.subP[i] = 0.0f;
  mem.marks[lane] = 0;
  for (int i = 0; i <= kA; ++i) mem.words[i][lane] = -1;
  if (threadIdx.x == 0) cta.appended = 0, cta.base = n0, cta.lastT = cta.lastU = -1;
  auto append = [&] {   // the next 32 places with a node, by one warp
    int base = cta.base;
    const int appended = cta.appended, lastT = cta.lastT, lastU = cta.lastU;
    __syncwarp();
    unsigned all = 0;
    for (; !all && base < n1; base += 32) {
      Step<VEC> x;
      x.t = x.u = -1;
      x.n = base + lane;
      if (x.n < n1) {
        const i64 node = (i64)b * a.N + x.n;
        x.t = a.frames[node], x.u = a.positions[node];
        x.terms = Terms::of(k.saved.node[node], k.weights[node] * k.scale);
        x.quick = QuickTerms<VEC>::of(x.terms, k.scale2);
      }
      const bool here = (unsigned)x.t < (unsigned)a.T && (unsigned)x.u < (unsigned)a.U;
      all = __ballot_sync(0xffffffffu, here);
      const unsigned before = all & ((1u << lane) - 1), after = all & ~before & ~(1u << lane);
      const int tBefore = __shfl_sync(0xffffffffu, x.t, before ? 31 - __clz(before) : 0);
      const int uBefore = __shfl_sync(0xffffffffu, x.u, before ? 31 - __clz(before) : 0);
      const int tAfter = __shfl_sync(0xffffffffu, x.t, after ? __ffs(after) - 1 : 0);
      x.flags = (x.t != (before ? tBefore : lastT) ? kNewFrame : 0) |
                (x.u != (before ? uBefore : lastU) ? kNewPosition : 0) | (after && x.t == tAfter ? kMoreOfFrame : 0);
      if (here && (x.flags & kNewPosition) && k.pgrads) {
        const int2 s = k.saved.spans[(i64)a.B * a.T + (i64)b * a.U + x.u];
        const int* frames = a.frames + (i64)b * a.N;
        const int from = frames[a.N - s.x] / k.saved.segFrames, to = frames[s.y - 1] / k.saved.segFrames;
        x.target = from == to ? (i64)x.u * a.V : -1 - (((i64)b * k.saved.segs + seg) * 2 + (from == seg ? 1 : 0)) * a.V;
      }
      if (here) {
        cta.steps[(appended + __popc(before)) % kSteps] = x;
        if (!before && appended > 0 && x.t == lastT) cta.steps[(appended - 1) % kSteps].flags |= kMoreOfFrame;
        if (!after) cta.lastT = x.t, cta.lastU = x.u;
      }
    }
    if (lane == 0) cta.appended = appended + __popc(all), cta.base = base;
  };
  __syncthreads();
  if (warp == 0) append();
  __syncthreads();
  int appended = cta.appended;
  bool more = cta.base < n1;
  typename T::Row p;
  float accP[COLS];
#pragma unroll
  for (int i = 0; i < COLS; ++i) accP[i] = 0.0f;
  i64 target = 0;   // of the position in use
  auto finish_position = [&] {
    if (k.pgrads) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {   // the shares
        float s[VEC];
        const float zero[VEC] = {};
        read_floats<VEC>(mem.subP + tile.place(j), s);
        write_floats<VEC>(mem.subP + tile.place(j), zero);
#pragma unroll
        for (int i = 0; i < VEC; ++i) accP[j * VEC + i] += s[i];
      }
      if (target >= 0) tile.store(static_cast<TIn*>(k.pgrads) + (i64)b * a.U * a.V + target, accP);
      else tile.store(k.partial + (-1 - target), accP);
    }
#pragma unroll
    for (int i = 0; i < COLS; ++i) accP[i] = 0.0f;
  };
  int ringTo = 0, recordTo = 0;
  const i64 firstNode = (i64)b * a.N;
  const TIn* P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
  int stepP = -1;   // whose row of P is in nextP, or on its way there
  auto fetch_row = [&](int i) {   // of step i, if it is a new one, and the step's record; a group of copies per step
    if (i < appended) {
      const Step<VEC>& x = cta.steps[i % kSteps];
      if (lane < k.K) {
        const i64 at = (firstNode + x.n) * k.K + lane;
        copy_async<4>(&mem.words[recordTo][lane], k.words + at);
        copy_async<8>(&mem.listed[recordTo][lane], k.saved.listed + at);
      }
      recordTo = recordTo == kA ? 0 : recordTo + 1;
      if (x.flags & kNewFrame) {
        tile.fetch(E + x.t * a.eStrideT, mem.rows[ringTo]);
        ringTo = ringTo == kA ? 0 : ringTo + 1;
      }
      if ((x.flags & kNewPosition) && stepP < 0) {
        tile.fetch(P + x.u * a.pStrideU, mem.nextP);
        stepP = i;
      }
    }
    commit_copies();
  };
  int slot = kA, recordAt = 0;
  for (int i = 0; i < appended; ++i) {
    while (more && appended < i + kA + 2) {
      __syncthreads();   // (everybody is here: the steps before are free)
      if (warp == 0) append();
      __syncthreads();
      appended = cta.appended;
      more = cta.base < n1;
    }
    if (i == 0)
      for (int j = 0; j < kA; ++j) fetch_row(j);
    fetch_row(i + kA);
    wait_copies<kA>();
    const Step<VEC>& step = cta.steps[i % kSteps];
    const int flags = step.flags;
    const Record record{(firstNode + step.n) * k.K, mem.words[recordAt][lane], mem.listed[recordAt][lane]};
    recordAt = recordAt == kA ? 0 : recordAt + 1;
    if (flags & kNewPosition) {
      if (i > 0) finish_position();
      target = step.target;
      if (stepP == i) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          p[j].clear();
          if (tile.in(j)) p[j].load(mem.nextP + tile.place(j));
        }
        stepP = -1;
      } else {
        tile.load(P + step.u * a.pStrideU, p);
      }
    }
    if (flags & kNewFrame) slot = slot == kA ? 0 : slot + 1;
    const TIn* row = mem.rows[slot];
    TIn* out = dE + (i64)step.t * a.V;
    const bool whole = (flags & (kNewFrame | kMoreOfFrame)) == kNewFrame;   // the frame's only node
    if (whole && step.quick.fits) {
      const QuickTerms<VEC> quick = step.quick;
      const float weight = step.terms.w;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        RawWords<TIn, VEC> e;
        e.clear();
        if (tile.in(j)) e.load(row + tile.place(j));
        quick.vector(e.words(), p[j].words(), k.scale2, accP + j * VEC,
                     dE && tile.in(j) ? out + tile.first + tile.place(j) : nullptr);
      }
      __syncwarp();
      // the listed words' gradients take the place of what has been stored for them
      Record r = record;
      for (int k0 = 0;;) {
        int at;
        if (r.template hits<32 * COLS>(tile.first, at)) {
          if (dE) from_f32(out[tile.first + at], weight * r.listed.y);
          mem.subP[at] -= weight * r.listed.x;
        }
        k0 += 32;
        if (k0 >= k.K) break;
        r.load(k, r.at, k0, lane);
      }
      __syncwarp();
      continue;
    }
    const Terms terms = step.terms;
    add_record<VEC, COLS>(k, record, terms.w, tile.first, mem.subE, mem.subP, mem.marks, lane);
    __syncwarp();
    const unsigned listed = mem.marks[lane];
    if (listed) mem.marks[lane] = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!tile.in(j)) break;
      RawWords<TIn, VEC> e;
      e.load(row + tile.place(j));
      const unsigned here = listed >> (j * VEC) & ((1u << VEC) - 1);
      float g[VEC];
      terms.vector(e.words(), p[j].words(), here, k.scale2, g);
#pragma unroll
      for (int c = 0; c < VEC; ++c) accP[j * VEC + c] += g[c];
      if (!whole || here) {   // what waits there joins the gradient
        float s[VEC];
        float* sub = mem.subE + tile.place(j);
        read_floats<VEC>(sub, s);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          g[c] += s[c];
          s[c] = flags & kMoreOfFrame ? g[c] : 0.0f;
        }
        write_floats<VEC>(sub, s);
      }
      if (dE && !(flags & kMoreOfFrame)) tile.store(out, j, g);
    }
    __syncwarp();
  }
  finish_position();
}

// 32 places of an utterance's nodes in a warp's shared memory.
struct Batch {
  float4 of[32];     // DistillSaved::node
  float weight[32];
  int t[32], u[32];
  // lane by lane; places from `end` on have no node
  __device__ __forceinline__ void fetch(const NodeArgs& a, const GradArgs& k, int b, int base, int end, int lane) {
    const i64 node = (i64)b * a.N + base + lane;
    if (base + lane < end) {
      copy_async<16>(&of[lane], k.saved.node + node);
      copy_async<4>(&weight[lane], k.weights + node);
      copy_async<4>(&t[lane], a.frames + node);
      copy_async<4>(&u[lane], a.positions + node);
    } else {
      t[lane] = -1;
    }
  }
  __device__ __forceinline__ bool here(const NodeArgs& a, int lane) const {
    return (unsigned)t[lane] < (unsigned)a.T && (unsigned)u[lane] < (unsigned)a.U;
  }
};

// Rows of either gradient of utterances whose nodes are not a path.  Tasks of an utterance: (row, split, tile) of E, then
// of P.
// Bound by the latency of a node's record and row, one node ahead, and by instructions: the whole lattices of 4
// utterances, 5700 nodes of 512 words, take 19 us, of which reading both sides' rows for every node is 4 at the L2's
// rate.  Utterances lie side by side in the grid (one after another in every warp they took 37).
template <typename TIn, int VEC>
__global__ void __launch_bounds__(kWarps * 32, 4) distill_rows_kernel(NodeArgs a, GradArgs k) {
  constexpr int COLS = kCols, NV = COLS / VEC;
  __shared__ __align__(16) float subAll[kWarps][32 * COLS];
  __shared__ unsigned marksAll[kWarps][32];
  __shared__ Batch batchAll[kWarps][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* sub = subAll[warp];
  unsigned* marks = marksAll[warp];
  Batch* const batch = batchAll[warp];
  for (int i = lane; i < 32 * COLS; i += 32) sub[i] = 0.0f;
  marks[lane] = 0;
  __syncwarp();
  const i64 ePer = (i64)a.T * k.eSplits * k.tiles, pPer = (i64)a.U * k.pSplits * k.tiles;   // tasks of an utterance
  const i64 step = (i64)gridDim.x * kWarps;
  // the utterances of this row of the grid: blockIdx.y, blockIdx.y + gridDim.y and so on
  const int utterances = (a.B - 1 - (int)blockIdx.y) / (int)gridDim.y + 1;
  int b = 0, at = -1;   // and which of them b is
  unsigned off = 0;     // of the 32 that it is one of, those off a path that are left
  auto next_off_path = [&] {
    auto numbered = [&](int i) { return i * (int)gridDim.y + (int)blockIdx.y; };
    for (int from = off ? at : (at + 32) / 32 * 32; !off; from += 32) {
      if (from >= utterances) return false;
      off = __ballot_sync(0xffffffffu, from + lane < utterances && k.saved.offPath[numbered(from + lane)]);
      at = from;
    }
    at = at / 32 * 32 + __ffs(off) - 1;
    off &= off - 1;
    b = numbered(at);
    return true;
  };
  while (next_off_path()) {
    for (i64 task = (i64)blockIdx.x * kWarps + warp; task < ePer + pPer; task += step) {
      const bool ofFrames = task < ePer;
      if ((ofFrames ? k.egrads : k.pgrads) == nullptr) continue;
      const i64 r = ofFrames ? task : task - ePer;
      const int splits = ofFrames ? k.eSplits : k.pSplits;
      const int own = (int)(r / (splits * k.tiles)), rem = (int)(r - (i64)own * splits * k.tiles);
      const int split = rem / k.tiles;
      using T = Tile<TIn, VEC, COLS>;
      const T tile{(rem - split * k.tiles) * 32 * COLS, a.V, lane};
      const TIn* E = static_cast<const TIn*>(a.E) + b * a.eStrideB;
      const TIn* P = static_cast<const TIn*>(a.P) + b * a.pStrideB;
      const int2 span = k.saved.spans[ofFrames ? (i64)b * a.T + own : (i64)a.B * a.T + (i64)b * a.U + own];
      const TIn* otherRows = ofFrames ? P : E;
      const i64 otherStride = ofFrames ? a.pStrideU : a.eStrideT;
      typename T::Row mine, theirs, next;
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
      const int first = a.N - span.x, count = span.y > 0 ? span.y - first : 0;
      const int n0 = first + (int)((i64)count * split / splits), n1 = first + (int)((i64)count * (split + 1) / splits);
      if (n0 < n1) tile.load(ofFrames ? E + own * a.eStrideT : P + own * a.pStrideU, mine);
      // the next node's row and record are on their way while a node is added up
      Record record;
      auto fetch = [&](const Batch& x, int base, int at) {
        tile.load(otherRows + (ofFrames ? x.u[at] : x.t[at]) * otherStride, next);
        record.load(k, ((i64)b * a.N + base + at) * k.K, 0, lane);
      };
      auto advance = [&](Batch& x, int& base) {   // to the next 32 places from `base` on with a node of this row
        for (;; base += 32) {
          x.fetch(a, k, b, base, n1, lane);
          commit_copies();
          wait_copies<0>();
          __syncwarp();
          const unsigned some =
              __ballot_sync(0xffffffffu, x.here(a, lane) && (ofFrames ? x.t[lane] : x.u[lane]) == own);
          if (some || base + 32 >= n1) return some;
          __syncwarp();
        }
      };
      int now = 0, base = n0, baseThen;
      unsigned todo = n0 < n1 ? advance(batch[0], base) : 0, todoThen = 0;
      if (todo) fetch(batch[0], base, __ffs(todo) - 1);
      for (; todo; now ^= 1, base = baseThen, todo = todoThen) {
        const Batch& here = batch[now];
        Batch& then = batch[now ^ 1];
        baseThen = base + 32;
        todoThen = baseThen < n1 ? advance(then, baseThen) : 0;
        while (todo) {
          const int bit = __ffs(todo) - 1;
          todo &= todo - 1;
          const Record theirRecord = record;
#pragma unroll
          for (int j = 0; j < NV; ++j) theirs[j] = next[j];
          if (todo) fetch(here, base, __ffs(todo) - 1);
          else if (todoThen) fetch(then, baseThen, __ffs(todoThen) - 1);
          const Terms terms = Terms::of(here.of[bit], here.weight[bit] * k.scale);
          add_record<VEC, COLS>(k, theirRecord, terms.w, tile.first, sub, nullptr, marks, lane);
          __syncwarp();
          const unsigned listed = marks[lane];
          marks[lane] = 0;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            float g[VEC];
            terms.vector(theirs[j].words(), mine[j].words(), listed >> (j * VEC), k.scale2, g);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[j * VEC + i] += g[i];
          }
          __syncwarp();
        }
        __syncwarp();   // (everybody is done with `here`, which is filled next)
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NV; ++j) {   // the shares
        float s[VEC];
        const float zero[VEC] = {};
        read_floats<VEC>(sub + tile.place(j), s);
        write_floats<VEC>(sub + tile.place(j), zero);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[j * VEC + i] += s[i];
      }
      __syncwarp();
      const i64 row = ofFrames ? (i64)b * a.T + own : (i64)b * a.U + own;
      if (splits == 1) {
        tile.store(static_cast<TIn*>(ofFrames ? k.egrads : k.pgrads) + row * a.V, acc);
      } else {
        const i64 rows = (i64)a.B * (ofFrames ? a.T : a.U);
        float* part = k.rowPartial + (ofFrames || k.eSplits == 1 ? 0 : (i64)k.eSplits * a.B * a.T * a.V);
        tile.store(part + (split * rows + row) * a.V, acc);
      }
    }
  }
}

// Rows that are added up from partial ones, and rows of P without nodes on a path.  A warp looks at `group` rows
// (up to 32), one in each lane, and adds up 128 words of those that ask for it.
constexpr int kJoinWords = 128;
template <typename TIn>
__global__ void __launch_bounds__(kWarps * 32) distill_join_kernel(NodeArgs a, GradArgs k, int eRows, int rows,
                                                                   int group, int chunks) {
  const int lane = threadIdx.x & 31;
  const i64 task = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int first = (int)(task / chunks) * group, chunk = (int)(task - (task / chunks) * chunks);
  if (first >= rows) return;
  // this lane's row: where its partial rows are, and how many (-1: it is written already)
  int row = first + lane, count = -1;
  const bool ofFrames = row < eRows;
  if (!ofFrames) row -= eRows;
  i64 at = 0, stride = 0;   // of k.partial, or (of nodes off a path) of k.rowPartial
  int used = -1;            // first entry of segUsed
  if (lane < group && first + lane < rows) {
    const int per = ofFrames ? a.T : a.U;
    const int b = row / per;
    if (k.saved.offPath[b]) {
      const int splits = ofFrames ? k.eSplits : k.pSplits;
      if (splits > 1) {
        count = splits;
        at = (!ofFrames && k.eSplits > 1 ? (i64)k.eSplits * a.B * a.T : 0) + row;
        stride = (i64)a.B * per;
      }
    } else if (!ofFrames) {
      const int2 s = k.saved.spans[(i64)a.B * a.T + row];
      if (s.y == 0) {
        count = 0;
      } else {
        const int* frames = a.frames + (i64)b * a.N;
        const int from = frames[a.N - s.x] / k.saved.segFrames, to = frames[s.y - 1] / k.saved.segFrames;
        if (from != to) {   // the part of the first segment is in its second place, the others' in their first
          count = to - from + 1;
          used = b * k.saved.segs + from;
          at = (i64)used * 2;
          stride = 2;
        }
      }
    }
  }
  for (unsigned todo = __ballot_sync(0xffffffffu, count >= 0); todo; todo &= todo - 1) {
    const int i = __ffs(todo) - 1;
    const int n = __shfl_sync(0xffffffffu, count, i), u = __shfl_sync(0xffffffffu, used, i);
    const i64 from = __shfl_sync(0xffffffffu, at, i), step = __shfl_sync(0xffffffffu, stride, i);
    const bool e = __shfl_sync(0xffffffffu, ofFrames ? 1 : 0, i);
    const i64 to = __shfl_sync(0xffffffffu, row, i);
    const float* part = (u < 0 ? k.rowPartial : k.partial) + from * a.V;
    float sum[kJoinWords / 32] = {};
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      const float* p = part + (u >= 0 && c == 0 ? 1 : c * step) * a.V;
      const bool there = u < 0 || k.saved.segUsed[u + c];   // (a segment without nodes has left nothing)
#pragma unroll
      for (int j = 0; j < kJoinWords / 32; ++j) {
        const int v = chunk * kJoinWords + j * 32 + lane;
        if (v < a.V && there) sum[j] += p[v];
      }
    }
    TIn* out = static_cast<TIn*>(e ? k.egrads : k.pgrads) + to * a.V;
#pragma unroll
    for (int j = 0; j < kJoinWords / 32; ++j) {
      const int v = chunk * kJoinWords + j * 32 + lane;
      if (v < a.V) from_f32(out[v], sum[j]);
    }
  }
}

constexpr int kLeastFrames = 16, kLeastNodes = 8, kTileWords = 32 * kCols;

struct Plan {
  int tiles, segFrames, segs, eSplits, pSplits;
};
Plan plan_of(int B, int T, int U, int V, int N) {
  Plan p{};
  p.tiles = div_up(V, kTileWords);
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
  return p;
}
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
// Of the paths' partial rows: the segments of all utterances are max(B, kTarget / tiles) at most, and a
// tile is kTileWords words.  (A bound on what the plan takes, so that no smaller call needs more.)
size_t path_floats(int B, int T, int V) {
  const size_t leastSegs = div_up(std::max(T, 1), kLeastFrames);
  return 2 * std::min(B * leastSegs * V, std::max((size_t)B * V, (size_t)kTarget * kTileWords));
}

}  // namespace

size_t distill_saved_bytes(int B, int T, int U, int N, int K) {
  if (B <= 0 || T < 0 || U < 0 || N < 0 || K <= 0) return 0;
  const size_t nodes = (size_t)B * N, segs = div_up(std::max(T, 1), kLeastFrames);
  return round256(sizeof(float4) * nodes) + round256(sizeof(float2) * nodes * K) +
         round256(sizeof(int) * B * (2 * ((size_t)T + U) + 1 + segs));
}

DistillSaved distill_saved(void* p, int B, int T, int U, int V, int N, int K) {
  DistillSaved s{};
  if (!p) return s;
  const Plan plan = plan_of(B, T, U, V, N);
  const size_t nodes = (size_t)B * N;
  char* at = static_cast<char*>(p);
  s.node = reinterpret_cast<float4*>(at);
  s.listed = reinterpret_cast<float2*>(at += round256(sizeof(float4) * nodes));
  s.spans = reinterpret_cast<int2*>(at + round256(sizeof(float2) * nodes * K));
  s.offPath = reinterpret_cast<int*>(s.spans + (i64)B * ((i64)T + U));
  s.segUsed = s.offPath + B;
  s.segFrames = plan.segFrames;
  s.segs = plan.segs;
  return s;
}

size_t distill_backward_workspace_bytes(int B, int T, int U, int V, int N) {
  if (B <= 0 || T < 0 || U < 0 || V <= 0 || N < 0) return 0;
  // (the splits of a side fill kTarget tiles at most)
  const size_t rows = 2 * std::min((size_t)N / kLeastNodes * B * V, (size_t)kTarget * kTileWords);
  return round256(sizeof(float) * path_floats(B, T, V)) + round256(sizeof(float) * rows);
}

void launch_distill_backward(const NodeArgs& a, const int* words, DistillSaved saved, const float* weights,
                             void* egrads, void* pgrads, int K, double temperature,
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
  k.partial = static_cast<float*>(workspace);
  k.rowPartial = k.partial + round256(sizeof(float) * path_floats(a.B, a.T, a.V)) / sizeof(float);
  k.tiles = p.tiles;
  k.eSplits = p.eSplits;
  k.pSplits = p.pSplits;
  const bool wide = node_rows_aligned(a) && reinterpret_cast<uintptr_t>(egrads) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(pgrads) % 16 == 0;
  auto run = [&](auto type, auto vec) {
    using TIn = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    {
      ScopedKernel prof("distill_path", stream);
      int warps = kPathWarps;   // with the fewest that have no tile
      for (int w = kPathWarps - 1; w > 0; --w)
        if (div_up(p.tiles, w) * w < div_up(p.tiles, warps) * warps) warps = w;
      const int smem = (int)sizeof(PathCta<VEC>) + warps * (int)sizeof(PathWarp<TIn>);
      allow_dyn_smem(distill_path_kernel<TIn, VEC>,
                     (int)sizeof(PathCta<VEC>) + kPathWarps * (int)sizeof(PathWarp<TIn>));
      const i64 ctas = (i64)a.B * p.segs * div_up(p.tiles, warps);
      distill_path_kernel<TIn, VEC><<<(unsigned)ctas, warps * 32, smem, stream>>>(a, k);
      TB200_CHECK_LAUNCH();
    }
    if (nodes > 1) {   // (a single node is a path)
      ScopedKernel prof("distill_rows", stream);
      const i64 tasks = ((i64)a.T * p.eSplits + (i64)a.U * p.pSplits) * p.tiles;
      // an utterance's tasks along x, and as many utterances side by side as fill the chip
      const i64 most = 148 * 6, x = std::min<i64>(div_up64(tasks, kWarps), most);
      const dim3 grid((unsigned)x, (unsigned)std::min<i64>(a.B, div_up64(most, x)));
      distill_rows_kernel<TIn, VEC><<<grid, kWarps * 32, 0, stream>>>(a, k);
      TB200_CHECK_LAUNCH();
    }
    const i64 eRows = p.eSplits > 1 ? frameRows : 0;
    if (eRows + posRows > 0) {
      ScopedKernel prof("distill_join", stream);
      const i64 rows = eRows + posRows, chunks = div_up(a.V, kJoinWords);
      const i64 group = std::min<i64>(32, std::max<i64>(1, rows * chunks / 8192));
      distill_join_kernel<TIn><<<(unsigned)div_up64(div_up64(rows, group) * chunks, kWarps), kWarps * 32, 0, stream>>>(
          a, k, (int)eRows, (int)rows, (int)group, (int)chunks);
      TB200_CHECK_LAUNCH();
    }
  };
  with_type(a.dtype, wide, run);
}

}  // namespace tb200
