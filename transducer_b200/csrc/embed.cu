// Rows of a table for words, scaled and with dropout, and the table's gradient.
//
// Row n is factor * table[words[n], h] where number (n, h) stays and 0 where it is dropped; which ones are is decided by
// 16 bits of Philox4x32-10 with counter (n, h / 8) and the seed as its key, eight numbers to a counter.  The bits are
// made again where they are needed: no mask is ever stored.  The gradient of row r adds up the gradients of the
// rows that are r's, in an order that follows from the words alone, in fp32: the words' places are sorted by word first,
// so that no sum needs atomics and the bits are the same from run to run.
//
// The bound is HBM without dropout.  With it no single unit is: of the 138 instructions (163 in the gradient's sums) that a warp
// executes per 256 numbers the generator needs 38 (18 products of 32 x 32 bits, 20 logical operations); issue slots are 71 % busy, the
// integer and the product pipe 63 to 64 %.  Rows of words that are none get their bits as well.  256 x 201 words, rows of 1024 bf16 numbers, a table of 32000: rows 22 us without dropout and 38 with it (105 MB
// written, 30 read: 21 us at the measured copy rate), the gradient's launches 12 + 30 + 4 and 12 + 46 + 4 (170 MB: 26 us).
#include <algorithm>

#include "kernels.h"
#include "node_rows.cuh"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kWarps = 8, kGroup = 8;   // numbers of one counter, all in one lane

struct Seed {
  unsigned low, high;
  __device__ __forceinline__ explicit Seed(const EmbedArgs& a) {
    const i64 s = a.seedAt ? *a.seedAt : a.seed;
    low = (unsigned)s, high = (unsigned)((unsigned long long)s >> 32);
  }
};

// Philox4x32-10 (Salmon, Moraes, Dror and Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) of several counters
// at once, which share the rounds' keys.
template <int K>
__device__ __forceinline__ void philox(uint4 (&c)[K], Seed key) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned long long a = (unsigned long long)c[k].x * 0xd2511f53u, b = (unsigned long long)c[k].z * 0xcd9e8d57u;
      c[k] = make_uint4((unsigned)(b >> 32) ^ c[k].y ^ key.low, (unsigned)b,
                        (unsigned)(a >> 32) ^ c[k].w ^ key.high, (unsigned)a);
    }
    key.low += 0x9e3779b9u, key.high += 0xbb67ae85u;
  }
}

// The numbers of a row that a lane of a warp has, of 256 that begin at `first`: vectors of 16 bytes, the lanes' side by
// side, where rows can be moved so, else every 32nd.
template <typename T, int VEC>
struct Numbers {
  static constexpr int kMoves = VEC == 1 ? kGroup : kGroup / VEC;
  RawWords<T, VEC> raw[kMoves];
  static __device__ __forceinline__ int at(int first, int lane, int move) {
    return first + 32 * VEC * move + VEC * lane;
  }
  __device__ __forceinline__ void load(const T* row, int first, int lane, int H) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      if (at(first, lane, i) < H) raw[i].load(row + at(first, lane, i));
      else raw[i].clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) raw[i].clear();
  }
  __device__ __forceinline__ void get(float (&x)[kGroup]) const {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const Words<VEC> w = raw[i].words();
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[VEC * i + j] = w.x[j];
    }
  }
  static __device__ __forceinline__ void store(T* row, int first, int lane, int H, const float (&x)[kGroup]) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      if (at(first, lane, i) < H) store_words<VEC>(row + at(first, lane, i), x + VEC * i);
  }
};

// Which of its numbers of a row a lane keeps: bits of the generator to be compared with 2^16 `dropped`, the
// number of row n and 256 that begin at `first`.  All lanes: each makes the bits of a whole counter.
template <int VEC>
struct Stays {
  uint4 bits;   // VEC < 8: bit i of x for number i
  __device__ __forceinline__ void get(bool (&stay)[kGroup], unsigned dropped) const {
    if constexpr (VEC < kGroup) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) stay[i] = bits.x >> i & 1;
    } else {
      const unsigned u[4] = {bits.x, bits.y, bits.z, bits.w}, least = dropped * 0x10001u;
#pragma unroll
      for (int i = 0; i < 4; ++i) __vibmax_u16x2(u[i], least, &stay[2 * i + 1], &stay[2 * i]);
    }
  }
};
template <int VEC, int K, typename N>
__device__ __forceinline__ void stays(Stays<VEC> (&out)[K], N place, int first, int lane, Seed seed, unsigned dropped) {
  uint4 c[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const unsigned long long n = place(k);
    c[k] = make_uint4((unsigned)n, (unsigned)(n >> 32), first / kGroup + lane, 0);
  }
  philox(c, seed);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (VEC < kGroup) {   // (the bits of a counter are several lanes')
      const Stays<kGroup> whole{c[k]};
      bool stay[kGroup];
      whole.get(stay, dropped);
      unsigned mine = 0, bits = 0;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) mine |= stay[i] ? 1u << i : 0u;
      constexpr int kLanes = kGroup / VEC;   // to a counter
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const unsigned theirs = __shfl_sync(0xffffffffu, mine, 32 / kLanes * i + lane / kLanes);
        bits |= (theirs >> lane % kLanes * VEC & ((1u << VEC) - 1)) << VEC * i;
      }
      out[k].bits.x = bits;
    } else {
      out[k].bits = c[k];
    }
  }
}

// A warp writes 256 numbers of each of ROWS rows that follow each other.
template <typename T, int VEC, bool DROP, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) embed_kernel(EmbedArgs a, T* __restrict__ rows, int* beyond) {
  const int lane = threadIdx.x & 31, first = blockIdx.y * 32 * kGroup;
  const i64 n0 = ((i64)blockIdx.x * kWarps + (threadIdx.x >> 5)) * ROWS;
  if (n0 >= a.N) return;
  int r[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) r[k] = n0 + k < a.N ? a.words[n0 + k] : -1;
  if (beyond) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (r[k] >= a.R) *beyond = 1;
  }
  Numbers<T, VEC> x[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k)
    if ((unsigned)r[k] < (unsigned)a.R) x[k].load(static_cast<const T*>(a.table) + r[k] * a.stride, first, lane, a.H);
    else x[k].clear();
  Stays<VEC> stay[ROWS];
  if constexpr (DROP)
    stays<VEC, ROWS>(stay, [&](int k) { return n0 + k; }, first, lane, Seed(a), a.dropped);
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (n0 + k >= a.N) break;
    float y[kGroup];
    bool keep[kGroup] = {true, true, true, true, true, true, true, true};
    x[k].get(y);
    if constexpr (DROP) stay[k].get(keep, a.dropped);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) y[i] = keep[i] ? y[i] * a.factor : 0.0f;
    Numbers<T, VEC>::store(rows + (n0 + k) * a.H, first, lane, a.H, y);
  }
}

// ---- the words' places in the order of the words ------------------------------------------------

constexpr int kSortRows = 256;   // of a CTA
// Words of a warp's that are its CTA's are listed; where there are more it looks again.
// (With room for 112 of them the most frequent words' CTA took 20 us instead of 14.)
constexpr int kSortListed = 1024;
template <int WARPS>
struct SortRoom {
  int count[WARPS][kSortRows];
  int total[kSortRows];
  int below;
  unsigned listed[WARPS][kSortListed];   // (place behind the warp's first, row of the CTA's)
};

// Words and their places, all of a word next to each other and in order.  Which word comes first does not matter.
struct Sorted {
  int2* order;   // (place, word), [N]
  int2* range;   // [R] where a row's begin and end; behind them how many there are in all
  int R;
  __device__ __forceinline__ int all() const { return range[R].x; }
};

// CTA c of 2^bits has the rows r with r mod 2^bits = c, so that frequent words that follow each other in the table are not
// all its own.  Every CTA goes through all words: it counts those of the CTAs before it, which tells where its own begin, and
// per warp those of each of its rows, which it lists; then every warp puts the places of its words where they belong.  One
// launch and no workspace but the result, for going through the words 128 times from L2: 51456 words take 10 us (uniform)
// to 14 (the n-th word 1 / n as frequent), 400000 words 45 to 130.
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) sort_words_kernel(const int* __restrict__ words, int N, int bits, Sorted out) {
  constexpr int kBatch = 16;   // words on their way at a time, per lane
  extern __shared__ __align__(16) char shared[];
  SortRoom<WARPS>& room = *reinterpret_cast<SortRoom<WARPS>*>(shared);
  auto& count = room.count;
  auto& total = room.total;
  auto& listed = room.listed;
  int& below = room.below;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, low = (1 << bits) - 1;
  cudaTriggerProgrammaticLaunchCompletion();
  for (int i = tid; i < WARPS * kSortRows; i += 32 * WARPS) (&count[0][0])[i] = 0;
  if (tid == 0) below = 0;
  __syncthreads();
  const int seg = (int)round_up64(div_up64(N, WARPS), 32);
  const int first = (int)min((i64)N, (i64)warp * seg), end = (int)min((i64)N, (i64)first + seg);
  // f(word or -1, place of the first) for the warp's words, 32 that follow each other at a time, in order
  auto each = [&](auto f) {
    int n = first;
#pragma unroll 1
    for (; end - n >= 32 * kBatch; n += 32 * kBatch) {
      int r[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) r[j] = words[n + 32 * j + lane];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) f(r[j], n + 32 * j);
    }
#pragma unroll 4
    for (int left = end - n; left > 0; left -= 32) {   // (n + 32 may pass 31 bits behind the last word)
      f(lane < left ? words[end - left + lane] : -1, end - left);
    }
  };
  const unsigned before = (1u << lane) - 1;
  int lower = 0, found = 0;
  each([&](int r, int n) {
    const bool is = (unsigned)r < (unsigned)out.R;
    lower += is && (r & low) < cta ? 1 : 0;
    const bool in = is && (r & low) == cta;
    const unsigned any = __ballot_sync(0xffffffffu, in);
    if (any == 0) return;
    if (in) {
      atomicAdd(&count[warp][r >> bits], 1);
      const int i = found + __popc(any & before);
      if (i < kSortListed) listed[warp][i] = (unsigned)(n + lane - first) << 8 | (unsigned)(r >> bits);
    }
    found += __popc(any);
  });
  lower = __reduce_add_sync(0xffffffffu, lower);
  if (lane == 0) atomicAdd(&below, lower);
  __syncthreads();
  int mine = 0;   // of row tid
  if (tid < kSortRows) {
#pragma unroll 8
    for (int w = 0; w < WARPS; ++w) {
      const int c = count[w][tid];
      count[w][tid] = mine;
      mine += c;
    }
    total[tid] = mine;
  }
  __syncthreads();
  if (warp == 0) {   // (the rows' sums to where each begins)
    int sum[kSortRows / 32], all = 0;
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) sum[i] = all, all += total[lane * (kSortRows / 32) + i];
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    upto += below - all;
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) total[lane * (kSortRows / 32) + i] = upto + sum[i];
    if (lane == 31 && cta == low) out.range[out.R] = make_int2(upto + all, 0);
  }
  __syncthreads();
  if (tid < kSortRows && ((i64)tid << bits) + cta < out.R)
    out.range[(tid << bits) + cta] = make_int2(total[tid], total[tid] + mine);
  int* const at = count[warp];
#pragma unroll
  for (int i = lane; i < kSortRows; i += 32) at[i] += total[i];
  __syncwarp();
  auto put = [&](int r, int n, bool in) {
    const unsigned any = __ballot_sync(0xffffffffu, in);
    if (!in) return;
    const unsigned same = __match_any_sync(any, r);
    const int rank = __popc(same & before);
    const int base = at[r >> bits];
    __syncwarp(any);
    out.order[base + rank] = make_int2(n, r);
    if (rank == 0) at[r >> bits] = base + __popc(same);
    __syncwarp(any);
  };
  if (found <= kSortListed && seg <= 1 << 24) {
#pragma unroll 1
    for (int i = 0; i < found; i += 32) {
      const unsigned x = i + lane < found ? listed[warp][i + lane] : 0;
      put((int)(x & 255) << bits | cta, first + (int)(x >> 8), i + lane < found);
    }
  } else {
    each([&](int r, int n) { put(r, (int)((unsigned)n + lane), (unsigned)r < (unsigned)out.R && (r & low) == cta); });
  }
}

// ---- the gradient -------------------------------------------------------------------------------

// An item is `part` places of the order that follow each other, a CTA's.  Rows that lie within one item are its sums; of the
// others every item leaves its share: slot 0 if it begins with the item or before it, else slot 1.
struct Parts {
  float* sums;   // [items, 2, pieces, 32 lanes, 8]
  int part, pieces;
  int items;
  __device__ __forceinline__ float4* at(int item, int slot, int piece, int lane) const {
    return reinterpret_cast<float4*>(sums + (((((i64)item * 2 + slot) * pieces + piece) * 32 + lane) * kGroup));
  }
};

// Adds up 256 numbers of the rows of `count` places that follow each other, at(i) the i-th place and its word; `before` and
// `behind` are the words next to them.  Rows that lie within are written to the gradient, the shares of others to
// part(slot): 0 where the row is the first, 1 where it is a later one.  Rows of vectors come through `ring`, the warp's shared
// memory, from which every lane reads what it has copied itself.
template <typename T, int VEC>
constexpr int kAddBatch = sizeof(T) == 2 && VEC > 1 ? 4 : 2;   // rows that are added at a time
template <typename T, int VEC, int BATCHES>
constexpr int kAddRing = VEC > 1 ? BATCHES * kAddBatch<T, VEC> * 32 * kGroup * (int)sizeof(T) : 0;   // bytes of a warp

template <typename T, int VEC, bool DROP, int BATCHES, typename At, typename Part>
__device__ __forceinline__ void add_places(const EmbedArgs& a, const T* deltas, int count, At at, int before, int behind,
                                           int first, int lane, T* grad, char* ring, Part part) {
  constexpr int kBatch = kAddBatch<T, VEC>, kMoves = Numbers<T, VEC>::kMoves;
  const Seed seed(a);
  float sum[kGroup] = {};
  int row = at(0).y;
  bool begins = true;   // the present row is the first
  auto finish = [&](bool ends) {   // `ends`: it is the last
    if (!(begins && row == before) && !(ends && row == behind)) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
      Numbers<T, VEC>::store(grad + (i64)row * a.H, first, lane, a.H, sum);
    } else {
      float4* p = part(begins ? 0 : 1, row);
      p[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
      p[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    }
  };
  Numbers<T, VEC> next[kBatch];   // (of single words: the next batch)
  auto place = [&](int i, int j) { return ring + ((i / kBatch % BATCHES * kBatch + j) * kMoves * 32 + lane) * 16; };
  auto bring = [&](int i) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const T* row = deltas + (i64)at(min(i + j, count - 1)).x * a.H;
      if (i + j >= count) break;
      if constexpr (VEC > 1) {
#pragma unroll
        for (int k = 0; k < kMoves; ++k)
          if (Numbers<T, VEC>::at(first, lane, k) < a.H)
            copy_async<16>(place(i, j) + 32 * 16 * k, row + Numbers<T, VEC>::at(first, lane, k));
      } else {
        next[j].load(row, first, lane, a.H);
      }
    }
    if constexpr (VEC > 1) commit_copies();
  };
  if constexpr (VEC > 1) {
#pragma unroll
    for (int k = 0; k < BATCHES - 1; ++k) bring(kBatch * k);
  } else {
    bring(0);
  }
#pragma unroll 1
  for (int i = 0; i < count; i += kBatch) {
    Numbers<T, VEC> x[kBatch];
    if constexpr (VEC > 1) {
      bring(i + kBatch * (BATCHES - 1));
      wait_copies<BATCHES - 1>();
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < kMoves; ++k) x[j].raw[k].load(reinterpret_cast<const T*>(place(i, j) + 32 * 16 * k));
    } else {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) x[j] = next[j];
      bring(i + kBatch);
    }
    Stays<VEC> stay[kBatch];
    if constexpr (DROP)
      stays<VEC, kBatch>(stay, [&](int k) { return at(min(i + k, count - 1)).x; }, first, lane, seed, a.dropped);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (i + j >= count) break;
      const int r = at(i + j).y;
      if (r != row) {
        finish(false);
#pragma unroll
        for (int k = 0; k < kGroup; ++k) sum[k] = 0.0f;
        row = r, begins = false;
      }
      float y[kGroup];
      bool keep[kGroup] = {true, true, true, true, true, true, true, true};
      x[j].get(y);
      if constexpr (DROP) stay[j].get(keep, a.dropped);
#pragma unroll
      for (int k = 0; k < kGroup; ++k)
        if (keep[k]) sum[k] += y[k];
    }
  }
  finish(true);
}

constexpr int kSumBatches = 3, kFilled = 8;   // kFilled: rows that a warp fills where no word has them

// CTAs (x, piece): the first sumCtas add up 256 numbers of an item's rows, an eighth of its places per warp; the others
// fill rows that no word has.
template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kWarps, 3) embed_sums_kernel(EmbedArgs a, const T* __restrict__ deltas, Sorted s,
                                                                 Parts parts, T* __restrict__ grad, int sumCtas) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  if (blockIdx.x >= sumCtas) {
    const i64 fill = ((i64)(blockIdx.x - sumCtas) * parts.pieces + blockIdx.y) * kWarps + warp;
    const i64 mine = fill * kFilled + lane;
    int2 range = make_int2(0, 1);
    if (lane < kFilled && mine < a.R) range = s.range[mine];
    unsigned empty = __ballot_sync(0xffffffffu, range.x == range.y);
    const float zero[kGroup] = {};
    for (; empty; empty &= empty - 1)
      for (int first = 0; first < a.H; first += 32 * kGroup)
        Numbers<T, VEC>::store(grad + (fill * kFilled + __ffs(empty) - 1) * a.H, first, lane, a.H, zero);
    return;
  }
  extern __shared__ __align__(16) char rings[];
  __shared__ float4 share[kWarps][2][32][2];   // what the warps leave, as the items do
  __shared__ int firstRow[kWarps], lastRow[kWarps];   // -1: the warp has no places
  const int item = blockIdx.x, piece = blockIdx.y, first = piece * 32 * kGroup, all = s.all(), own = parts.part / kWarps;
  if ((i64)item * parts.part >= all) return;
  const int end = (int)min((i64)(item + 1) * parts.part, (i64)all);   // of the item
  const int from = (int)min((i64)item * parts.part + warp * own, (i64)end), to = from + min(own, end - from);
  // lane i: the warp's place i
  const int2 mine = lane < to - from ? s.order[from + lane] : make_int2(0, -1);
  auto at = [&](int i) {
    return make_int2(__shfl_sync(0xffffffffu, mine.x, i & 31), __shfl_sync(0xffffffffu, mine.y, i & 31));
  };
  const int before = from > 0 ? s.order[from - 1].y : -1, behind = to < all ? s.order[to].y : -1;
  const int behindAll = end < all ? s.order[end].y : -1;
  const int begins = at(0).y, ends = at(to - from - 1).y;
  if (lane == 0) firstRow[warp] = from < to ? begins : -1, lastRow[warp] = from < to ? ends : -1;
  if (from < to)
    add_places<T, VEC, DROP, kSumBatches>(a, deltas, to - from, at, before, behind, first, lane, grad,
                                          rings + warp * kAddRing<T, VEC, kSumBatches>,
                                          [&](int slot, int) { return share[warp][slot][lane]; });
  __syncthreads();
  if (from >= to) return;
  // rows that the warp is the first of the item to have and has not written
  const bool single = begins == ends;
#pragma unroll 1
  for (int slot = 0; slot < 2; ++slot) {
    const int row = slot == 0 ? begins : ends;
    const bool onward = (slot == 1 || single) && ends == behind;
    if (slot == 0 ? !(begins == before || onward) || (warp > 0 && begins == before) : single || !onward) continue;
    float4 x = share[warp][slot][lane][0], y = share[warp][slot][lane][1];
    bool more = onward;   // the row goes on behind what has been added
    for (int w = warp + 1; more && w < kWarps && firstRow[w] >= 0; ++w) {
      const float4 u = share[w][0][lane][0], v = share[w][0][lane][1];
      x = make_float4(x.x + u.x, x.y + u.y, x.z + u.z, x.w + u.w);
      y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
      more = lastRow[w] == row && (w + 1 < kWarps && firstRow[w + 1] >= 0 ? firstRow[w + 1] : behindAll) == row;
    }
    const bool start = warp == 0 && slot == 0;
    if (more || (start && begins == before)) {
      float4* p = parts.at(item, start ? 0 : 1, piece, lane);
      p[0] = x, p[1] = y;
    } else {
      const float sum[kGroup] = {x.x * a.factor, x.y * a.factor, x.z * a.factor, x.w * a.factor,
                                 y.x * a.factor, y.y * a.factor, y.z * a.factor, y.w * a.factor};
      Numbers<T, VEC>::store(grad + (i64)row * a.H, first, lane, a.H, sum);
    }
  }
}

constexpr int kJoinWarps = 8;

// Rows that lie in several items, each by the warp (or, of many items, the CTA) that has the first of them.
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) embed_join_kernel(EmbedArgs a, Sorted s, Parts parts,
                                                                 T* __restrict__ grad) {
  constexpr int kMany = 16;   // items from which on the CTA adds them up together
  __shared__ float4 shares[kJoinWarps][32][2];
  struct Row {
    int row, slot;   // -1: none begins in the item
    int item, items;
  };
  __shared__ Row many[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, piece = blockIdx.y;
  cudaGridDependencySynchronize();
  auto row_of = [&](int item) {
    Row x{-1, 0, item, 0};
    const i64 last = (i64)item * parts.part + parts.part - 1;
    if (last >= s.all()) return x;
    const int r = s.order[last].y;
    const int2 range = s.range[r];
    x.items = (range.y - 1) / parts.part - item + 1;
    x.slot = range.x % parts.part == 0 ? 0 : 1;
    if (range.x / parts.part == item && x.items > 1) x.row = r;
    return x;
  };
  // the row's shares of its items [from, to)
  auto add = [&](const Row& row, int from, int to, float (&sum)[kGroup]) {
    constexpr int kBatch = 4;
#pragma unroll 1
    for (int i = from; i < to; i += kBatch) {
      float4 x[kBatch][2];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j < to) {
          const float4* p = parts.at(row.item + i + j, i + j == 0 ? row.slot : 0, piece, lane);
          x[j][0] = p[0], x[j][1] = p[1];
        }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j < to) {
          sum[0] += x[j][0].x, sum[1] += x[j][0].y, sum[2] += x[j][0].z, sum[3] += x[j][0].w;
          sum[4] += x[j][1].x, sum[5] += x[j][1].y, sum[6] += x[j][1].z, sum[7] += x[j][1].w;
        }
    }
  };
  auto write = [&](int r, float (&sum)[kGroup]) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
    Numbers<T, VEC>::store(grad + (i64)r * a.H, piece * 32 * kGroup, lane, a.H, sum);
  };
  const Row own = row_of(blockIdx.x * kJoinWarps + warp);
  if (lane == 0) many[warp] = own;
  if (own.row >= 0 && own.items < kMany) {
    float sum[kGroup] = {};
    add(own, 0, own.items, sum);
    write(own.row, sum);
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < kJoinWarps; ++w) {
    const Row row = many[w];
    if (row.row < 0 || row.items < kMany) continue;
    const int share = div_up(row.items, kJoinWarps);
    float sum[kGroup] = {};
    add(row, min(row.items, warp * share), min(row.items, (warp + 1) * share), sum);
    shares[warp][lane][0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    shares[warp][lane][1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    __syncthreads();
    if (warp == w) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) {
        const float4 x = shares[i][lane][0], y = shares[i][lane][1];
        sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
      }
      write(row.row, sum);
    }
    __syncthreads();
  }
}

// ---- few words: all in one launch ---------------------------------------------------------------

constexpr int kDirectWords = 4096, kDirectWarps = 8, kDirectBatches = 4;

struct DirectRoom {
  int count[kDirectWarps][kSortRows];
  int start[kSortRows + 1];
  unsigned order[kDirectWords];   // (place, row of the CTA's)
  float4 share[kDirectWarps][2][32][2];
};

// CTA (c, piece) of 2^bits has 256 numbers of the rows r with r mod 2^bits = c: it sorts its words as sort_words_kernel does,
// adds them up, an eighth of the places per warp, and joins what lies with several warps.
template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kDirectWarps, 2) embed_direct_kernel(EmbedArgs a, const T* __restrict__ deltas,
                                                                            T* __restrict__ grad, int bits) {
  constexpr int kOwn = kDirectWords / kDirectWarps / 32;   // words of a lane
  extern __shared__ __align__(16) char shared[];
  DirectRoom& room = *reinterpret_cast<DirectRoom*>(shared);
  char* const ring = shared + sizeof(DirectRoom);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, low = (1 << bits) - 1, first = blockIdx.y * 32 * kGroup, N = (int)a.N;
  const int seg = (div_up(N, kDirectWarps) + 31) / 32 * 32, from = warp * seg;
  int r[kOwn], rank[kOwn];
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const int i = 32 * j + lane;
    r[j] = i < seg && from + i < N ? a.words[from + i] : -1;
  }
  for (int i = tid; i < kDirectWarps * kSortRows; i += 32 * kDirectWarps) (&room.count[0][0])[i] = 0;
  __syncthreads();
  int* const count = room.count[warp];
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const bool in = (unsigned)r[j] < (unsigned)a.R && (r[j] & low) == cta;
    const unsigned any = __ballot_sync(0xffffffffu, in);
    rank[j] = -1;
    if (in) {
      const unsigned same = __match_any_sync(any, r[j]);
      const int base = count[r[j] >> bits];
      rank[j] = base + __popc(same & ((1u << lane) - 1));
      __syncwarp(any);
      if ((same & ((1u << lane) - 1)) == 0) count[r[j] >> bits] = base + __popc(same);
      __syncwarp(any);
    }
    __syncwarp();
  }
  __syncthreads();
  {   // (thread i: row i of the CTA's)
    int mine = 0;
#pragma unroll
    for (int w = 0; w < kDirectWarps; ++w) {
      const int c = room.count[w][tid];
      room.count[w][tid] = mine;
      mine += c;
    }
    room.start[tid] = mine;
  }
  __syncthreads();
  if (warp == 0) {
    int sum[kSortRows / 32], all = 0;
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) sum[i] = all, all += room.start[lane * (kSortRows / 32) + i];
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) room.start[lane * (kSortRows / 32) + i] = upto - all + sum[i];
    if (lane == 31) room.start[kSortRows] = upto;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kOwn; ++j)
    if (rank[j] >= 0) {
      const int row = r[j] >> bits;
      room.order[room.start[row] + count[row] + rank[j]] = (unsigned)row << 16 | (unsigned)(from + 32 * j + lane);
    }
  __syncthreads();
  const int all = room.start[kSortRows], part = div_up(all, kDirectWarps);
  const int begin = warp * part, end = min(all, begin + part);
  auto word = [&](int i) { return (int)(room.order[i] >> 16) << bits | cta; };
  if (begin < end) {
    auto at = [&](int i) { return make_int2((int)(room.order[begin + i] & 0xffffu), word(begin + i)); };
    add_places<T, VEC, DROP, kDirectBatches>(a, deltas, end - begin, at, begin > 0 ? word(begin - 1) : -1, end < all ? word(end) : -1, first,
                             lane, grad, ring + warp * kAddRing<T, VEC, kDirectBatches>,
                             [&](int slot, int) { return room.share[warp][slot][lane]; });
  }
  // rows that no word has
  const float zero[kGroup] = {};
#pragma unroll 1
  for (int row = warp; row < kSortRows && (((i64)row << bits) | cta) < a.R; row += kDirectWarps)
    if (room.start[row] == room.start[row + 1])
      Numbers<T, VEC>::store(grad + (((i64)row << bits) | cta) * a.H, first, lane, a.H, zero);
  __syncthreads();
  // rows that lie with several warps, by the first of them
  if (begin < end) {
    const int row = room.order[end - 1] >> 16, last = (room.start[row + 1] - 1) / part;
    if (room.start[row] / part == warp && last > warp) {
      float sum[kGroup] = {};
      for (int w = warp; w <= last; ++w) {
        const float4* p = room.share[w][w == warp && room.start[row] != begin ? 1 : 0][lane];
        const float4 x = p[0], y = p[1];
        sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
      }
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
      Numbers<T, VEC>::store(grad + ((i64)row << bits | cta) * a.H, first, lane, a.H, sum);
    }
  }
}

// Places per item: 8 to a warp while those warps fit the chip at once, so that their rows are read at once, else 32 (64 x 101
// words, rows of 256 numbers: 21 us with 8, 25 with 32; 256 x 201 words, rows of 1024: 96 with 8, 82 with 32).
int places_per_item(i64 N, int pieces) { return kWarps * (N * pieces <= 32 * 148 * 16 ? 8 : 32); }

bool aligned(const EmbedArgs& a, const void* rows) {
  const int size = a.dtype == kDtypeBf16 ? 2 : 4;
  const i64 all = (i64)reinterpret_cast<uintptr_t>(a.table) | (i64)reinterpret_cast<uintptr_t>(rows) |
                  a.stride * size | (i64)a.H * size;
  return all % 16 == 0;
}

template <typename F>
void with_variant(const EmbedArgs& a, bool wide, F launch) {
  with_type(a.dtype, wide, [&](auto type, auto vec) {
    if (a.dropped) launch(type, vec, std::true_type{});
    else launch(type, vec, std::false_type{});
  });
}

unsigned ctas(i64 warps, int ofCta = kWarps) {
  const i64 n = div_up64(warps, ofCta);
  if (n > 0x7fffffffLL) throw std::invalid_argument("too many rows");
  return (unsigned)n;
}

// Whether the gradient is made in one launch.  A frequent word is one CTA's there, for every 256 numbers: of 4096 words in a
// table of 30 rows it takes 23 us instead of 16 in three launches, in one of 1025 rows 16 instead of 17.
bool in_one_launch(i64 N, int R) { return N <= kDirectWords && N <= 32ll * R && R <= 128 * kSortRows; }
// CTAs that the rows are shared between, as a power of two: up to `most`, and no more than 256 rows each.
int row_bits(int R, int most) {
  int bits = 0;
  while ((2 << bits <= std::min(R, most)) || (i64)kSortRows << bits < R) ++bits;
  return bits;
}

// The launches of one call: each begins while the one before it ends, and waits for its results.
template <typename... P, typename... A>
void launch_early(void (*kernel)(P...), dim3 ctas, int threads, int smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = ctas, config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem, config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early, config.numAttrs = 1;
  TB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
}

}  // namespace

void launch_embed_words(const EmbedArgs& a, void* rows, int* beyond, cudaStream_t stream) {
  if (a.N == 0 || (a.H == 0 && !beyond)) return;
  const int pieces = std::max(1, div_up(a.H, 32 * kGroup));   // (rows of nothing have words to look at)
  with_variant(a, aligned(a, rows), [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool DROP = decltype(drop)::value;
    ScopedKernel prof("embed_words", stream);
    // a row per warp while they all fit the chip at once (64 x 16 rows of 640 bf16 numbers: 3.0 us, with four 3.9), else four
    // (256 x 201 rows of 1024: 25 us, with one 31)
    if (a.N * pieces <= 148 * 64)
      embed_kernel<T, VEC, DROP, 1><<<dim3(ctas(a.N), pieces), 32 * kWarps, 0, stream>>>(a, static_cast<T*>(rows), beyond);
    else
      embed_kernel<T, VEC, DROP, 4>
          <<<dim3(ctas(div_up64(a.N, 4)), pieces), 32 * kWarps, 0, stream>>>(a, static_cast<T*>(rows), beyond);
    TB200_CHECK_LAUNCH();
  });
}

size_t embed_backward_workspace_bytes(i64 N, int R, int H) {
  if (N <= 0 || R <= 0 || H <= 0) return 0;
  const int pieces = div_up(H, 32 * kGroup);
  if (in_one_launch(N, R)) return 0;
  return (size_t)(round_up64(N * 8, 16) + round_up64((R + 1ll) * 8, 16) +
                  div_up64(N, places_per_item(N, pieces)) * 2 * pieces * 32 * kGroup * 4);
}

void launch_embed_backward(const EmbedArgs& a, const void* deltas, void* grad, void* workspace, cudaStream_t stream) {
  if (a.R == 0 || a.H == 0) return;
  const int size = a.dtype == kDtypeBf16 ? 2 : 4;
  if (a.N == 0) {
    TB200_CUDA_CHECK(cudaMemsetAsync(grad, 0, (size_t)a.R * a.H * size, stream));
    return;
  }
  const int pieces = div_up(a.H, 32 * kGroup), part = places_per_item(a.N, pieces);
  EmbedArgs d = a;
  d.table = deltas, d.stride = a.H;
  const bool wide = aligned(d, grad);
  if (in_one_launch(a.N, a.R)) {
    with_variant(a, wide, [&](auto type, auto vec, auto drop) {
      using T = decltype(type);
      auto kernel = embed_direct_kernel<T, decltype(vec)::value, decltype(drop)::value>;
      constexpr int smem = sizeof(DirectRoom) + kDirectWarps * kAddRing<T, decltype(vec)::value, kDirectBatches>;
      allow_dyn_smem(kernel, smem);
      const int bits = row_bits(a.R, std::min(128, 2 * 148 / pieces));   // (two CTAs per SM at once)
      ScopedKernel prof("embed_direct", stream);
      kernel<<<dim3(1u << bits, pieces), 32 * kDirectWarps, smem, stream>>>(
          a, static_cast<const T*>(deltas), static_cast<T*>(grad), bits);
      TB200_CHECK_LAUNCH();
    });
    return;
  }
  char* at = static_cast<char*>(workspace);
  Sorted s;
  s.order = reinterpret_cast<int2*>(at), at += round_up64(a.N * 8, 16);
  s.range = reinterpret_cast<int2*>(at), at += round_up64((a.R + 1ll) * 8, 16);
  s.R = a.R;
  const Parts parts{reinterpret_cast<float*>(at), part, pieces, (int)div_up64(a.N, part)};
  {
    const int bits = row_bits(a.R, 128);
    ScopedKernel prof("embed_sort", stream);
    auto sort = [&](auto warps) {
      constexpr int WARPS = decltype(warps)::value;
      allow_dyn_smem(sort_words_kernel<WARPS>, sizeof(SortRoom<WARPS>));
      sort_words_kernel<WARPS><<<1u << bits, 32 * WARPS, sizeof(SortRoom<WARPS>), stream>>>(a.words, (int)a.N, bits, s);
      TB200_CHECK_LAUNCH();
    };
    if (a.N <= 4096) sort(std::integral_constant<int, 8>{});   // (of tables beyond what one launch does)
    else sort(std::integral_constant<int, 32>{});
  }
  with_variant(a, wide, [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool DROP = decltype(drop)::value;
    {
      ScopedKernel prof("embed_sums", stream);
      allow_dyn_smem(embed_sums_kernel<T, VEC, DROP>, kWarps * kAddRing<T, VEC, kSumBatches>);
      const int sumCtas = parts.items, filled = kFilled * kWarps * pieces;
      launch_early(embed_sums_kernel<T, VEC, DROP>, dim3(sumCtas + div_up(a.R, filled), pieces), 32 * kWarps,
                   kWarps * kAddRing<T, VEC, kSumBatches>, stream, a, static_cast<const T*>(deltas), s, parts, static_cast<T*>(grad), sumCtas);
    }
    if (parts.items > 1) {
      ScopedKernel prof("embed_join", stream);
      launch_early(embed_join_kernel<T, VEC>, dim3(ctas(parts.items, kJoinWarps), pieces), 32 * kJoinWarps, 0, stream, a, s, parts,
                   static_cast<T*>(grad));
    }
  });
}

}  // namespace tb200
