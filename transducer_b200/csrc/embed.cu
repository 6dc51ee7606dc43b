// Rows of a table for words, scaled and with dropout, and the table's gradient.
//
// Row n is factor * table[words[n], h] where number (n, h) stays and 0 where it is dropped; which ones are is decided by
// 16 bits of Philox4x32-10 with counter (n, h / 8) and the seed as its key, eight numbers to a counter.  The bits are
// made again where they are needed: no mask is ever stored.  The gradient of row r adds up the gradients of the
// rows that are r's, in their order, in fp32: the words' places are sorted by word first, so that no sum needs atomics
// and the bits are the same from run to run.
#include <algorithm>

#include "kernels.h"
#include "node_rows.cuh"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kWarps = 8, kGroup = 8;   // numbers of one counter, all in one lane

// Philox4x32-10 (Salmon, Moraes, Dror and Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011).
__device__ __forceinline__ uint4 philox(uint4 c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long a = 0xd2511f53ull * c.x, b = 0xcd9e8d57ull * c.z;
    c = make_uint4((unsigned)(b >> 32) ^ c.y ^ k0, (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ k1, (unsigned)a);
    k0 += 0x9e3779b9u, k1 += 0xbb67ae85u;
  }
  return c;
}

struct Seed {
  unsigned low, high;
  __device__ __forceinline__ explicit Seed(const EmbedArgs& a) {
    const i64 s = a.seedAt ? *a.seedAt : a.seed;
    low = (unsigned)s, high = (unsigned)((unsigned long long)s >> 32);
  }
};

// Bit i: number i of the group stays.
__device__ __forceinline__ unsigned kept(i64 n, int group, Seed seed, unsigned dropped) {
  const uint4 x = philox(make_uint4((unsigned)n, (unsigned)((unsigned long long)n >> 32), group, 0), seed.low, seed.high);
  const unsigned u[4] = {x.x, x.y, x.z, x.w};
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bits |= (u[i] & 0xffffu) >= dropped ? 1u << 2 * i : 0u;
    bits |= u[i] >> 16 >= dropped ? 2u << 2 * i : 0u;
  }
  return bits;
}

// The numbers of a row that a lane of a warp has, of 256 that begin at `first`: eight that follow each other where rows
// can be moved in 16-byte vectors, else every 32nd.
template <typename T, int VEC>
struct Numbers {
  static constexpr int kMoves = VEC == 1 ? kGroup : kGroup / VEC;
  RawWords<T, VEC> raw[kMoves];
  static __device__ __forceinline__ int at(int first, int lane, int move) {
    return first + (VEC == 1 ? 32 * move + lane : kGroup * lane + VEC * move);
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

// Bit i: number i that a lane has of row n stays.  All lanes: each makes the bits of a whole counter.
template <int VEC>
__device__ __forceinline__ unsigned stays(i64 n, int first, int lane, Seed seed, unsigned dropped) {
  const unsigned mine = kept(n, first / kGroup + lane, seed, dropped);
  if constexpr (VEC > 1) return mine;
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < kGroup; ++i)
    bits |= (__shfl_sync(0xffffffffu, mine, 4 * i + lane / kGroup) >> lane % kGroup & 1) << i;
  return bits;
}

// A warp writes 256 numbers of each of ROWS rows that follow each other.
template <typename T, int VEC, bool DROP, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) embed_kernel(EmbedArgs a, T* __restrict__ rows, int pieces) {
  const i64 id = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, first = (int)(id % pieces) * 32 * kGroup;
  const i64 n0 = id / pieces * ROWS;
  if (n0 >= a.N) return;
  int r[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) r[k] = n0 + k < a.N ? a.words[n0 + k] : -1;
  Numbers<T, VEC> x[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k)
    if ((unsigned)r[k] < (unsigned)a.R) x[k].load(static_cast<const T*>(a.table) + r[k] * a.stride, first, lane, a.H);
    else x[k].clear();
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (n0 + k >= a.N) break;
    float y[kGroup];
    x[k].get(y);
    unsigned stay = (unsigned)r[k] < (unsigned)a.R ? 0xff : 0;
    if constexpr (DROP)
      if (stay) stay = stays<VEC>(n0 + k, first, lane, Seed(a), a.dropped);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) y[i] = stay >> i & 1 ? y[i] * a.factor : 0.0f;
    Numbers<T, VEC>::store(rows + (n0 + k) * a.H, first, lane, a.H, y);
  }
}

// ---- the words' places in the order of the words ------------------------------------------------

constexpr int kSortWarps = 32, kSortRows = 256;   // rows per CTA

// A word and its place; places [start[r], start[r + 1]) of the order are row r's.
struct Sorted {
  int2* order;   // (place, word), [N]
  int* start;    // [R + 1]
};

// CTA c has the rows from c * rows on.  Every CTA goes through all words: it counts those of lower rows, which tells where
// its own begin, and per warp those of each of its rows; then every warp puts the places of its words where they belong.
__global__ void __launch_bounds__(32 * kSortWarps) sort_words_kernel(const int* __restrict__ words, i64 N, int R, int rows,
                                                                     Sorted out) {
  constexpr int kBatch = 16;   // words on their way at a time, per lane
  __shared__ int count[kSortWarps][kSortRows];
  __shared__ int total[kSortRows];
  __shared__ int below;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = blockIdx.x * rows, mine = min(rows, R - lo);
  cudaTriggerProgrammaticLaunchCompletion();
  for (int i = tid; i < kSortWarps * kSortRows; i += 32 * kSortWarps) (&count[0][0])[i] = 0;
  if (tid == 0) below = 0;
  __syncthreads();
  const i64 seg = round_up64(div_up64(N, kSortWarps), 32);
  const i64 first = warp * seg, end = min(N, first + seg);
  // f(words, places of the first) for the warp's words, 32 that follow each other at a time, in order
  auto each = [&](auto f) {
#pragma unroll 1
    for (i64 n = first; n < end; n += 32 * kBatch) {
      int r[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) r[j] = n + 32 * j + lane < end ? words[n + 32 * j + lane] : -1;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) f(r[j], n + 32 * j);
    }
  };
  int lower = 0;
  each([&](int r, i64) {
    lower += (unsigned)r < (unsigned)lo ? 1 : 0;
    if ((unsigned)r - (unsigned)lo < (unsigned)mine) atomicAdd(&count[warp][r - lo], 1);
  });
  lower = __reduce_add_sync(0xffffffffu, lower);
  if (lane == 0) atomicAdd(&below, lower);
  __syncthreads();
  if (tid < kSortRows) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = count[w][tid];
      count[w][tid] = sum;
      sum += c;
    }
    total[tid] = sum;
  }
  __syncthreads();
  if (warp == 0) {   // (the rows' sums to where each begins)
    int sum[kSortRows / 32], all = 0;
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) sum[i] = all, all += total[lane * (kSortRows / 32) + i];
    int before = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    before += below - all;
#pragma unroll
    for (int i = 0; i < kSortRows / 32; ++i) total[lane * (kSortRows / 32) + i] = before + sum[i];
    if (lane == 31 && lo + mine == R) out.start[R] = before + all;
  }
  __syncthreads();
  if (tid < mine) out.start[lo + tid] = total[tid];
  int* const at = count[warp];
  for (int i = lane; i < mine; i += 32) at[i] += total[i];
  __syncwarp();
  each([&](int r, i64 n) {
    const bool in = (unsigned)r - (unsigned)lo < (unsigned)mine;
    const unsigned any = __ballot_sync(0xffffffffu, in);
    if (!in) return;
    const unsigned same = __match_any_sync(any, r);
    const int rank = __popc(same & ((1u << lane) - 1));
    const int base = at[r - lo];
    __syncwarp(any);
    out.order[base + rank] = make_int2((int)n + lane, r);
    if (rank == 0) at[r - lo] = base + __popc(same);
    __syncwarp(any);
  });
}

// ---- the gradient -------------------------------------------------------------------------------

// An item is `part` places of the order that follow each other.  Rows that lie within one item are its sums; of the
// others every item leaves its share: slot 0 if it begins with the item, else slot 1.
struct Parts {
  float* sums;   // [items, 2, pieces, 32 lanes, 8]
  int part, pieces;
  i64 items;
  __device__ __forceinline__ float4* at(i64 item, int slot, int piece, int lane) const {
    return reinterpret_cast<float4*>(sums + ((((item * 2 + slot) * pieces + piece) * 32 + lane) * kGroup));
  }
};

constexpr int kMostPart = 32;

// The first items * pieces warps add up 256 numbers of an item's rows each; the others fill a row that no word has.
template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kWarps) embed_sums_kernel(EmbedArgs a, const T* __restrict__ deltas, Sorted s,
                                                                 Parts parts, T* __restrict__ grad) {
  constexpr int kBatch = 8;   // rows on their way at a time
  const i64 id = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const i64 fill = id - parts.items * parts.pieces;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  if (fill >= 0) {
    if (fill >= a.R || s.start[fill] != s.start[fill + 1]) return;
    const float zero[kGroup] = {};
    for (int first = 0; first < a.H; first += 32 * kGroup)
      Numbers<T, VEC>::store(grad + fill * a.H, first, lane, a.H, zero);
    return;
  }
  const i64 item = id / parts.pieces;
  const int piece = (int)(id % parts.pieces), first = piece * 32 * kGroup;
  const int from = (int)(item * parts.part), all = s.start[a.R];
  if (from >= all) return;
  const int to = (int)min((i64)from + parts.part, (i64)all);
  // lane i: the item's place i; the rows before it and behind it
  const int2 mine = lane < to - from ? s.order[from + lane] : make_int2(0, -1);
  const int before = from > 0 ? s.order[from - 1].y : -1, behind = to < all ? s.order[to].y : -1;
  const Seed seed(a);
  float sum[kGroup] = {};
  int row = __shfl_sync(0xffffffffu, mine.y, 0);
  bool begins = true;   // the present row is the item's first
  auto finish = [&](bool ends) {   // `ends`: it is the item's last
    const bool whole = !(begins && row == before) && !(ends && row == behind);
    if (whole) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
      Numbers<T, VEC>::store(grad + (i64)row * a.H, first, lane, a.H, sum);
    } else {
      float4* p = parts.at(item, begins ? 0 : 1, piece, lane);
      p[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
      p[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    }
  };
#pragma unroll 1
  for (int i = 0; i < to - from; i += kBatch) {
    Numbers<T, VEC> x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int n = __shfl_sync(0xffffffffu, mine.x, i + j);
      if (i + j < to - from) x[j].load(deltas + (i64)n * a.H, first, lane, a.H);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (i + j >= to - from) break;
      const int n = __shfl_sync(0xffffffffu, mine.x, i + j), r = __shfl_sync(0xffffffffu, mine.y, i + j);
      if (r != row) {
        finish(false);
#pragma unroll
        for (int k = 0; k < kGroup; ++k) sum[k] = 0.0f;
        row = r, begins = false;
      }
      float y[kGroup];
      x[j].get(y);
      unsigned stay = 0xff;
      if constexpr (DROP) stay = stays<VEC>(n, first, lane, seed, a.dropped);
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] += stay >> k & 1 ? y[k] : 0.0f;
    }
  }
  finish(true);
}

// Rows that lie in several items, each by the warp (or, of many items, the CTA) that has the first of them.
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kWarps) embed_join_kernel(EmbedArgs a, Sorted s, Parts parts,
                                                                 T* __restrict__ grad) {
  constexpr int kMany = 32;   // items from which on the CTA adds them up together
  __shared__ float4 shares[kWarps][32][2];
  __shared__ int many[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const i64 base = (i64)blockIdx.x * kWarps;
  cudaGridDependencySynchronize();
  // the row that warp w begins, or -1
  auto row_of = [&](int w, int& slot, i64& items) {
    const i64 item = (base + w) / parts.pieces;
    const i64 last = item * parts.part + parts.part - 1;
    if (item >= parts.items || last >= s.start[a.R]) return -1;
    const int r = s.order[last].y, from = s.start[r];
    items = (s.start[r + 1] - 1) / parts.part - item + 1;
    slot = from % parts.part == 0 ? 0 : 1;
    return from / parts.part == item && items > 1 ? r : -1;
  };
  // items [from, to) of the row, the first of them at `slot`
  auto add = [&](i64 item, int piece, int slot, i64 from, i64 to, float (&sum)[kGroup]) {
#pragma unroll 8
    for (i64 i = from; i < to; ++i) {
      const float4* p = parts.at(item + i, i == 0 ? slot : 0, piece, lane);
      const float4 x = p[0], y = p[1];
      sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
      sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
    }
  };
  auto write = [&](int r, int piece, float (&sum)[kGroup]) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
    Numbers<T, VEC>::store(grad + (i64)r * a.H, piece * 32 * kGroup, lane, a.H, sum);
  };
  int slot = 0;
  i64 items = 0;
  const int r = row_of(warp, slot, items);
  if (lane == 0) many[warp] = r >= 0 && items >= kMany;
  if (r >= 0 && items < kMany) {
    float sum[kGroup] = {};
    add((base + warp) / parts.pieces, (int)((base + warp) % parts.pieces), slot, 0, items, sum);
    write(r, (int)((base + warp) % parts.pieces), sum);
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) {
    if (!many[w]) continue;
    const int row = row_of(w, slot, items);
    const i64 item = (base + w) / parts.pieces;
    const int piece = (int)((base + w) % parts.pieces);
    const i64 share = div_up64(items, kWarps);
    float sum[kGroup] = {};
    add(item, piece, slot, warp * share, min(items, (warp + 1) * share), sum);
    shares[warp][lane][0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    shares[warp][lane][1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    __syncthreads();
    if (warp == w) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float4 x = shares[i][lane][0], y = shares[i][lane][1];
        sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
      }
      write(row, piece, sum);
    }
    __syncthreads();
  }
}

// Places per item: few where there are few warps, so that the rows are read at once; their shares then weigh more.
int places_per_item(i64 N, int pieces) { return N * pieces <= 32 * 148 * 16 ? 8 : kMostPart; }

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

unsigned ctas(i64 rows, int pieces) {
  const i64 n = div_up64(rows * pieces, kWarps);
  if (n > 0x7fffffffLL) throw std::invalid_argument("too many rows");
  return (unsigned)n;
}

// The launches of one call: each begins while the one before it ends, and waits for its results.
template <typename... P, typename... A>
void launch_early(void (*kernel)(P...), unsigned ctas, int threads, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas), config.blockDim = dim3(threads), config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early, config.numAttrs = 1;
  TB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
}

}  // namespace

void launch_embed_words(const EmbedArgs& a, void* rows, cudaStream_t stream) {
  if (a.N == 0 || a.H == 0) return;
  const int pieces = div_up(a.H, 32 * kGroup);
  with_variant(a, aligned(a, rows), [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool DROP = decltype(drop)::value;
    ScopedKernel prof("embed_words", stream);
    if (a.N * pieces <= 148 * 64)   // (a row per warp fits the chip at once)
      embed_kernel<T, VEC, DROP, 1><<<ctas(a.N, pieces), 32 * kWarps, 0, stream>>>(a, static_cast<T*>(rows), pieces);
    else
      embed_kernel<T, VEC, DROP, 4>
          <<<ctas(div_up64(a.N, 4), pieces), 32 * kWarps, 0, stream>>>(a, static_cast<T*>(rows), pieces);
    TB200_CHECK_LAUNCH();
  });
}

size_t embed_backward_workspace_bytes(i64 N, int R, int H) {
  if (N <= 0 || R <= 0 || H <= 0) return 0;
  const int pieces = div_up(H, 32 * kGroup);
  return (size_t)(round_up64(N * 8, 16) + round_up64((R + 1ll) * 4, 16) +
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
  char* at = static_cast<char*>(workspace);
  Sorted s;
  s.order = reinterpret_cast<int2*>(at), at += round_up64(a.N * 8, 16);
  s.start = reinterpret_cast<int*>(at), at += round_up64((a.R + 1ll) * 4, 16);
  const Parts parts{reinterpret_cast<float*>(at), part, pieces, div_up64(a.N, part)};
  {
    const int rows = std::max(1, std::min(kSortRows, div_up(a.R, 148)));
    ScopedKernel prof("embed_sort", stream);
    sort_words_kernel<<<div_up(a.R, rows), 32 * kSortWarps, 0, stream>>>(a.words, a.N, a.R, rows, s);
    TB200_CHECK_LAUNCH();
  }
  EmbedArgs d = a;
  d.table = deltas, d.stride = a.H;
  with_variant(a, aligned(d, grad), [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool DROP = decltype(drop)::value;
    {
      ScopedKernel prof("embed_sums", stream);
      launch_early(embed_sums_kernel<T, VEC, DROP>, ctas(parts.items * pieces + a.R, 1), 32 * kWarps, stream, a,
                   static_cast<const T*>(deltas), s, parts, static_cast<T*>(grad));
    }
    if (parts.items > 1) {
      ScopedKernel prof("embed_join", stream);
      launch_early(embed_join_kernel<T, VEC>, ctas(parts.items, pieces), 32 * kWarps, stream, a, s, parts,
                   static_cast<T*>(grad));
    }
  });
}

}  // namespace tb200
