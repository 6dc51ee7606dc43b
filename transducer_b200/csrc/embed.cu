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

// Eight numbers of a row from h on, as far as it goes (VEC > 1: 16 bytes at a time, whole groups only).
template <typename T, int VEC>
__device__ __forceinline__ void load_group(const T* row, int h, int H, float (&x)[kGroup]) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int i = 0; i < kGroup; i += VEC)
      if (h + i < H) {
        const Words<VEC> w = load_words<VEC>(row + h + i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i + j] = w.x[j];
      }
  } else {
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
      if (h + i < H) x[i] = to_f32(row[h + i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_group(T* row, int h, int H, const float (&x)[kGroup]) {
#pragma unroll
  for (int i = 0; i < kGroup; i += VEC)
    if (h + i < H) store_words<VEC>(row + h + i, x + i);
}

// A warp writes 256 numbers of a row.
template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kWarps) embed_kernel(EmbedArgs a, T* __restrict__ rows, int pieces) {
  const i64 id = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const i64 n = id / pieces;
  const int h = ((int)(id % pieces) * 32 + (threadIdx.x & 31)) * kGroup;
  if (n >= a.N || h >= a.H) return;
  const int r = a.words[n];
  float x[kGroup] = {};
  if ((unsigned)r < (unsigned)a.R) {
    load_group<T, VEC>(static_cast<const T*>(a.table) + r * a.stride, h, a.H, x);
    unsigned stay = 0xff;
    if constexpr (DROP) stay = kept(n, h / kGroup, Seed(a), a.dropped);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) x[i] = stay >> i & 1 ? x[i] * a.factor : 0.0f;
  }
  store_group<T, VEC>(rows + n * a.H, h, a.H, x);
}

// ---- the words' places in the order of the words ------------------------------------------------

constexpr int kSortWarps = 32, kSortRows = 256;   // rows per CTA

// CTA c has the rows from c * rows on.  Every CTA goes through all words: it counts those of lower rows, which tells where
// its own begin, and per warp those of each of its rows; then every warp puts the places of its words where they belong.
__global__ void __launch_bounds__(32 * kSortWarps) sort_words_kernel(const int* __restrict__ words, i64 N, int R, int rows,
                                                                     int* __restrict__ order, int* __restrict__ start) {
  __shared__ int count[kSortWarps][kSortRows];
  __shared__ int total[kSortRows];
  __shared__ int below;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = blockIdx.x * rows, mine = min(rows, R - lo);
  for (int i = tid; i < kSortWarps * kSortRows; i += 32 * kSortWarps) (&count[0][0])[i] = 0;
  if (tid == 0) below = 0;
  __syncthreads();
  const i64 seg = round_up64(div_up64(N, kSortWarps), 32);
  const i64 first = warp * seg, end = min(N, first + seg);
  int lower = 0;
#pragma unroll 4
  for (i64 n = first + lane; n < end; n += 32) {
    const int r = words[n];
    lower += (unsigned)r < (unsigned)lo ? 1 : 0;
    if ((unsigned)(r - lo) < (unsigned)mine) atomicAdd(&count[warp][r - lo], 1);
  }
  lower = __reduce_add_sync(0xffffffffu, lower);
  if (lane == 0) atomicAdd(&below, lower);
  __syncthreads();
  if (tid < kSortRows) {
    int sum = 0;
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
    if (lane == 31 && lo + mine == R) start[R] = before + all;
  }
  __syncthreads();
  if (tid < mine) start[lo + tid] = total[tid];
  int* const at = count[warp];
  for (int i = lane; i < mine; i += 32) at[i] += total[i];
  __syncwarp();
#pragma unroll 4
  for (i64 n = first + lane; n - lane < end; n += 32) {
    const int r = n < end ? words[n] - lo : -1;
    const bool in = (unsigned)r < (unsigned)mine;
    const unsigned any = __ballot_sync(0xffffffffu, in);
    if (any == 0) continue;
    if (in) {
      const unsigned same = __match_any_sync(any, r);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int base = at[r];
      __syncwarp(any);
      order[base + rank] = (int)n;
      if (rank == 0) at[r] = base + __popc(same);
      __syncwarp(any);
    }
  }
}

// ---- the gradient -------------------------------------------------------------------------------

constexpr int kPart = 64;   // places that are added up apart, of rows that have so many

struct Sorted {
  const int *order, *start;
  float* parts;   // [N / kPart, ldParts]: part p of row r is at start[r] / kPart + p
  int ld;
};

// sum += the gradients of the rows in places [from, to).
template <typename T, int VEC, bool DROP>
__device__ __forceinline__ void add_places(const EmbedArgs& a, const T* deltas, const int* order, i64 from, i64 to, i64 step,
                                           int h, Seed seed, float (&sum)[kGroup]) {
  constexpr int kBatch = 4;
#pragma unroll 1
  for (i64 i = from; i < to; i += kBatch * step) {
    float x[kBatch][kGroup];
    i64 n[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) n[j] = i + j * step < to ? order[i + j * step] : -1;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (n[j] >= 0 && h < a.H) load_group<T, VEC>(deltas + n[j] * a.H, h, a.H, x[j]);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (n[j] >= 0 && h < a.H) {
        unsigned stay = 0xff;
        if constexpr (DROP) stay = kept(n[j], h / kGroup, seed, a.dropped);
#pragma unroll
        for (int k = 0; k < kGroup; ++k) sum[k] += h + k < a.H && stay >> k & 1 ? x[j][k] : 0.0f;
      }
  }
}

// Whole parts of rows that have at least one.
template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kWarps) embed_parts_kernel(EmbedArgs a, const T* __restrict__ deltas, Sorted s,
                                                                  int pieces) {
  const i64 id = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const i64 part = id / pieces;
  const int h = ((int)(id % pieces) * 32 + (threadIdx.x & 31)) * kGroup;
  const i64 last = part * kPart + kPart - 1;   // (a place within the part)
  if (last >= s.start[a.R]) return;
  const int r = a.words[s.order[last]];
  const int from = s.start[r], whole = (s.start[r + 1] - from) / kPart;
  const i64 p = part - from / kPart;
  if (p < 0 || p >= whole || h >= a.H) return;
  float sum[kGroup] = {};
  add_places<T, VEC, DROP>(a, deltas, s.order, from + p * kPart, from + (p + 1) * kPart, 1, h, Seed(a), sum);
  store_group<float, 4>(s.parts + part * s.ld, h, s.ld, sum);
}

template <typename T, int VEC, bool DROP>
__global__ void __launch_bounds__(32 * kWarps) embed_rows_kernel(EmbedArgs a, const T* __restrict__ deltas, Sorted s,
                                                                 T* __restrict__ grad, int pieces) {
  const i64 id = (i64)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const i64 r = id / pieces;
  const int h = ((int)(id % pieces) * 32 + (threadIdx.x & 31)) * kGroup;
  if (r >= a.R || h >= a.H) return;
  const int from = s.start[r], to = s.start[r + 1], whole = (to - from) / kPart;
  float sum[kGroup] = {};
  const float* part = s.parts + (i64)(from / kPart) * s.ld;
#pragma unroll 4
  for (int p = 0; p < whole; ++p) {
    float x[kGroup];
    load_group<float, 4>(part + (i64)p * s.ld, h, s.ld, x);
#pragma unroll
    for (int k = 0; k < kGroup; ++k) sum[k] += x[k];
  }
  add_places<T, VEC, DROP>(a, deltas, s.order, from + whole * kPart, to, 1, h, Seed(a), sum);
#pragma unroll
  for (int k = 0; k < kGroup; ++k) sum[k] *= a.factor;
  store_group<T, VEC>(grad + r * a.H, h, a.H, sum);
}

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

}  // namespace

void launch_embed_words(const EmbedArgs& a, void* rows, cudaStream_t stream) {
  if (a.N == 0 || a.H == 0) return;
  const int pieces = div_up(a.H, 32 * kGroup);
  with_variant(a, aligned(a, rows), [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    ScopedKernel prof("embed_words", stream);
    embed_kernel<T, decltype(vec)::value, decltype(drop)::value>
        <<<ctas(a.N, pieces), 32 * kWarps, 0, stream>>>(a, static_cast<T*>(rows), pieces);
    TB200_CHECK_LAUNCH();
  });
}

size_t embed_backward_workspace_bytes(i64 N, int R, int H) {
  if (N <= 0 || R <= 0 || H <= 0) return 0;
  return (size_t)(round_up64(N * 4, 16) + round_up64((R + 1ll) * 4, 16) + N / kPart * round_up64(H, kGroup) * 4);
}

void launch_embed_backward(const EmbedArgs& a, const void* deltas, void* grad, void* workspace, cudaStream_t stream) {
  if (a.R == 0 || a.H == 0) return;
  const int size = a.dtype == kDtypeBf16 ? 2 : 4;
  if (a.N == 0) {
    TB200_CUDA_CHECK(cudaMemsetAsync(grad, 0, (size_t)a.R * a.H * size, stream));
    return;
  }
  int* order = static_cast<int*>(workspace);
  int* start = order + round_up64(a.N, 4);
  float* parts = reinterpret_cast<float*>(start + round_up64(a.R + 1ll, 4));
  const Sorted s{order, start, parts, (int)round_up64(a.H, kGroup)};
  {
    const int rows = std::max(1, std::min(kSortRows, div_up(a.R, 148)));
    ScopedKernel prof("embed_sort", stream);
    sort_words_kernel<<<div_up(a.R, rows), 32 * kSortWarps, 0, stream>>>(a.words, a.N, a.R, rows, order, start);
    TB200_CHECK_LAUNCH();
  }
  const int pieces = div_up(a.H, 32 * kGroup);
  EmbedArgs d = a;
  d.table = deltas, d.stride = a.H;
  with_variant(a, aligned(d, grad), [&](auto type, auto vec, auto drop) {
    using T = decltype(type);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool DROP = decltype(drop)::value;
    const T* from = static_cast<const T*>(deltas);
    if (a.N >= kPart) {
      ScopedKernel prof("embed_parts", stream);
      embed_parts_kernel<T, VEC, DROP>
          <<<ctas(a.N / kPart, pieces), 32 * kWarps, 0, stream>>>(a, from, s, pieces);
      TB200_CHECK_LAUNCH();
    }
    ScopedKernel prof("embed_rows", stream);
    embed_rows_kernel<T, VEC, DROP>
        <<<ctas(a.R, pieces), 32 * kWarps, 0, stream>>>(a, from, s, static_cast<T*>(grad), pieces);
    TB200_CHECK_LAUNCH();
  });
}

}  // namespace tb200
