// States that follow their hypotheses: row w of an utterance becomes what row parents[w] was, in every tensor of a
// list at once.
#include <algorithm>
#include <cstdlib>
#include <vector>

#include "kernels.h"
#include "profile.h"

namespace tb200 {
namespace {

constexpr int kMostStates = 24;        // of a launch (they travel as kernel arguments)
constexpr int kShifted = -16, kShiftedRow = 64;   // rows that long are moved in vectors whatever their alignment
constexpr int kWarps = 8, kBatch = 8;  // a warp moves kBatch vectors per lane at a time

struct Item {
  States s;
  unsigned firstWarp;   // of the launch
  int pieces, bytes;    // of a row; bytes of a vector (kShifted: see move_shifted)
};
struct Batch {
  Item item[kMostStates];
  int count;
};

template <typename T>
__device__ __forceinline__ void move_row(const char* from, char* to, i64 bytes, int lane) {
  const T* f = reinterpret_cast<const T*>(from);
  T* t = reinterpret_cast<T*>(to);
  const int n = (int)(bytes / sizeof(T));
  T x[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (lane + 32 * j < n) x[j] = from ? f[lane + 32 * j] : T{};
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (lane + 32 * j < n) t[lane + 32 * j] = x[j];
}

// Bytes of any alignment: stored in 16-byte vectors, loaded as the aligned words that hold them.
__device__ __forceinline__ void move_shifted(const char* from, char* to, int bytes, int lane) {
  const int head = min(bytes, (int)(-(uintptr_t)to & 15)), vectors = (bytes - head) / 16, tail = head + 16 * vectors;
  const char* at = from + head;
  const int shift = (int)((uintptr_t)at & 3);
  const unsigned* words = reinterpret_cast<const unsigned*>(at - shift);
  unsigned x[kBatch][5];
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int v = lane + 32 * j;
    if (v < vectors) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = from ? words[4 * v + i] : 0u;
      x[j][4] = from && shift ? words[4 * v + 4] : 0u;
    }
  }
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int v = lane + 32 * j;
    if (v < vectors) {
      uint4 y;
      y.x = __funnelshift_r(x[j][0], x[j][1], 8 * shift), y.y = __funnelshift_r(x[j][1], x[j][2], 8 * shift);
      y.z = __funnelshift_r(x[j][2], x[j][3], 8 * shift), y.w = __funnelshift_r(x[j][3], x[j][4], 8 * shift);
      reinterpret_cast<uint4*>(to + head)[v] = y;
    }
  }
  if (lane < head) to[lane] = from ? from[lane] : 0;
  if (tail + lane < bytes) to[tail + lane] = from ? from[tail + lane] : 0;
}

__global__ void __launch_bounds__(32 * kWarps) reorder_kernel(const __grid_constant__ Batch batch,
                                                              const int* __restrict__ parents, int N, int W,
                                                              bool kept, unsigned warps, int* beyond) {
  const unsigned id = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (id >= warps) return;
  int k = 0;
  while (k + 1 < batch.count && batch.item[k + 1].firstWarp <= id) ++k;
  const Item& it = batch.item[k];
  const unsigned row = (id - it.firstWarp) / (unsigned)it.pieces;
  const int n = parents[row];
  const int b = row / (unsigned)W, w = row % (unsigned)W;
  const bool here = (unsigned)n < (unsigned)N;
  if (beyond && n >= N) *beyond = 1;
  if (!here && kept) return;
  const i64 piece = 32ll * kBatch * abs(it.bytes), at = (id - it.firstWarp) % (unsigned)it.pieces * piece;
  const i64 bytes = min(piece, it.s.rowBytes - at);
  const char* from = here ? it.s.from + b * it.s.fromB + n * it.s.fromN + at : nullptr;
  char* to = it.s.to + b * it.s.toB + w * it.s.toW + at;
  switch (it.bytes) {
    case kShifted: move_shifted(from, to, (int)bytes, lane); break;
    case 16: move_row<uint4>(from, to, bytes, lane); break;
    case 8: move_row<uint2>(from, to, bytes, lane); break;
    case 4: move_row<unsigned>(from, to, bytes, lane); break;
    case 2: move_row<unsigned short>(from, to, bytes, lane); break;
    default: move_row<unsigned char>(from, to, bytes, lane);
  }
}

// In place: a CTA has a piece of the rows of all hypotheses of an utterance and reads it whole before it writes.
template <typename T>
__device__ __forceinline__ void move_in_place(const States& s, const int* parents, i64 b, i64 at, int units, int N, int W,
                                              T* held) {
  for (int i = threadIdx.x; i < W * units; i += blockDim.x) {
    const int w = i / units, n = parents[w];
    if ((unsigned)n < (unsigned)N && n != w)
      held[i] = reinterpret_cast<const T*>(s.from + b * s.fromB + n * s.fromN + at)[i % units];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < W * units; i += blockDim.x) {
    const int w = i / units, n = parents[w];
    if ((unsigned)n < (unsigned)N && n != w)
      reinterpret_cast<T*>(s.to + b * s.toB + w * s.toW + at)[i % units] = held[i];
  }
}

__global__ void __launch_bounds__(256) reorder_in_place_kernel(const __grid_constant__ Batch batch,
                                                               const int* __restrict__ parents, int N, int W,
                                                               int held, int* beyond) {
  extern __shared__ __align__(16) char room[];
  const unsigned id = blockIdx.x;
  int k = 0;
  while (k + 1 < batch.count && batch.item[k + 1].firstWarp <= id) ++k;   // (CTAs here)
  const Item& it = batch.item[k];
  const i64 b = (id - it.firstWarp) / (unsigned)it.pieces, at = (id - it.firstWarp) % (unsigned)it.pieces * (i64)held;
  const int units = (int)(min((i64)held, it.s.rowBytes - at) / it.bytes);
  parents += b * W;
  if (beyond)
    for (int w = threadIdx.x; w < W; w += blockDim.x)
      if (parents[w] >= N) *beyond = 1;
  switch (it.bytes) {
    case 16: move_in_place(it.s, parents, b, at, units, N, W, reinterpret_cast<uint4*>(room)); break;
    case 8: move_in_place(it.s, parents, b, at, units, N, W, reinterpret_cast<uint2*>(room)); break;
    case 4: move_in_place(it.s, parents, b, at, units, N, W, reinterpret_cast<unsigned*>(room)); break;
    case 2: move_in_place(it.s, parents, b, at, units, N, W, reinterpret_cast<unsigned short*>(room)); break;
    default: move_in_place(it.s, parents, b, at, units, N, W, reinterpret_cast<unsigned char*>(room));
  }
}

int vector_bytes(const States& s) {
  i64 all = (i64)reinterpret_cast<uintptr_t>(s.from) | (i64)reinterpret_cast<uintptr_t>(s.to) | s.fromB | s.fromN |
            s.toB | s.toW | s.rowBytes;
  for (int bytes = 16; bytes > 1; bytes /= 2)
    if (all % bytes == 0) return bytes;
  return 1;
}

}  // namespace

void launch_reorder_states(const States* states, int count, const int* parents, int B, int N, int W, bool kept,
                           int* beyond, cudaStream_t stream) {
  if ((i64)B * W == 0) return;
  std::vector<Item> apart, inPlace;
  for (int i = 0; i < count; ++i) {
    if (states[i].rowBytes == 0) continue;
    Item it{states[i], 0, 0, vector_bytes(states[i])};
    (states[i].from == states[i].to ? inPlace : apart).push_back(it);
  }
  // (nothing is to be moved, but the parents are to be looked at)
  if (beyond && count > 0 && apart.empty() && inPlace.empty()) apart.push_back(Item{states[0], 0, 0, 1});
  // a piece of a row in place: with W of them 32 KB, a vector at least
  const int held = std::max(16, 32 * 1024 / std::max(W, 1) / 16 * 16);
  for (size_t i = 0; i < apart.size();) {
    Batch batch{};
    i64 warps = 0;
    for (; i < apart.size() && batch.count < kMostStates; ++i) {
      Item it = apart[i];
      if (it.bytes < 16 && it.s.rowBytes >= kShiftedRow) it.bytes = kShifted;
      it.firstWarp = (unsigned)warps;
      it.pieces = (int)std::max<i64>(1, div_up64(it.s.rowBytes, 32ll * kBatch * std::abs(it.bytes)));
      const i64 more = (i64)B * W * it.pieces;
      if (warps + more > 0xfffffff0LL) {
        if (batch.count == 0) throw std::invalid_argument("the states are too large");
        break;
      }
      batch.item[batch.count++] = it;
      warps += more;
    }
    ScopedKernel prof("reorder_states", stream);
    reorder_kernel<<<(unsigned)div_up64(warps, kWarps), 32 * kWarps, 0, stream>>>(batch, parents, N, W, kept,
                                                                                 (unsigned)warps, beyond);
    TB200_CHECK_LAUNCH();
  }
  for (size_t first = 0; first < inPlace.size(); first += kMostStates) {
    Batch batch{};
    i64 ctas = 0;
    for (size_t i = first; i < inPlace.size() && batch.count < kMostStates; ++i) {
      Item& it = batch.item[batch.count++] = inPlace[i];
      it.firstWarp = (unsigned)ctas;
      it.pieces = (int)div_up64(it.s.rowBytes, held);
      ctas += (i64)B * it.pieces;
    }
    if (ctas > 0x7fffffffLL) throw std::invalid_argument("the states are too large");
    allow_dyn_smem(reorder_in_place_kernel, 16 * kMaxReorderedWidth);
    ScopedKernel prof("reorder_in_place", stream);
    reorder_in_place_kernel<<<(unsigned)ctas, 256, held * W, stream>>>(batch, parents, N, W, held, beyond);
    TB200_CHECK_LAUNCH();
  }
}

}  // namespace tb200
