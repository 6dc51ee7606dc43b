// States that follow their hypotheses: row w of an utterance becomes what row parents[w] was, in every tensor of a
// list at once.  Copies, bound by HBM: 32 x 16 hypotheses with 410 KB each (339 MB read and written, parents that
// have several successors read once) take 55 us, 52 at the measured copy rate; in place 64; 4 x 8 hypotheses with
// 10 KB 4 us, latency.  A warp has 4 KB of a row, eight vectors a lane on their way.
#include <algorithm>
#include <cstdlib>
#include <vector>

#include "kernels.h"
#include "node_rows.cuh"
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

// Bytes of any alignment: stored in 16-byte vectors, loaded as the aligned words that hold them.  (64 x 24 rows of 641 bf16
// numbers, five states: 6.4 us; two bytes at a time 10.3.)
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

// In place: a CTA has a piece of the rows of all hypotheses of an utterance and has read what moves before it writes any of
// it.  The rows are brought as the aligned 16-byte vectors that hold them (of which others may be writing the bytes of
// other rows, and of which bytes may lie outside the tensor; those are not looked at).  Only what moves is read and written; number by number through shared memory it
// took 88 us where this takes 64, and 41 instead of 9 where everything stays.
__global__ void __launch_bounds__(32 * kWarps) reorder_in_place_kernel(const __grid_constant__ Batch batch,
                                                                       const int* __restrict__ parents, int N, int W,
                                                                       int held, int* beyond) {
  extern __shared__ __align__(16) char room[];   // W rows of held + 32 bytes, then the hypotheses that move
  __shared__ int moved;
  int* const list = reinterpret_cast<int*>(room + (size_t)W * (held + 32));
  const unsigned id = blockIdx.x;
  int k = 0;
  while (k + 1 < batch.count && batch.item[k + 1].firstWarp <= id) ++k;   // (CTAs here)
  const Item& it = batch.item[k];
  const i64 b = (id - it.firstWarp) / (unsigned)it.pieces, at = (id - it.firstWarp) % (unsigned)it.pieces * (i64)held;
  const int bytes = (int)min((i64)held, it.s.rowBytes - at);
  parents += b * W;
  if (threadIdx.x == 0) moved = 0;
  __syncthreads();
  for (int w = threadIdx.x; w < W; w += blockDim.x) {
    const int n = parents[w];
    if (beyond && n >= N) *beyond = 1;
    if ((unsigned)n < (unsigned)N && n != w) list[atomicAdd(&moved, 1)] = w;
  }
  __syncthreads();
  const int moves = moved;
  const int stride = held + 32;
  const unsigned lanes = min(32, held / 16 + 1);   // that a row takes, at most 32 vectors at a time
  auto from_of = [&](int w) { return it.s.from + b * it.s.fromB + parents[w] * it.s.fromN + at; };
  for (unsigned i = threadIdx.x; i < moves * lanes; i += blockDim.x) {
    const unsigned m = i / lanes;
    const char* from = from_of(list[m]);
    const int before = (int)((uintptr_t)from & 15);
    for (unsigned v = i % lanes; 16 * v < before + bytes; v += lanes)
      copy_async<16>(room + m * stride + 16 * v, from - before + 16 * v);
  }
  commit_copies();
  wait_copies<0>();
  __syncthreads();
  for (unsigned i = threadIdx.x; i < moves * lanes; i += blockDim.x) {
    const unsigned m = i / lanes, lane = i % lanes;
    const int w = list[m];
    const char* from = room + m * stride + ((uintptr_t)from_of(w) & 15);
    char* to = it.s.to + b * it.s.toB + w * it.s.toW + at;
    const int head = min(bytes, (int)(-(uintptr_t)to & 15)), vectors = (bytes - head) / 16, tail = head + 16 * vectors;
    const int shift = (int)((uintptr_t)(from + head) & 15);
    const unsigned* words = reinterpret_cast<const unsigned*>(from + head - (shift & 3));
    uint4* vec = reinterpret_cast<uint4*>(to + head);
    for (int v = lane; v < vectors; v += lanes) {
      if (shift == 0) {
        vec[v] = reinterpret_cast<const uint4*>(words)[v];
      } else {
        const unsigned x[5] = {words[4 * v], words[4 * v + 1], words[4 * v + 2], words[4 * v + 3], words[4 * v + 4]};
        const int s = 8 * (shift & 3);
        vec[v] = make_uint4(__funnelshift_r(x[0], x[1], s), __funnelshift_r(x[1], x[2], s), __funnelshift_r(x[2], x[3], s),
                            __funnelshift_r(x[3], x[4], s));
      }
    }
    for (int j = lane; j < head; j += lanes) to[j] = from[j];
    for (int j = tail + lane; j < bytes; j += lanes) to[j] = from[j];
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
  // a piece of a row in place: with W of them 48 KB, a vector at least
  const int held = std::min(4096, std::max(16, (48 * 1024 / std::max(W, 1) - 32) / 16 * 16));
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
    allow_dyn_smem(reorder_in_place_kernel, 52 * kMaxReorderedWidth);
    ScopedKernel prof("reorder_in_place", stream);
    reorder_in_place_kernel<<<(unsigned)ctas, 32 * kWarps, (held + 36) * W, stream>>>(batch, parents, N, W, held, beyond);
    TB200_CHECK_LAUNCH();
  }
}

}  // namespace tb200
