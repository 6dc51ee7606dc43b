// Rows of scores at single lattice nodes, shared by the node kernels (node_top.cu, node_sample.cu,
// node_distill.cu).  Node n of utterance b is frame frames[b,n] and label position
// positions[b,n]; its scores are E[b,frame,v] + P[b,position,v], one addition in fp32.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace tb200 {

// Words are moved VEC at a time: 16 bytes where every row starts on a 16-byte boundary, else one word.
template <int VEC>
struct Words {
  float x[VEC];
};
// ... and in storage form, as they come.
template <typename TIn, int VEC>
struct RawWords {
  static_assert(VEC == 1 || VEC * sizeof(TIn) == 16);
  std::conditional_t<VEC == 1, TIn, uint4> bits;
  __device__ __forceinline__ void load(const TIn* p) { bits = *reinterpret_cast<const decltype(bits)*>(p); }
  __device__ __forceinline__ void clear() { bits = {}; }
  __device__ __forceinline__ Words<VEC> words() const {
    Words<VEC> w;
    if constexpr (VEC == 1) {
      w.x[0] = to_f32(bits);
    } else {
      const unsigned u[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VEC == 4) {
          w.x[i] = __uint_as_float(u[i]);
        } else {
          w.x[2 * i] = __uint_as_float(u[i] << 16);
          w.x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
      }
    }
    return w;
  }
};
template <int VEC, typename TIn>
__device__ __forceinline__ Words<VEC> load_words(const TIn* p) {
  RawWords<TIn, VEC> r;
  r.load(p);
  return r.words();
}
template <int VEC>
__device__ __forceinline__ void store_words(float* p, const float* x) {
  if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else *p = x[0];
}
template <int VEC>
__device__ __forceinline__ void store_words(bf16* p, const float* x) {
  if constexpr (VEC == 8) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    from_f32(*p, x[0]);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous copies to shared memory.
// (16 bytes: past the L1)
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// The scores of one node.
template <typename TIn>
struct NodeScores {
  const TIn *e, *p;
  int t, u;
  bool here;
};
template <typename TIn>
__device__ __forceinline__ NodeScores<TIn> node_scores(const NodeArgs& a, i64 node) {
  const i64 b = (unsigned)node / (unsigned)a.N;   // (fewer than 2^31 nodes)
  const int t = a.frames[node], u = a.positions[node];
  NodeScores<TIn> s;
  s.t = t, s.u = u;
  s.here = (unsigned)t < (unsigned)a.T && (unsigned)u < (unsigned)a.U;
  s.e = static_cast<const TIn*>(a.E) + b * a.eStrideB + (s.here ? t : 0) * a.eStrideT;
  s.p = static_cast<const TIn*>(a.P) + b * a.pStrideB + (s.here ? u : 0) * a.pStrideU;
  return s;
}

// Sums and maxima over a group of G threads (a warp, or the CTA): every thread gets the result, and
// its bits do not depend on anything but the values.  `scratch`: two sets of 32 places of 16 bytes in
// shared memory, used in turn, so that one barrier per reduction is enough.
template <int G>
struct Group {
  static constexpr int kWarps = G / 32;
  int tid, lane, warp;
  double2* scratch;   // [2][32], of the CTA; unused by a warp
  int turn = 0;
  __device__ __forceinline__ Group(int tid_, double2* scratch_)
      : tid(tid_), lane(tid_ & 31), warp(tid_ >> 5), scratch(scratch_) {}

  __device__ __forceinline__ void sync() const {
    if constexpr (G == 32) __syncwarp();
    else __syncthreads();
  }
  // The warps' values v (the same in all lanes of a warp) in the order of the warps: lane i gets that
  // of warp i % kWarps.
  template <typename T>
  __device__ __forceinline__ T exchange(T v) {
    if constexpr (G > 32) {
      T* s = reinterpret_cast<T*>(scratch + 32 * turn);
      turn ^= 1;
      if (lane == 0) s[warp] = v;
      __syncthreads();
      v = s[lane % kWarps];
    }
    return v;
  }
  template <typename T, typename Op>
  __device__ __forceinline__ T reduce(T v, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return across(v, op);
  }
  __device__ __forceinline__ float sum(float v) { return reduce(v, [](float a, float b) { return a + b; }); }
  __device__ __forceinline__ double sum(double v) { return reduce(v, [](double a, double b) { return a + b; }); }
  // two sums at once
  __device__ __forceinline__ void sum(double& a, float& b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (G > 32) {
      const double2 v = exchange(make_double2(a, (double)b));
      a = v.x, b = (float)v.y;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    }
  }
  __device__ __forceinline__ int sum(int v) {
    return across(__reduce_add_sync(0xffffffffu, v), [](int a, int b) { return a + b; });
  }
  __device__ __forceinline__ float max(float v) { return reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
  __device__ __forceinline__ int max(int v) {
    return across(__reduce_max_sync(0xffffffffu, v), [](int a, int b) { return a < b ? b : a; });
  }
  __device__ __forceinline__ unsigned max(unsigned v) {
    return across(__reduce_max_sync(0xffffffffu, v), [](unsigned a, unsigned b) { return a < b ? b : a; });
  }
  __device__ __forceinline__ unsigned min(unsigned v) { return ~max(~v); }

 private:
  template <typename T, typename Op>
  __device__ __forceinline__ T across(T v, Op op) {
    if constexpr (G > 32) {
      v = exchange(v);
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
  }
};

// launch(storage type, words moved at a time), `wide`: 16 bytes.
template <typename F>
void with_type(int dtype, bool wide, F launch) {
  using std::integral_constant;
  if (dtype == kDtypeBf16) {
    if (wide) launch(bf16{}, integral_constant<int, 8>{});
    else launch(bf16{}, integral_constant<int, 1>{});
  } else {
    if (wide) launch(float{}, integral_constant<int, 4>{});
    else launch(float{}, integral_constant<int, 1>{});
  }
}

// Order-preserving integer of a score: NaN above everything, -0 as +0; 0 is below every score.
__device__ __forceinline__ unsigned score_key(float z) {
  if (z != z) return 0xffffffffu;
  const unsigned u = __float_as_uint(z + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_score(unsigned k) {
  return __uint_as_float(k ^ ((unsigned)((int)~k >> 31) | 0x80000000u));
}

}  // namespace tb200
