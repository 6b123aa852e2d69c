// Shared by the layer-norm, linear and log-probability kernels (gfx950).
//
// The three storage types, 16-byte vector access that does not ask for
// alignment, and reductions over a wave and a block.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace cpd {

using bf16_t = __bf16;
using f16_t = _Float16;

// What a tensor's elements are stored in; the launchers switch on it.
enum class Dt : int { f32 = 0, bf16 = 1, f16 = 2 };

inline int dt_size(Dt d) { return d == Dt::f32 ? 4 : 2; }

// 16 bytes of T.  The type asks only for T's own alignment: gfx950 runs with
// unaligned access on, so rows of an odd length still move as 16-byte
// accesses (they cost one more cache line now and then, not a factor).
template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// N elements from p as floats; elements at or behind `left` are `fill`.
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int left, float fill,
                                         float* out) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) {
    const auto v = *reinterpret_cast<const typename Vec16<T>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < left ? (float)p[i] : fill;
  }
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, int left, const float* in) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) {
    typename Vec16<T>::type v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)in[i];
    *reinterpret_cast<typename Vec16<T>::type*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)in[i];
  }
}

template <typename T, int N>
__device__ __forceinline__ void load_some(const T* p, int left, float* out) {
  typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  if (left >= N) {
    const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < left ? (float)p[i] : 0.f;
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_some(T* p, int left, const float* in) {
  typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  if (left >= N) {
    V v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)in[i];
    *reinterpret_cast<V*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)in[i];
  }
}

// N elements of a vector whose type is known at run time only (weights and
// biases: the activations' type, or float).
template <int N>
__device__ __forceinline__ void load_learned(const void* p, Dt dt, long at,
                                             int left, float* out) {
  if (dt == Dt::f32)
    load_some<float, N>(static_cast<const float*>(p) + at, left, out);
  else if (dt == Dt::bf16)
    load_some<bf16_t, N>(static_cast<const bf16_t*>(p) + at, left, out);
  else
    load_some<f16_t, N>(static_cast<const f16_t*>(p) + at, left, out);
}

__device__ __forceinline__ void store_as(void* p, Dt dt, long at, float v) {
  if (dt == Dt::f32)
    static_cast<float*>(p)[at] = v;
  else if (dt == Dt::bf16)
    static_cast<bf16_t*>(p)[at] = (bf16_t)v;
  else
    static_cast<f16_t*>(p)[at] = (f16_t)v;
}

// Sum over groups of `W` neighbouring lanes (a power of two up to 64); every
// lane of a group gets it.
template <int W>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int d = W / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// Sum over the TPR threads that share a row: within a wave by lanes, over
// waves through `smem` (two floats a wave; `turn` alternates 0/1 from call to
// call, so that one barrier a call is enough).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* smem, int turn) {
  if constexpr (TPR <= 64) {
    return group_sum<TPR>(v);
  } else {
    constexpr int WAVES = TPR / 64;
    v = group_sum<64>(v);
    float* s = smem + turn * WAVES;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += s[w];
    return v;
  }
}

}  // namespace cpd
