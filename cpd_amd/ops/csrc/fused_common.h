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

// 16 bytes as they are; elements at or behind `left` are `fill`.
template <typename T>
__device__ __forceinline__ typename Vec16<T>::type load_raw(const T* p, int left,
                                                            T fill = (T)0.f) {
  typedef typename Vec16<T>::type V;
  if (left >= Vec16<T>::N) return *reinterpret_cast<const V*>(p);
  V v;
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) {
    v[i] = fill;
    if (i < left) v[i] = p[i];
  }
  return v;
}

// v of the lane `N` places on within its 16 lanes, round and round.
template <int N>
__device__ __forceinline__ float rotate16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(
      0, __float_as_int(v), 0x120 + N, 0xf, 0xf, true));
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Sum over groups of `W` = 16 or 64 neighbouring lanes, all of them active;
// every lane of a group gets it.  (Rotations within the instruction: a shuffle
// through LDS takes ten times as long.)
template <int W>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(W == 16 || W == 64, "a quarter of a wave, or a wave");
  v += rotate16<8>(v);
  v += rotate16<4>(v);
  v += rotate16<2>(v);
  v += rotate16<1>(v);
  if constexpr (W == 64)
    v = (lane_value(v, 0) + lane_value(v, 16)) +
        (lane_value(v, 32) + lane_value(v, 48));
  return v;
}

// The largest of a wave's values, NaN passed over.
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, rotate16<8>(v));
  v = fmaxf(v, rotate16<4>(v));
  v = fmaxf(v, rotate16<2>(v));
  v = fmaxf(v, rotate16<1>(v));
  return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)),
               fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// Sums of two values over the TPR threads that share a row: within a wave by
// lanes, over waves through `smem` (4 TPR/64 floats).  `turn` alternates 0/1
// from call to call, so that one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float* smem,
                                         int turn) {
  constexpr int WAVES = TPR / 64;
  if constexpr (TPR <= 64) {
    a = group_sum<TPR>(a);
    b = group_sum<TPR>(b);
  } else {
    a = group_sum<64>(a);
    b = group_sum<64>(b);
    float* s = smem + turn * 2 * WAVES;
    if ((threadIdx.x & 63) == 0) {
      s[threadIdx.x >> 6] = a;
      s[WAVES + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      a += s[w];
      b += s[WAVES + w];
    }
  }
}

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* smem, int turn) {
  float none = 0.f;
  row_sums<TPR>(v, none, smem, turn);
  return v;
}

}  // namespace cpd
