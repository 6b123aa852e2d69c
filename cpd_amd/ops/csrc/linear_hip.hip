// Linear layer with its epilogue for gfx950:
//
//   z = x W^T + bias,   y = act(z) + residual
//
// and backward, with dz = dy * act'(z):
//
//   dx = dz W,   dW = dz^T x,   dbias = sum over rows of dz,   dresidual = dy
//
// All three products run on the matrix cores with 32-bit accumulators; what
// follows a product (bias, activation, residual) is applied to the
// accumulators before the one rounding to the output's type.
#include "fused_ops.h"

namespace cpd {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

__device__ __forceinline__ float act_value(float z, Act act) {
  switch (act) {
    case Act::relu:
      return z > 0.f || z != z ? z : 0.f;
    case Act::gelu:
      return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case Act::silu:
      return z / (1.f + expf(-z));
    default:
      return z;
  }
}

// (relu's is a choice, not a factor: an infinite gradient times zero is NaN)
__device__ __forceinline__ float act_slope(float z, Act act) {
  switch (act) {
    case Act::gelu:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
             z * 0.3989422804014327f * expf(-0.5f * z * z);
    case Act::silu: {
      const float s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    default:
      return 1.f;
  }
}

// y and z of one element.
template <typename T>
__device__ __forceinline__ void finish(const GemmArgs& g, int row, int col,
                                       float v, float bias) {
  v += bias;
  if (g.z) static_cast<T*>(g.z)[(long)row * g.n + col] = (T)v;
  v = act_value(v, g.act);
  if (g.res)
    v += (float)static_cast<const T*>(g.res)[(long)row * g.res_ld + col];
  static_cast<T*>(g.y)[(long)row * g.y_ld + col] = (T)v;
}

// ---------------------------------------------------------------------------
// Any sizes, strides and alignment: 64x64 tile, four waves of 32x32.
// ---------------------------------------------------------------------------

template <typename T>
constexpr int kAnyK = 64 / sizeof(T);  // k of a tile: 64 bytes

// A 64-row tile of an operand into LDS as [row][k]; zeros behind its ends.
template <typename T>
__device__ __forceinline__ void any_stage(const Operand& o, int row0, int rows,
                                          int k0, int k,
                                          T (*to)[kAnyK<T> + 16 / sizeof(T)]) {
  constexpr int BK = kAnyK<T>, VEC = 16 / sizeof(T);
  const T* p = static_cast<const T*>(o.p);
  typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  // 64 * BK elements, one vector a thread
  if (!o.across) {
    const int r = threadIdx.x / (BK / VEC), c = threadIdx.x % (BK / VEC) * VEC;
    const int left = row0 + r < rows ? k - (k0 + c) : 0;
    const T* at = p + (long)(row0 + r) * o.ld + k0 + c;
    V v = {};
    if (left >= VEC) {
      v = *reinterpret_cast<const V*>(at);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < left) v[i] = at[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) to[r][c + i] = v[i];
  } else {
    const int kk = threadIdx.x / (64 / VEC), r = threadIdx.x % (64 / VEC) * VEC;
    const int left = k0 + kk < k ? rows - (row0 + r) : 0;
    const T* at = p + (long)(k0 + kk) * o.ld + row0 + r;
    V v = {};
    if (left >= VEC) {
      v = *reinterpret_cast<const V*>(at);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < left) v[i] = at[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) to[r + i][kk] = v[i];
  }
}

template <typename T>
__device__ __forceinline__ f32x4 mfma_row(const T* a, const T* b, int lane,
                                          f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma_row<bf16_t>(const bf16_t* a,
                                                  const bf16_t* b, int lane,
                                                  f32x4 c) {
  const int k = (lane >> 4) * 8;
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      *reinterpret_cast<const bf16x8*>(a + k),
      *reinterpret_cast<const bf16x8*>(b + k), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_row<f16_t>(const f16_t* a,
                                                 const f16_t* b, int lane,
                                                 f32x4 c) {
  const int k = (lane >> 4) * 8;
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      *reinterpret_cast<const f16x8*>(a + k),
      *reinterpret_cast<const f16x8*>(b + k), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_row<float>(const float* a,
                                                 const float* b, int lane,
                                                 f32x4 c) {
#pragma unroll
  for (int k = 0; k < 16; k += 4)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k + (lane >> 4)],
                                             b[k + (lane >> 4)], c, 0, 0, 0);
  return c;
}

template <typename T>
__global__ __launch_bounds__(256) void gemm_any_kernel(GemmArgs g, int tiles_n) {
  constexpr int BK = kAnyK<T>;
  __shared__ __attribute__((aligned(16))) T as[64][BK + 16 / sizeof(T)];
  __shared__ __attribute__((aligned(16))) T bs[64][BK + 16 / sizeof(T)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = (int)(blockIdx.x / tiles_n) * 64;
  const int n0 = (int)(blockIdx.x % tiles_n) * 64;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < g.k; k0 += BK) {
    __syncthreads();
    any_stage<T>(g.a, m0, g.m, k0, g.k, as);
    any_stage<T>(g.b, n0, g.n, k0, g.k, bs);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = mfma_row<T>(as[wm + i * 16 + (lane & 15)],
                                bs[wn + j * 16 + (lane & 15)], lane, acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int col = n0 + wn + j * 16 + (lane & 15);
    if (col >= g.n) continue;
    float bias = 0.f;
    if (g.bias) load_learned<1>(g.bias, g.bias_dt, col, 1, &bias);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m0 + wm + i * 16 + (lane >> 4) * 4 + r;
        if (row < g.m) finish<T>(g, row, col, acc[i][j][r], bias);
      }
  }
}

template <typename T>
void gemm_any(const GemmArgs& g, hipStream_t st) {
  const long tm = ((long)g.m + 63) / 64, tn = ((long)g.n + 63) / 64;
  gemm_any_kernel<T><<<dim3((unsigned)(tm * tn)), dim3(256), 0, st>>>(g, (int)tn);
}

// ---------------------------------------------------------------------------
// The activation's gradient and the sums of its columns
// ---------------------------------------------------------------------------

// A block has 64 vectors of columns and a slice of the rows, its four waves
// every fourth row of it.  The sums go over slices in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void act_grad_kernel(ActGradArgs a,
                                                       int rows_per) {
  constexpr int VEC = Vec16<T>::N;
  __shared__ float add[4][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = (int)(blockIdx.x * 64 + lane) * VEC;
  const int left = a.n - col;
  const int from = blockIdx.y * rows_per;
  const int to = a.m - from < rows_per ? a.m : from + rows_per;
  float sum[VEC] = {};
  if (left > 0) {
    for (int row = from + wave; row < to; row += 4) {
      float g[VEC];
      load_vec<T>(static_cast<const T*>(a.dy) + (long)row * a.dy_ld + col, left,
                  0.f, g);
      if (a.act != Act::none) {
        float z[VEC];
        load_vec<T>(static_cast<const T*>(a.z) + (long)row * a.z_ld + col, left,
                    0.f, z);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          g[i] = a.act == Act::relu ? (z[i] > 0.f ? g[i] : 0.f)
                                    : g[i] * act_slope(z[i], a.act);
      }
      if (a.dz)
        store_vec<T>(static_cast<T*>(a.dz) + (long)row * a.dz_ld + col, left, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] += g[i];
    }
  }
  if (!a.dbias) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) add[wave][i * 64 + lane] = sum[i];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < left)
        a.partial[(long)blockIdx.y * a.n + col + i] =
            add[0][i * 64 + lane] + add[1][i * 64 + lane] +
            add[2][i * 64 + lane] + add[3][i * 64 + lane];
  }
}

__global__ __launch_bounds__(256) void column_join_kernel(
    const float* __restrict__ partial, int slices, int n, void* out, Dt dt) {
  __shared__ float add[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = (int)(blockIdx.x * 64 + lane);
  float t = 0.f;
  if (col < n)
    for (int s = wave; s < slices; s += 4) t += partial[(long)s * n + col];
  add[wave][lane] = t;
  __syncthreads();
  if (wave == 0 && col < n)
    store_as(out, dt, col,
             add[0][lane] + add[1][lane] + add[2][lane] + add[3][lane]);
}

}  // namespace

void gemm_fused(const GemmArgs& g, hipStream_t st) {
  if (g.m == 0 || g.n == 0) return;
  if (g.dt == Dt::f32)
    gemm_any<float>(g, st);
  else if (g.dt == Dt::bf16)
    gemm_any<bf16_t>(g, st);
  else
    gemm_any<f16_t>(g, st);
}

int act_grad_slices(int m, int n, Dt dt) {
  const int width = 64 * 16 / dt_size(dt);
  const int across = (n + width - 1) / width;
  int slices = (2048 + across - 1) / across;  // eight blocks a CU
  const int most = (m + 15) / 16;             // four rows a wave at least
  return slices < most ? slices : most;
}

void act_grad(const ActGradArgs& a, hipStream_t st) {
  if (a.m == 0 || a.n == 0) return;
  const int width = 64 * 16 / dt_size(a.dt);
  const int slices = act_grad_slices(a.m, a.n, a.dt);
  const int per = (a.m + slices - 1) / slices;
  const dim3 grid((a.n + width - 1) / width, slices);
  if (a.dt == Dt::f32)
    act_grad_kernel<float><<<grid, dim3(256), 0, st>>>(a, per);
  else if (a.dt == Dt::bf16)
    act_grad_kernel<bf16_t><<<grid, dim3(256), 0, st>>>(a, per);
  else
    act_grad_kernel<f16_t><<<grid, dim3(256), 0, st>>>(a, per);
  if (a.dbias)
    column_join_kernel<<<dim3((a.n + 63) / 64), dim3(256), 0, st>>>(
        a.partial, slices, a.n, a.dbias, a.bias_dt);
}

}  // namespace cpd
