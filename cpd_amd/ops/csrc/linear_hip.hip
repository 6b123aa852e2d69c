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
#include <type_traits>

#include "gemm_tiles.h"

namespace cpd {
namespace {

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
// 16-bit products by tiles (gemm_tiles.h)
// ---------------------------------------------------------------------------

// Blocks go to the eight XCDs in turn, and each XCD has its own L2: give each
// a run of neighbouring tiles, in bands of eight rows of tiles.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& m, int& n) {
  const int all = tm * tn, each = all / 8, over = all % 8;
  const int xcd = id % 8;
  id = id / 8 + xcd * each + (xcd < over ? xcd : over);
  const int band = id / (8 * tn);
  const int rows = tm - band * 8 < 8 ? tm - band * 8 : 8;
  id -= band * 8 * tn;
  m = band * 8 + id % rows;
  n = id / rows;
}

// Eight neighbouring results of a row: bias, z, activation, residual.
template <typename T>
__device__ __forceinline__ void finish8(const GemmArgs& g, int row, int col,
                                        float (&v)[8], const float* bias) {
  const int left = g.n - col;
  if (row >= g.m || left <= 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (g.z) store_vec<T>(static_cast<T*>(g.z) + (long)row * g.n + col, left, v);
  if (g.act == Act::relu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], Act::relu);
  } else if (g.act == Act::gelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], Act::gelu);
  } else if (g.act == Act::silu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], Act::silu);
  }
  if (g.res) {
    float r[8];
    load_vec<T>(static_cast<const T*>(g.res) + (long)row * g.res_ld + col, left,
                0.f, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store_vec<T>(static_cast<T*>(g.y) + (long)row * g.y_ld + col, left, v);
}

template <typename T>
__device__ __forceinline__ void leave_finished(const GemmArgs& g, char* lds,
                                               f32x4 (&v)[4][4], int row0,
                                               int col0, int lane) {
  float bias[8] = {};
  const int col = col0 + (lane & 7) * 8;
  if (g.bias) load_learned<8>(g.bias, g.bias_dt, col, g.n - col, bias);
  leave(lds, v, lane, [&](int row, int c, float (&out)[8]) {
    finish8<T>(g, row0 + row, col0 + c, out, bias);
  });
}

// 256 by 256 results, eight waves, one block a CU.  Each wave has 64 rows of
// either half of A by 32 of either half of B (B's halves are woven, so that
// those are 64 neighbouring columns); a tile of 64 k is four phases, one for
// each pair of halves.  A phase first reads what it needs from LDS
// and orders copies for later tiles, then runs 16 matrix instructions; the
// two parts are set apart by barriers, and waves 4-7 run one part behind waves
// 0-3, so that on each SIMD one wave computes while the other one reads.
//
// LDS has two tiles.  A half tile is ordered as soon as its place is free:
// A0, B0 and B1 of tile t + 2 in phases 1, 2 and 3 of tile t (their places
// were last read in phases 0, 0 and 1), A1 of tile t + 1 in phase 0.  So at
// the end of a phase everything but the newest five halves (ten copies a
// lane) has to have landed, and a copy has more than a tile's time to do so.
template <typename T, bool AX, bool BX>
__global__ __launch_bounds__(512, 2) void gemm_256_kernel(GemmArgs g, int tm,
                                                          int tn) {
  __shared__ __attribute__((aligned(1024))) char lds[8 * kHalf];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bm, bn;
  tile_of(blockIdx.x, tm, tn, bm, bn);
  const int m0 = bm * 256, n0 = bn * 256;
  const int wm = (wave >> 2) * 64, wn = (wave & 3) * 32;
  const u32 lds0 = lds_address(lds);
  Copier<AX, 8, false> ca;
  Copier<BX, 8, true> cb;
  ca.start(g.a, m0, g.m, wave, lane);
  cb.start(g.b, n0, g.n, wave, lane);
  const int tiles = g.k / kTileK, left = g.k % kTileK;

  // places of the halves: [buffer][A0 A1 B0 B1]
  auto copy_a = [&](int t, int h) {
    ca.half(t, h, lds0 + (t & 1) * (4 * kHalf) + h * kHalf);
  };
  auto copy_b = [&](int t, int h) {
    cb.half(t, h, lds0 + (t & 1) * (4 * kHalf) + (2 + h) * kHalf);
  };

  f32x4 acc[2][4][4] = {};  // half of A, 16 rows, 16 columns
  s16x8 fa[4][2], fb[2][2][2];

  auto read_a = [&](const char* buf, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        fa[i][kk] = fragment<AX>(buf + h * kHalf, wm + i * 16, kk, lane);
  };
  auto read_b = [&](const char* buf, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        fb[h][j][kk] = fragment<BX>(buf + (2 + h) * kHalf, wn + j * 16, kk, lane);
  };
  auto multiply = [&](f32x4 (&c)[4][4], int h) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[i][h * 2 + j] = mfma<T>(fb[h][j][kk], fa[i][kk], c[i][h * 2 + j]);
    __builtin_amdgcn_s_setprio(0);
  };

  if (tiles > 0) {
    copy_a(0, 0);
    copy_b(0, 0);
    copy_b(0, 1);
    copy_a(0, 1);
    if (tiles > 1) {
      copy_a(1, 0);
      copy_b(1, 0);
      copy_b(1, 1);
    }
    if (tiles > 1)
      wait_copies<10>();
    else
      wait_copies<0>();
    block_barrier();
    if (wave >= 4) block_barrier();

    auto tile = [&](int t, auto last) {
      // `last`: one of the last two tiles, which order less and wait for all
      constexpr bool LAST = decltype(last)::value;
      constexpr int NEW = LAST ? 0 : 10;
      const char* buf = lds + (t & 1) * (4 * kHalf);
      read_a(buf, 0);
      read_b(buf, 0);
      if (!LAST || t + 1 < tiles) copy_a(t + 1, 1);
      wait_copies<NEW>();
      block_barrier();
      multiply(acc[0], 0);
      block_barrier();

      read_b(buf, 1);
      if (!LAST) copy_a(t + 2, 0);
      wait_copies<NEW>();
      block_barrier();
      multiply(acc[0], 1);
      block_barrier();

      read_a(buf, 1);
      if (!LAST) copy_b(t + 2, 0);
      wait_copies<NEW>();
      block_barrier();
      multiply(acc[1], 1);
      block_barrier();

      if (!LAST) copy_b(t + 2, 1);
      wait_copies<NEW>();
      block_barrier();
      multiply(acc[1], 0);
      block_barrier();
    };
    int t = 0;
    for (; t + 2 < tiles; ++t) tile(t, std::false_type{});
    for (; t < tiles; ++t) tile(t, std::true_type{});
    if (wave < 4) block_barrier();
  }
  if (left) {
    ca.rest(tiles, 0, lds, left, lane);
    ca.rest(tiles, 1, lds + kHalf, left, lane);
    cb.rest(tiles, 0, lds + 2 * kHalf, left, lane);
    cb.rest(tiles, 1, lds + 3 * kHalf, left, lane);
    __syncthreads();
    read_b(lds, 0);
    read_b(lds, 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      read_a(lds, h);
      multiply(acc[h], 0);
      multiply(acc[h], 1);
    }
  }

  __syncthreads();  // the tiles have been read
#pragma unroll
  for (int h = 0; h < 2; ++h)
    leave_finished<T>(g, lds + wave * kHalf, acc[h], m0 + h * 128 + wm,
                      n0 + (wave & 3) * 64, lane);
}

// 128 by 128 results, four waves of 64 by 64, two blocks a CU; the tiles of k
// may be shared out over `slices` blocks, whose sums then go to `part` as
// they are.  One barrier a tile: a wave that has passed it has its copies of
// this tile and knows that the others are done with the one before.
template <typename T, bool AX, bool BX>
__global__ __launch_bounds__(256, 2) void gemm_128_kernel(GemmArgs g, int tm,
                                                          int tn, int slices,
                                                          float* part) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * kHalf];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slice = blockIdx.x / (tm * tn);
  int bm, bn;
  tile_of(blockIdx.x % (tm * tn), tm, tn, bm, bn);
  const int m0 = bm * 128, n0 = bn * 128;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const u32 lds0 = lds_address(lds);
  Copier<AX, 4, false> ca;
  Copier<BX, 4, false> cb;
  ca.start(g.a, m0, g.m, wave, lane);
  cb.start(g.b, n0, g.n, wave, lane);
  const int whole = g.k / kTileK;
  const int per = (whole + slices - 1) / slices;
  const int from = min(slice * per, whole), to = min(from + per, whole);
  const int left = slice == slices - 1 ? g.k % kTileK : 0;

  f32x4 acc[4][4] = {};
  auto copy = [&](int t, int buf) {
    ca.half(t, 0, lds0 + buf * (2 * kHalf));
    cb.half(t, 0, lds0 + buf * (2 * kHalf) + kHalf);
  };
  auto compute = [&](const char* buf) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      s16x8 fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[i] = fragment<AX>(buf, wm + i * 16, kk, lane);
        fb[i] = fragment<BX>(buf + kHalf, wn + i * 16, kk, lane);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fb[j], fa[i], acc[i][j]);
    }
  };
  if (from < to) copy(from, 0);
  for (int t = from; t < to; ++t) {
    const int buf = (t - from) & 1;
    wait_copies<0>();
    block_barrier();
    if (t + 1 < to) copy(t + 1, buf ^ 1);
    compute(lds + buf * (2 * kHalf));
  }
  if (left) {
    __syncthreads();
    ca.rest(whole, 0, lds, left, lane);
    cb.rest(whole, 0, lds + kHalf, left, lane);
    __syncthreads();
    compute(lds);
  }
  __syncthreads();
  if (!part) {
    leave_finished<T>(g, lds + wave * kHalf, acc, m0 + wm, n0 + wn, lane);
    return;
  }
  leave(lds + wave * kHalf, acc, lane, [&](int row, int col, float (&out)[8]) {
    row += m0 + wm;
    col += n0 + wn;
    if (row >= g.m) return;
    float* p = part + ((long)slice * g.m + row) * g.n + col;
    store_vec<float>(p, g.n - col, out);
    store_vec<float>(p + 4, g.n - col - 4, out + 4);
  });
}

// The slices' sums, in order, and what follows the product.
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs g, int slices,
                                                        const float* part) {
  const int chunks = (g.n + 7) / 8;
  const long all = (long)g.m * chunks;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all;
       i += (long)gridDim.x * 256) {
    const int row = (int)(i / chunks), col = (int)(i % chunks) * 8;
    float v[8] = {}, bias[8] = {};
    for (int s = 0; s < slices; ++s) {
      float u[8];
      load_some<float, 8>(part + ((long)s * g.m + row) * g.n + col, g.n - col, u);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += u[q];
    }
    if (g.bias) load_learned<8>(g.bias, g.bias_dt, col, g.n - col, bias);
    finish8<T>(g, row, col, v, bias);
  }
}

// How a 16-bit product is cut up.
struct Plan {
  int tile;    // 256 or 128
  int slices;  // of k, for 128
};

Plan plan_for(long m, long n, long k) {
  if (m < 1 || n < 1) return {128, 1};  // nothing will be launched
  const long big = ((m + 255) / 256) * ((n + 255) / 256);
  if (big >= 192) return {256, 1};
  const long small = ((m + 127) / 128) * ((n + 127) / 128);
  long slices = (512 + small - 1) / small;  // two blocks a CU
  const long most = k / (kTileK * 4);       // four tiles a slice at least
  if (slices > most) slices = most;
  return {128, (int)(slices < 1 ? 1 : slices)};
}

template <typename T, bool AX, bool BX>
void gemm_tiles_t(const GemmArgs& g, hipStream_t st) {
  const Plan p = plan_for(g.m, g.n, g.k);
  const int tm = (g.m + p.tile - 1) / p.tile, tn = (g.n + p.tile - 1) / p.tile;
  if (p.tile == 256) {
    gemm_256_kernel<T, AX, BX><<<dim3(tm * tn), dim3(512), 0, st>>>(g, tm, tn);
    return;
  }
  float* part = p.slices > 1 ? g.work : nullptr;
  gemm_128_kernel<T, AX, BX><<<dim3(tm * tn * p.slices), dim3(256), 0, st>>>(
      g, tm, tn, p.slices, part);
  if (part) {
    const long blocks = ((long)g.m * ((g.n + 7) / 8) + 255) / 256;
    gemm_join_kernel<T><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)),
                          dim3(256), 0, st>>>(g, p.slices, part);
  }
}

template <typename T>
void gemm_tiles(const GemmArgs& g, hipStream_t st) {
  if (!g.a.across && !g.b.across)
    gemm_tiles_t<T, false, false>(g, st);
  else if (!g.a.across)
    gemm_tiles_t<T, false, true>(g, st);
  else
    gemm_tiles_t<T, true, true>(g, st);
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
    gemm_tiles<bf16_t>(g, st);
  else
    gemm_tiles<f16_t>(g, st);
}

long gemm_work_floats(long m, long n, long k, Dt dt) {
  if (dt == Dt::f32) return 0;
  const Plan p = plan_for(m, n, k);
  return p.slices > 1 ? p.slices * m * n : 0;
}

bool gemm_takes(const Operand& o, long rows) {
  return (uintptr_t)o.p % 16 == 0 && o.ld % 8 == 0 &&
         (!o.across || rows % 8 == 0 || o.padded);
}

namespace {
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(const T* from, long ld,
                                                       T* to, long to_ld,
                                                       int rows, int cols) {
  const int chunks = (int)(to_ld / 8);
  const long all = (long)rows * chunks;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all;
       i += (long)gridDim.x * 256) {
    const long row = i / chunks;
    const int col = (int)(i % chunks) * 8;
    float v[8];
    load_some<T, 8>(from + row * ld + col, cols - col, v);
    store_vec<T>(to + row * to_ld + col, 8, v);
  }
}
}  // namespace

void pad_rows(const void* from, long ld, void* to, long to_ld, int rows,
              int cols, Dt dt, hipStream_t st) {
  const long all = (long)rows * (to_ld / 8), blocks = (all + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  if (dt == Dt::bf16)
    pad_rows_kernel<bf16_t><<<grid, dim3(256), 0, st>>>(
        static_cast<const bf16_t*>(from), ld, static_cast<bf16_t*>(to), to_ld,
        rows, cols);
  else
    pad_rows_kernel<f16_t><<<grid, dim3(256), 0, st>>>(
        static_cast<const f16_t*>(from), ld, static_cast<f16_t*>(to), to_ld,
        rows, cols);
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
