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
//
// bf16 at 8192^3: 1.46 PFLOP/s forward, 1.32 dx, 1.31 dW (the library's plain
// product: 1.48, 1.39, 1.20); 2048^3: 0.83; floats at 8192 x 2048 x 8192: 0.21.
#include <type_traits>
#include <utility>

#include "gemm_tiles.h"

namespace cpd {
namespace {

// The activations and their slopes.  What is stored in 16 bits takes the
// machine's exp2 and reciprocal (1 ulp each) and, for the normal distribution's
// cdf, the polynomial of Abramowitz and Stegun 7.1.26 (1.5e-7 off at most, a
// two-thousandth of fp16's half step at 1; of gelu's own value in the far tail
// 7e-4 at -4.2, 3e-3 at -5.7 and 7e-3 at -7.1, where that is 5e-12), whose
// exponential is the density's too: erff alone is some 40 instructions, which
// bound the gradient's pass.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
  return EXACT ? expf(x) : __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}
template <bool EXACT>
__device__ __forceinline__ float inverse(float x) {
  return EXACT ? 1.f / x : __builtin_amdgcn_rcpf(x);
}

// The normal distribution's cdf at z, and its density there if asked for.
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float* density) {
  const float e = density || !EXACT ? exp_of<EXACT>(-0.5f * z * z) : 0.f;
  if (density) *density = 0.3989422804014327f * e;
  if constexpr (EXACT) {
    return 0.5f * (1.f + erff(z * 0.70710678118654752f));
  } else {
    const float t = inverse<false>(1.f + 0.3275911f * 0.70710678118654752f *
                                             fabsf(z));
    float p = 1.061405429f;
    p = p * t - 1.453152027f;
    p = p * t + 1.421413741f;
    p = p * t - 0.284496736f;
    p = p * t + 0.254829592f;
    const float tail = 0.5f * p * t * e;
    return z < 0.f ? tail : 1.f - tail;
  }
}

template <typename T>
__device__ __forceinline__ float act_value(float z, Act act) {
  constexpr bool EXACT = __is_same(T, float);
  switch (act) {
    case Act::relu:
      return z > 0.f || z != z ? z : 0.f;
    case Act::gelu:
      return z * normal_cdf<EXACT>(z, nullptr);
    case Act::silu:
      return z * inverse<EXACT>(1.f + exp_of<EXACT>(-z));
    default:
      return z;
  }
}

// (relu's is a choice, not a factor: an infinite gradient times zero is NaN.  An
// argument that 16 bits do not hold is kept as an infinity, where the slopes have
// their limits: 0 and 1.)
template <typename T>
__device__ __forceinline__ float act_slope(float z, Act act) {
  constexpr bool EXACT = __is_same(T, float);
  if (!EXACT && fabsf(z) == INFINITY) return z > 0.f ? 1.f : 0.f;
  switch (act) {
    case Act::gelu: {
      float density;
      const float cdf = normal_cdf<EXACT>(z, &density);
      return cdf + z * density;
    }
    case Act::silu: {
      const float s = inverse<EXACT>(1.f + exp_of<EXACT>(-z));
      return s * (1.f + z * (1.f - s));
    }
    default:
      return 1.f;
  }
}

// ---------------------------------------------------------------------------
// Products by tiles (gemm_tiles.h)
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

// N neighbouring results of a row: bias, z, activation, residual.
template <typename T, int N>
__device__ __forceinline__ void finish(const GemmArgs& g, int row, int col,
                                       float (&v)[N], const float* bias) {
  const int left = g.n - col;
  if (row >= g.m || left <= 0) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += bias[i];
  if (g.z)
    store_some<T, N>(static_cast<T*>(g.z) + (long)row * g.n + col, left, v);
  if (g.act == Act::relu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_value<T>(v[i], Act::relu);
  } else if (g.act == Act::gelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_value<T>(v[i], Act::gelu);
  } else if (g.act == Act::silu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_value<T>(v[i], Act::silu);
  }
  if (g.res) {
    float r[N];
    load_some<T, N>(static_cast<const T*>(g.res) + (long)row * g.res_ld + col,
                    left, r);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += r[i];
  }
  store_some<T, N>(static_cast<T*>(g.y) + (long)row * g.y_ld + col, left, v);
}

template <typename T, int F>
__device__ __forceinline__ void leave_finished(const GemmArgs& g, char* lds,
                                               const f32x4 (*v)[4], int row0,
                                               int col0, int lane) {
  float bias[8] = {};
  const int col = col0 + (lane & 7) * 8;
  if (g.bias) load_learned<8>(g.bias, g.bias_dt, col, g.n - col, bias);
  leave<F>(lds, v, lane, [&](int row, int c, float (&out)[8]) {
    finish<T, 8>(g, row0 + row, col0 + c, out, bias);
  });
}

// The same, or a slice's sums to the workspace.
template <typename T, int F>
__device__ __forceinline__ void leave_block(const GemmArgs& g, char* lds,
                                            const f32x4 (*v)[4], int row0,
                                            int col0, int lane, int slice) {
  if (g.slices == 1) {
    leave_finished<T, F>(g, lds, v, row0, col0, lane);
    return;
  }
  leave<F>(lds, v, lane, [&](int row, int col, float (&out)[8]) {
    row += row0;
    col += col0;
    if (row < g.m && col < g.n)
      store_some<float, 8>(g.work + ((long)slice * g.m + row) * g.n + col,
                           g.n - col, out);
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
__device__ __forceinline__ void tile_256(const GemmArgs& g, int id, char* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bm, bn;
  tile_of(id, (g.m + 255) / 256, (g.n + 255) / 256, bm, bn);
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
    leave_finished<T, 4>(g, lds + wave * kHalf, acc[h], m0 + h * 128 + wm,
                      n0 + (wave & 3) * 64, lane);
}

// 128 by 128 results, eight waves, one block a CU: four of 64 by 64 on the
// first 32 k of a tile, four on the other 32.  LDS has four tiles, and a tile
// is read into registers one step before it is multiplied, so that LDS reads
// go on under the matrix instructions (read and multiplied in the same step a
// tile took 0.74 us) and copies have three steps to land.  One barrier a
// step: a wave that has passed it has its copies of tile t + 1 and knows that
// all have read tile t, whose place tile t + 4 takes.  The tiles of k may be
// shared out over `slices` blocks, whose sums then go to the workspace as they are.
template <typename T, bool AX, bool BX>
__device__ __forceinline__ void tile_128(const GemmArgs& g, int id, char* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tm = (g.m + 127) / 128, tn = (g.n + 127) / 128, slices = g.slices;
  const int slice = id / (tm * tn);
  int bm, bn;
  tile_of(id % (tm * tn), tm, tn, bm, bn);
  const int m0 = bm * 128, n0 = bn * 128;
  const int wk = wave >> 2, wm = (wave >> 1 & 1) * 64, wn = (wave & 1) * 64;
  const u32 lds0 = lds_address(lds);
  Copier<AX, 8, false> ca;
  Copier<BX, 8, false> cb;
  ca.start(g.a, m0, g.m, wave, lane);
  cb.start(g.b, n0, g.n, wave, lane);
  const int whole = g.k / kTileK;
  const int per = (whole + slices - 1) / slices;
  const int from = min(slice * per, whole), to = min(from + per, whole);
  const int left = slice == slices - 1 ? g.k % kTileK : 0;

  f32x4 acc[4][4] = {};
  // With one row of tiles, blocks are bound by reading B, and with its rows a
  // multiple of 4 KB apart all that is read at a time, 128 bytes a row, lies on a
  // few memory channels: each block begins elsewhere in its k (48 rows with
  // 134 MB, k 16384: 35 us, 41 without).
  const bool apart = tm == 1 && !BX && (g.b.ld * 2) % 4096 == 0 && to > from;
  const int turn = apart ? (bn * 5 + slice * 3) % (to - from) : 0;
  auto copy = [&](int t) {
    const u32 at = lds0 + ((t - from) & 3) * (2 * kHalf);
    int k = t + turn;
    k = k < to ? k : k - (to - from);
    ca.half(k, 0, at);
    cb.half(k, 0, at + kHalf);
  };
  struct Fragments {
    s16x8 a[4], b[4];
  };
  auto read = [&](const char* buf, Fragments& f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.a[i] = fragment<AX>(buf, wm + i * 16, wk, lane);
      f.b[i] = fragment<BX>(buf + kHalf, wn + i * 16, wk, lane);
    }
  };
  auto multiply = [&](const Fragments& f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] = mfma<T>(f.b[j], f.a[i], acc[i][j]);
  };
  Fragments f0, f1;
  if (from < to) {
    for (int t = from; t < min(from + 4, to); ++t) copy(t);
    // four copies a lane for each tile
    if (from + 4 <= to)
      wait_copies<12>();
    else
      wait_copies<0>();
    block_barrier();
    read(lds, f0);
  }
  // (No branch around the reads, and nothing moved across them: where the
  // compiler cannot tell how many LDS reads are in flight, the matrix
  // instructions wait for all of them, and left to itself it reads behind them.)
  auto step = [&](int t, const Fragments& now, Fragments& next, auto steady) {
    constexpr bool STEADY = decltype(steady)::value;
    if (STEADY || t + 3 < to)
      wait_copies<8>();
    else
      wait_copies<0>();
    block_barrier();
    if (STEADY || t + 4 < to) copy(t + 4);
    read(lds + ((t + 1 - from) & 3) * (2 * kHalf), next);
    __builtin_amdgcn_sched_barrier(0);
    multiply(now);
  };
  const std::true_type steady;
  const std::false_type ending;
  int t = from;
  for (; t + 5 < to; t += 2) {
    step(t, f0, f1, steady);
    step(t + 1, f1, f0, steady);
  }
  for (; t + 2 < to; t += 2) {
    step(t, f0, f1, ending);
    step(t + 1, f1, f0, ending);
  }
  if (t + 1 < to) {
    step(t, f0, f1, ending);
    multiply(f1);
  } else if (t < to) {
    multiply(f0);
  }
  __syncthreads();
  if (left) {
    ca.rest(whole, 0, lds, left, lane);
    cb.rest(whole, 0, lds + kHalf, left, lane);
    __syncthreads();
    read(lds, f0);
    multiply(f0);
    __syncthreads();
  }
  // the two halves of k: each wave finishes 32 of its 64 rows
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4*>(lds + wave * 8192 + (i * 4 + j) * 1024 +
                                lane * 16) = wk ? acc[i][j] : acc[2 + i][j];
  __syncthreads();
  f32x4 out[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      out[i][j] = (wk ? acc[2 + i][j] : acc[i][j]) +
                  *reinterpret_cast<const f32x4*>(
                      lds + (wave ^ 4) * 8192 + (i * 4 + j) * 1024 + lane * 16);
  __syncthreads();
  leave_block<T, 2>(g, lds + wave * 8192, out, m0 + wm + wk * 32, n0 + wn, lane,
                    slice);
}

// 128 by 128 results of floats, or of a float A and a B of T (gemm_tiles.h: P
// parts of each), tiles of 32 k.  Waves 4-11 read
// floats three tiles ahead, cut them into planes and write those to LDS; waves
// 0-3, one on each SIMD beside two of the others, multiply 64 by 64 each.  So
// the cutting goes on under the matrix instructions (1536 cycles a tile).  With
// both done by all of eight waves in turn a tile took 1.6 us, with four waves
// that cut 1.3 us, which was their time.
template <typename T, bool AX, bool BX>
__device__ __forceinline__ void tile_floats(const GemmArgs& g, int id,
                                            char* lds) {
  constexpr int P = __is_same(T, float) ? 3 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tm = (g.m + 127) / 128, tn = (g.n + 127) / 128, slices = g.slices;
  const int slice = id / (tm * tn);
  int bm, bn;
  tile_of(id % (tm * tn), tm, tn, bm, bn);
  const int m0 = bm * 128, n0 = bn * 128;
  const int all = (g.k + kFloatK - 1) / kFloatK;
  const int per = (all + slices - 1) / slices;
  const int from = min(slice * per, all), to = min(from + per, all);
  // All of the waves pass one barrier a tile, and none elsewhere.
  auto meet = [] {  // (not __syncthreads: loads stay in flight)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();
  };
  if (wave >= 4) {
    FloatStager<float, P, AX> sa;
    FloatStager<T, P, BX> sb;
    sa.start(g.a, m0, g.m, threadIdx.x - 256);
    sb.start(g.b, n0, g.n, threadIdx.x - 256);
    struct Raw {
      float a[8], b[8];
    };
    auto load = [&](int t, Raw& r) {
      if (t >= to) return;
      sa.load(t, g.k - t * kFloatK, r.a);
      sb.load(t, g.k - t * kFloatK, r.b);
    };
    // writes tile t, orders tile t + 3 in its place
    auto step = [&](int t, Raw& r) {
      if (t >= to) return;
      char* buf = lds + ((t - from) & 1) * (2 * P * kPlane);
      sa.store(buf, r.a);
      sb.store(buf + P * kPlane, r.b);
      load(t + 3, r);
      // tile t is there; and tile t - 1 has been read, whose place t + 1 takes
      meet();
    };
    Raw r0, r1, r2;
    load(from, r0);
    load(from + 1, r1);
    load(from + 2, r2);
    for (int t = from; t < to; t += 3) {
      step(t, r0);
      step(t + 1, r1);
      step(t + 2, r2);
    }
    return;
  }
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x4 acc[4][4] = {};
  for (int t = from; t < to; ++t) {
    meet();
    const char* buf = lds + ((t - from) & 1) * (2 * P * kPlane);
    s16x8 fa[P][4], fb[P][4];
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[q][i] = float_fragment<AX>(buf + q * kPlane, wm + i * 16, lane);
        fb[q][i] = float_fragment<BX>(buf + (P + q) * kPlane, wn + i * 16, lane);
      }
    // in the order in which the planes arrive
#pragma unroll
    for (int sum = 0; sum < P; ++sum)
#pragma unroll
      for (int q = 0; q <= sum; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = mfma<bf16_t>(fb[sum - q][j], fa[q][i], acc[i][j]);
  }
  // The producers wrote their last tile before the last barrier; but the other
  // waves may still be reading it, so each wave leaves through the half of LDS
  // that the last tile is not in, 4 P KB a wave: 48 rows, then 16, or 32 twice.
  char* free = lds + ((to - from) & 1) * (2 * P * kPlane) + wave * (P * 4096);
  leave_block<T, P>(g, free, acc, m0 + wm, n0 + wn, lane, slice);
  leave_block<T, 4 - P>(g, free, acc + P, m0 + wm + P * 16, n0 + wn, lane, slice);
}

// What a launch's tiles are: 256 or 128 (of floats 128 by 32 k), or kWide, those
// of a float A and a 16-bit B.
constexpr int kWide = 1;

template <typename T, int TILE>
constexpr int kThreads = __is_same(T, float) || TILE == kWide ? 768 : 512;
template <typename T, int TILE>
constexpr int kLds = __is_same(T, float) ? 12 * kPlane
                     : TILE == kWide     ? 8 * kPlane
                                         : 8 * kHalf;

template <typename T, bool AX, bool BX, int TILE>
__device__ __forceinline__ void tile_any(const GemmArgs& g, int id, char* lds) {
  if constexpr (__is_same(T, float) || TILE == kWide)
    tile_floats<T, AX, BX>(g, id, lds);
  else if constexpr (TILE == 256)
    tile_256<T, AX, BX>(g, id, lds);
  else
    tile_128<T, AX, BX>(g, id, lds);
}

template <typename T, bool AX, bool BX, int TILE>
__global__ __launch_bounds__((kThreads<T, TILE>),
                             (kThreads<T, TILE> / 256)) void gemm_kernel(GemmArgs g) {
  __shared__ __attribute__((aligned(1024))) char lds[kLds<T, TILE>];
  tile_any<T, AX, BX, TILE>(g, blockIdx.x, lds);
}

// dx and dW in one launch, so that neither's last round leaves CUs idle and
// fewer slices of k fill them: backward of 3000 x 2500 by 2500 bf16 took 131 us
// in two launches and takes 102, of 512 x 2048 by 1000 floats 56 and 46.  `first`
// blocks are dx's, or dW's if those take longer.
template <typename T, int DX, int DW>
__global__ __launch_bounds__((kThreads<T, DX>), (kThreads<T, DX> / 256)) void
gemm_two_kernel(GemmArgs dx, GemmArgs dw, int first, bool dw_first) {
  static_assert(kThreads<T, DX> == kThreads<T, DW>, "one block, one size");
  __shared__ __attribute__((aligned(1024))) char lds[kLds<T, DX>];
  const int id = blockIdx.x;
  const bool second = id >= first;
  if (second == dw_first)
    tile_any<T, false, true, DX>(dx, second ? id - first : id, lds);
  else
    tile_any<T, true, true, DW>(dw, second ? id - first : id, lds);
}

// Few rows of A (16 F), both operands along: bound by reading B once.  A block
// has 16 W rows of B; its eight waves share out k and add up through LDS.  B
// goes straight into registers, a whole 128-byte line a row at a time, and A
// comes from the caches, two batches of lines in flight a wave; nothing asks
// for alignment.  Where there are few blocks and much k, `slices` of them share
// a row's k as above.
//
// A is read once for every 16 W rows of B, which limits how many rows pay.  With
// 134 MB of 16-bit B (k 4096, k 16384, k 5000) 1 row takes 26, 29 and 34 us, 16
// take 28, 32 and 43, 32 take 36, 39 and 55, and by tiles of 128 16 take 34, 34
// and 41, 32 take 31, 33 and 42; with 34 MB 16 take 10, 32 take 14 and by tiles 15;
// with 8 MB 32 and 48 took 7 and 9, by tiles 14.  Floats of more than 16 MB go to
// gemm_narrow_kernel: with 134 MB 1, 16 and 32 rows take 30, 31 and 35 there, 32, 37
// and 48 here, and by tiles 32 take 54.
template <typename T, int F, int W>
__global__ __launch_bounds__(512) void gemm_rows_kernel(GemmArgs g) {
  constexpr int VEC = 16 / sizeof(T);    // a lane's elements of a load
  constexpr int UNIT = 128 / sizeof(T);  // k of a line; a lane has two loads
  constexpr int BATCH = F == 1 ? (W == 1 ? 4 : 2) : F == 2 && W == 1 ? 2 : 1;
  typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  __shared__ f32x4 sums[8][F * W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int blocks = (g.n + 16 * W - 1) / (16 * W);
  const int slice = blockIdx.x / blocks;
  const int n0 = (blockIdx.x % blocks) * (16 * W);
  const int units = (g.k + UNIT - 1) / UNIT;
  const int per = (units + g.slices - 1) / g.slices;
  const int from = slice * per, to = min(from + per, units);
  const int k0 = (lane >> 4) * 2 * VEC;
  // (as in tile_128: with all blocks from their first k on 1 row and k 4096 took 31
  // us instead of 26, with steps of a whole kilobyte between them 30)
  const bool apart = (g.b.ld * (long)sizeof(T)) % 4096 == 0 && to > from;
  const int turn = apart ? (int)(blockIdx.x * 5) % (to - from) : 0;
  // (rows behind the last one repeat it: their results are not stored)
  const T *a[F], *b[W];
#pragma unroll
  for (int w = 0; w < W; ++w)
    b[w] = static_cast<const T*>(g.b.p) +
           (long)min(n0 + w * 16 + (lane & 15), g.n - 1) * g.b.ld + k0;
#pragma unroll
  for (int f = 0; f < F; ++f)
    a[f] = static_cast<const T*>(g.a.p) +
           (long)min(f * 16 + (lane & 15), g.m - 1) * g.a.ld + k0;

  struct Lines {
    V b[BATCH][W][2], a[BATCH][F][2];
  };
  auto fetch = [&](const T* p, int k, bool in, V (&v)[2]) {
    const int left = in ? g.k - k - k0 : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (left >= (h + 1) * VEC) {
        v[h] = *reinterpret_cast<const V*>(p + k + h * VEC);
      } else {
        v[h] = V{};
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (h * VEC + i < left) v[h][i] = p[k + h * VEC + i];
      }
    }
  };
  // unit u and the BATCH - 1 that this wave has behind it
  auto load = [&](int u, Lines& l) {
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const bool in = u + q * 8 < to;
      const int at = u + q * 8 + turn;
      const int k = (at < to ? at : at - (to - from)) * UNIT;
#pragma unroll
      for (int w = 0; w < W; ++w) fetch(b[w], k, in, l.b[q][w]);
#pragma unroll
      for (int f = 0; f < F; ++f) fetch(a[f], k, in, l.a[q][f]);
    }
  };
  f32x4 acc[F][W] = {};
  auto multiply = [&](const Lines& l) {
#pragma unroll
    for (int q = 0; q < BATCH; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int w = 0; w < W; ++w) {
            if constexpr (__is_same(T, float)) {
              // any order of k does, if it is both operands'
#pragma unroll
              for (int i = 0; i < VEC; ++i)
                acc[f][w] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    l.b[q][w][h][i], l.a[q][f][h][i], acc[f][w], 0, 0, 0);
            } else {
              acc[f][w] = mfma<T>(__builtin_bit_cast(s16x8, l.b[q][w][h]),
                                  __builtin_bit_cast(s16x8, l.a[q][f][h]),
                                  acc[f][w]);
            }
          }
  };
  constexpr int STRIDE = 8 * BATCH;
  Lines l0, l1;
  int u = from + wave;
  if (u < to) load(u, l0);
  for (; u < to; u += 2 * STRIDE) {
    if (u + STRIDE < to) load(u + STRIDE, l1);
    multiply(l0);
    if (u + STRIDE < to) {
      if (u + 2 * STRIDE < to) load(u + 2 * STRIDE, l0);
      multiply(l1);
    }
  }
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int w = 0; w < W; ++w) sums[wave][f * W + w][lane] = acc[f][w];
  __syncthreads();
  // 16 by 16 results a wave, four neighbours a lane
  for (int i = wave; i < F * W; i += 8) {
    f32x4 t = sums[0][i][lane];
#pragma unroll
    for (int s = 1; s < 8; ++s) t += sums[s][i][lane];
    const int row = i / W * 16 + (lane & 15);
    const int col = n0 + i % W * 16 + (lane >> 4) * 4;
    float v[4] = {t[0], t[1], t[2], t[3]}, bias[4] = {};
    if (g.slices > 1) {
      if (row < g.m && col < g.n)
        store_some<float, 4>(g.work + ((long)slice * g.m + row) * g.n + col,
                             g.n - col, v);
      continue;
    }
    if (g.bias) load_learned<4>(g.bias, g.bias_dt, col, g.n - col, bias);
    finish<T, 4>(g, row, col, v, bias);
  }
}

// Few features of floats: a block has ROWS rows of one operand ("many") by all of
// at most 16 F of the other ("few"), so that many is read once, and multiplies them
// by the float matrix instructions (a tile of 128 by 128 would be cut into parts
// and multiplied for the few columns that it has).  A tile is 4096 / ROWS of k.
// Its 512 threads read three tiles ahead into registers and write to LDS, which has
// two; its eight waves have 16 rows and 32 k of a tile each, and add up through LDS.
// A fragment's eight k are 8 (lane / 16) and on: adjacent in LDS if the operand
// lies along, its chunks swizzled; RS + 2 apart if across, which keeps the four
// groups of lanes off each other's banks.
//
// Bound by reading many: 590 MB, 16384 x 9000 to 8, take 103 us forward and 110 for
// dW (5.7 and 5.4 TB/s; by tiles 182 and 202; 186 where dW follows dx, whose writes
// drain meanwhile).
template <int RS, int K, bool ACROSS>
struct NarrowStager {  // a thread's share of RS rows by K k
  static constexpr int CHUNKS = RS * K / 4;
  static constexpr int PASSES = (CHUNKS + 511) / 512;
  static constexpr int BYTES = ACROSS ? K * (RS + 2) * 4 : RS * K * 4;
  const float* p[PASSES];
  int at[PASSES];   // this thread's first k in a tile, or its k
  u32 place[PASSES];
  long step;
  int rows_left[PASSES];  // across: rows from its first on
  bool on;

  __device__ __forceinline__ void start(const Operand& o, int row0, int rows, int tid) {
    const float* base = static_cast<const float*>(o.p);
    on = tid < CHUNKS;  // (or CHUNKS is a multiple of 512)
    step = ACROSS ? K * o.ld : K;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int id = tid + 512 * i;
      if constexpr (!ACROSS) {
        const int r = id / (K / 4), chunk = id % (K / 4);
        at[i] = chunk * 4;
        rows_left[i] = 4;
        // (rows behind the last one repeat it: their results are not stored)
        p[i] = base + (long)min(row0 + r, rows - 1) * o.ld + at[i];
        place[i] = r * (K * 4) + ((chunk ^ (r & 7)) << 4);
      } else {
        const int chunk = id % (RS / 4);
        at[i] = id / (RS / 4);
        rows_left[i] = rows - (row0 + chunk * 4);
        p[i] = base + (long)at[i] * o.ld + row0 + chunk * 4;
        place[i] = (at[i] * (RS + 2) + chunk * 4) * 4;
      }
    }
  }
  // `left`: k from this tile's first on
  __device__ __forceinline__ void load(int tile, int left, float (&v)[PASSES][4]) const {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
      load_some<float, 4>(p[i] + tile * step,
                          ACROSS ? (at[i] < left ? rows_left[i] : 0) : left - at[i],
                          v[i]);
  }
  __device__ __forceinline__ void store(char* lds, const float (&v)[PASSES][4]) const {
    if (!on) return;
    typedef float V __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      if constexpr (!ACROSS) {
        *reinterpret_cast<f32x4*>(lds + place[i]) =
            f32x4{v[i][0], v[i][1], v[i][2], v[i][3]};
      } else {
        *reinterpret_cast<V*>(lds + place[i]) = V{v[i][0], v[i][1]};
        *reinterpret_cast<V*>(lds + place[i] + 8) = V{v[i][2], v[i][3]};
      }
    }
  }
  // 16 rows from `row`, 32 k from `k`
  static __device__ __forceinline__ void fragment(const char* lds, int row, int k, int lane,
                                                  float (&v)[8]) {
    const int r = row + (lane & 15), group = lane >> 4;
    if constexpr (!ACROSS) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 u = *reinterpret_cast<const f32x4*>(
            lds + r * (K * 4) + (((k / 4 + group * 2 + h) ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[h * 4 + i] = u[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = *reinterpret_cast<const float*>(lds + ((k + group * 8 + i) * (RS + 2) + r) * 4);
    }
  }
};

// MX, FX: many, few lie across.  MANY_A: many is A, otherwise B.
template <int F, int ROWS, bool MX, bool FX, bool MANY_A>
__global__ __launch_bounds__(512) void gemm_narrow_kernel(GemmArgs g) {
  constexpr int K = 4096 / ROWS, GROUPS = ROWS / 16, SHARES = 8 / GROUPS;
  using Many = NarrowStager<ROWS, K, MX>;
  using Few = NarrowStager<16 * F, K, FX>;
  constexpr int BUF = Many::BYTES + Few::BYTES;
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF];
  static_assert(2 * BUF >= 8 * F * 1024, "sums through LDS");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int many = MANY_A ? g.m : g.n, few = MANY_A ? g.n : g.m;
  const int blocks = (many + ROWS - 1) / ROWS;
  const int slice = blockIdx.x / blocks, row0 = blockIdx.x % blocks * ROWS;
  const int all = (g.k + K - 1) / K;
  const int per = (all + g.slices - 1) / g.slices;
  const int from = min(slice * per, all), to = min(from + per, all);
  const int mine = wave % GROUPS * 16, share = wave / GROUPS;
  Many sm;
  Few sf;
  sm.start(MANY_A ? g.a : g.b, row0, many, threadIdx.x);
  sf.start(MANY_A ? g.b : g.a, 0, few, threadIdx.x);
  f32x4 acc[F] = {};
  struct Raw {
    float m[Many::PASSES][4], f[Few::PASSES][4];
  };
  // (blocks begin at different k, as in gemm_rows_kernel: 12 x 16384 to 16384 took
  // 225 us with all from their first on)
  const bool apart = !MX && ((MANY_A ? g.a : g.b).ld * 4) % 4096 == 0 && to > from;
  const int turn = apart ? (int)(blockIdx.x * 5) % (to - from) : 0;
  auto load = [&](int t, Raw& r) {
    if (t >= to) return;
    const int k = t + turn < to ? t + turn : t + turn - (to - from);
    sm.load(k, g.k - k * K, r.m);
    sf.load(k, g.k - k * K, r.f);
  };
  auto step = [&](int t, Raw& r) {
    if (t >= to) return;
    // (tile t - 2, whose place this takes, was read before the last barrier)
    char* buf = lds + ((t - from) & 1) * BUF;
    sm.store(buf, r.m);
    sf.store(buf + Many::BYTES, r.f);
    load(t + 3, r);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (loads stay in flight)
    block_barrier();
    float vm[8], vf[F][8];
    Many::fragment(buf, mine, share * 32, lane, vm);
#pragma unroll
    for (int f = 0; f < F; ++f)
      Few::fragment(buf + Many::BYTES, f * 16, share * 32, lane, vf[f]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int f = 0; f < F; ++f)
        // (a lane gets four neighbouring columns of the result)
        acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(
            MANY_A ? vf[f][i] : vm[i], MANY_A ? vm[i] : vf[f][i], acc[f], 0, 0, 0);
  };
  Raw r0, r1, r2;
  load(from, r0);
  load(from + 1, r1);
  load(from + 2, r2);
  for (int t = from; t < to; t += 3) {
    step(t, r0);
    step(t + 1, r1);
    step(t + 2, r2);
  }
  if constexpr (SHARES > 1) {
    __syncthreads();  // the tiles have been read
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int f = 0; f < F; ++f) sums[(wave * F + f) * 64 + lane] = acc[f];
    __syncthreads();
    if (share > 0) return;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int q = 1; q < SHARES; ++q)
        acc[f] += sums[((wave + q * GROUPS) * F + f) * 64 + lane];
  }
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int row = (MANY_A ? row0 + mine : f * 16) + (lane & 15);
    const int col = (MANY_A ? f * 16 : row0 + mine) + (lane >> 4) * 4;
    float v[4] = {acc[f][0], acc[f][1], acc[f][2], acc[f][3]}, bias[4] = {};
    if (g.slices > 1) {
      if (row < g.m && col < g.n)
        store_some<float, 4>(g.work + ((long)slice * g.m + row) * g.n + col, g.n - col, v);
      continue;
    }
    if (g.bias) load_learned<4>(g.bias, g.bias_dt, col, g.n - col, bias);
    finish<float, 4>(g, row, col, v, bias);
  }
}

// Sums of at most 16 Q floats: bound by writing the result.  A wave keeps 64 of B's
// rows in registers and goes down `rows_per` rows of A, sixteen at a time, the next
// ones in flight; it has no LDS and no barrier, so that waves write while others
// load.  A lane's elements of a sum are 4 Q (lane / 16) and on.  16384 x 9000 out of
// sums of 8, 590 MB: 126 us in a training step (4.7 TB/s), 190 one after the other
// (by tiles 245).
template <int Q, bool AX, bool BX>
__global__ __launch_bounds__(256) void gemm_short_kernel(GemmArgs g, int rows_per) {
  constexpr int N = 4 * Q;
  const int lane = threadIdx.x & 63;
  const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int strips = (g.n + 63) / 64;
  const int col0 = wave % strips * 64;
  const long first = (long)(wave / strips) * rows_per;
  if (first >= g.m) return;
  const int from = (int)first, to = min(g.m - from, rows_per) + from;
  const int k0 = (lane >> 4) * N;
  float b[4][N], bias[4][4] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    // (rows behind the last one repeat it: their results are not stored)
    const long row = min(col0 + w * 16 + (lane & 15), g.n - 1);
    if constexpr (BX) {
      const float* p = static_cast<const float*>(g.b.p) + (long)k0 * g.b.ld + row;
#pragma unroll
      for (int i = 0; i < N; ++i) b[w][i] = k0 + i < g.k ? p[i * g.b.ld] : 0.f;
    } else {
      const float* p = static_cast<const float*>(g.b.p) + row * g.b.ld + k0;
#pragma unroll
      for (int q = 0; q < Q; ++q)
        load_some<float, 4>(p + 4 * q, g.k - k0 - 4 * q, &b[w][4 * q]);
    }
    const int col = col0 + w * 16 + (lane >> 4) * 4;
    if (g.bias) load_learned<4>(g.bias, g.bias_dt, col, g.n - col, bias[w]);
  }
  auto load = [&](int row, float (&a)[N]) {
    const long mine = min(row + (lane & 15), g.m - 1);
    if constexpr (AX) {
      const float* p = static_cast<const float*>(g.a.p) + (long)k0 * g.a.ld + mine;
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = k0 + i < g.k ? p[i * g.a.ld] : 0.f;
    } else {
      const float* p = static_cast<const float*>(g.a.p) + mine * g.a.ld + k0;
#pragma unroll
      for (int q = 0; q < Q; ++q)
        load_some<float, 4>(p + 4 * q, g.k - k0 - 4 * q, &a[4 * q]);
    }
  };
  auto work = [&](int row, const float (&a)[N]) {
    f32x4 acc[4] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        acc[w] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[w][i], a[i], acc[w], 0, 0, 0);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float v[4] = {acc[w][0], acc[w][1], acc[w][2], acc[w][3]};
      finish<float, 4>(g, row + (lane & 15), col0 + w * 16 + (lane >> 4) * 4, v, bias[w]);
    }
  };
  float a0[N], a1[N];
  load(from, a0);
  for (int row = from; row < to; row += 32) {
    if (row + 16 < to) load(row + 16, a1);
    work(row, a0);
    if (row + 16 >= to) break;
    if (row + 32 < to) load(row + 32, a0);
    work(row + 16, a1);
  }
}

// The slices' sums, in order, and what follows the product.
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs g) {
  const int chunks = (g.n + 7) / 8;
  const long all = (long)g.m * chunks;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all;
       i += (long)gridDim.x * 256) {
    const int row = (int)(i / chunks), col = (int)(i % chunks) * 8;
    float v[8] = {}, bias[8] = {};
    for (int s = 0; s < g.slices; ++s) {
      float u[8];
      load_some<float, 8>(g.work + ((long)s * g.m + row) * g.n + col, g.n - col, u);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += u[q];
    }
    if (g.bias) load_learned<8>(g.bias, g.bias_dt, col, g.n - col, bias);
    finish<T, 8>(g, row, col, v, bias);
  }
}

}  // namespace

// Whether gemm_rows_kernel takes a product of operands along (its figures).
bool gemm_few_rows(long m, long n, long k, Dt dt) {
  const long bytes = n * k * dt_size(dt);
  if (m <= 64 && bytes <= (16L << 20)) return true;
  // (floats of up to 32 rows otherwise: few features, with less time)
  return dt != Dt::f32 && (m <= 16 || (m <= 32 && bytes <= (48L << 20)));
}

namespace {

// Up to how many rows or features of floats are few.  (Kernels of a pass forward and
// backward without bias, by 128-tiles and as few, us: 16384 x 5000 to 17 349 and 280,
// 16384 x 8 to 9000 653 and 426, 4000 x 10000 to 10 185 and 131, 4 x 12608 to 11709
// 617 and 397, 1152 x 1088 to 25 33 and 30.  From 33 on a step with bias took longer:
// 8192 x 48 to 4096 182 and 211, 16384 x 2048 to 64 168 and 182.)
constexpr int kFew = 32;

// How a product is cut up, and the time that it takes.  The tile kernels have
// one block a CU, so time goes by rounds of 256 blocks.  In units of a 128-tile's
// 64 k (0.48 us): a 256-tile's take 2.4, 32 k of floats 2.3 (also taken for a
// float A beside 16 bits, which has half the instructions), what a block does
// before and behind its loop 10 and 16, and the joining kernel 8 and 8 bytes for
// each partial sum at 4 TB/s.
struct Plan {
  int tile;      // 256 or 128; 32 or 16 for gemm_rows_kernel
  int slices;    // of k; 1 for 256
  long blocks;
  double block;  // a block's time
  double join;   // the joining kernel's
};

Plan plan_of(const GemmArgs& g, int tile, int slices) {
  const bool floats = g.dt == Dt::f32 || g.wide;
  const long tile_k = floats ? kFloatK : kTileK;
  const long tiles = (g.k + tile_k - 1) / tile_k;
  const long tm = (g.m + tile - 1) / tile, tn = (g.n + tile - 1) / tile;
  const double k = (double)((tiles + slices - 1) / slices);
  return {tile, slices, tm * tn * slices,
          tile == 256 ? 2.4 * k + 16 : (floats ? 2.3 : 1) * k + 10,
          slices > 1 ? 8 + slices * (double)g.m * g.n * 8 / 1.9e6 : 0};
}

// Calls f with the ways there are; at least four tiles of k a slice.
template <typename F>
void each_plan(const GemmArgs& g, bool powers, F f) {
  const bool floats = g.dt == Dt::f32 || g.wide;
  if (!floats) f(plan_of(g, 256, 1));
  const long tiles = g.k / (floats ? kFloatK : kTileK);
  for (int s = 1; s <= 32 && (s == 1 || tiles / s >= 4); s = powers ? 2 * s : s + 1)
    f(plan_of(g, 128, s));
}

double rounds(long blocks) { return (double)((blocks + 255) / 256); }

double time_of(const Plan& p) { return rounds(p.blocks) * p.block + p.join; }

// Blocks of two kinds, the longer ones first, on 256 CUs.
double time_of_two(Plan a, Plan b) {
  if (a.block < b.block) std::swap(a, b);
  const long over = a.blocks % 256;  // CUs that have one of the first kind more
  const double start = a.blocks / 256 * a.block;
  const double busy = over ? start + a.block : start;
  // what the other CUs do of the second kind meanwhile
  const long turns = over ? (long)(a.block / b.block) : 0;
  const long done = (256 - over) * turns;
  const double joins = a.join + b.join;
  if (over && b.blocks <= done) return busy + joins;
  const long left = b.blocks - done, last = left % 256;
  const double free = start + turns * b.block, whole = left / 256 * b.block;
  const double end = last == 0            ? whole
                     : last <= 256 - over ? free - busy + whole + b.block
                                          : whole + b.block;
  return busy + (end > whole ? end : whole) + joins;
}

void take(GemmArgs& g, const Plan& p) {
  g.tile = p.tile;
  g.slices = p.slices;
}

unsigned blocks_of(const GemmArgs& g) {
  const int tm = (g.m + g.tile - 1) / g.tile, tn = (g.n + g.tile - 1) / g.tile;
  switch (g.way) {
    case Way::brief:  // four waves a block
      return (unsigned)(((long)tm * ((g.n + 63) / 64) + 3) / 4);
    case Way::rows:
    case Way::narrow_a:
      return (unsigned)(tn * g.slices);
    case Way::narrow_b:
      return (unsigned)(tm * g.slices);
    default:
      return (unsigned)(tm * tn * g.slices);
  }
}

template <typename O>
void join_slices(const GemmArgs& g, hipStream_t st) {
  if (g.slices == 1) return;
  const long blocks = ((long)g.m * ((g.n + 7) / 8) + 255) / 256;
  gemm_join_kernel<O><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)),
                        dim3(256), 0, st>>>(g);
}

template <typename T, bool AX, bool BX>
void gemm_tiles_t(const GemmArgs& g, hipStream_t st) {
  const dim3 grid(blocks_of(g)), threads(kThreads<T, 128>);
  if (g.wide) {
    if constexpr (!__is_same(T, float) && BX)
      gemm_kernel<T, AX, BX, kWide>
          <<<grid, dim3(kThreads<T, kWide>), 0, st>>>(g);
  } else if (g.way == Way::tiles) {
    if (g.tile == 128) {
      gemm_kernel<T, AX, BX, 128><<<grid, threads, 0, st>>>(g);
    } else if constexpr (!__is_same(T, float)) {
      gemm_kernel<T, AX, BX, 256><<<grid, threads, 0, st>>>(g);
    }
  } else if (g.way == Way::brief) {
    if constexpr (__is_same(T, float)) {
      auto start = [&](auto q) {
        gemm_short_kernel<decltype(q)::value, AX, BX>
            <<<grid, dim3(256), 0, st>>>(g, g.tile);
      };
      using std::integral_constant;
      g.k <= 16 ? start(integral_constant<int, 1>()) : start(integral_constant<int, 2>());
    }
  } else if (g.way == Way::narrow_a || g.way == Way::narrow_b) {
    if constexpr (__is_same(T, float)) {
      using std::integral_constant;
      auto start = [&](auto f) {
        constexpr int F = decltype(f)::value;
        // (many lies across: 32 or 128 rows of it a block; along: 32)
        auto block = [&](auto rows, auto many_a) {
          constexpr bool MANY_A = decltype(many_a)::value;
          gemm_narrow_kernel<F, decltype(rows)::value, MANY_A ? AX : BX,
                             MANY_A ? BX : AX, MANY_A>
              <<<grid, dim3(512), 0, st>>>(g);
        };
        const integral_constant<int, 32> few_rows;
        const integral_constant<int, 128> rows;
        if (g.way == Way::narrow_b) {
          if constexpr (AX) {
            if (g.tile == 128) return block(rows, std::true_type{});
          }
          block(few_rows, std::true_type{});
        } else {
          if constexpr (BX) {
            if (g.tile == 128) return block(rows, std::false_type{});
          }
          block(few_rows, std::false_type{});
        }
      };
      const int few = g.way == Way::narrow_b ? g.n : g.m;
      few <= 16 ? start(integral_constant<int, 1>()) : start(integral_constant<int, 2>());
    }
  } else if constexpr (!AX && !BX) {
    auto start = [&](auto f, auto w) {
      gemm_rows_kernel<T, decltype(f)::value, decltype(w)::value>
          <<<grid, dim3(512), 0, st>>>(g);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    auto sixteen = [&] {
      g.m <= 16 ? start(one, one) : g.m <= 32 ? start(two, one) : start(four, one);
    };
    if constexpr (__is_same(T, float))
      sixteen();  // (plan_rows: more than 48 MB of floats go elsewhere)
    else
      g.tile == 32 ? start(one, two) : sixteen();
  }
  join_slices<T>(g, st);
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

template <typename T>
void gemm_two_tiles(const GemmArgs& dx, const GemmArgs& dw, hipStream_t st) {
  const bool dw_first = plan_of(dw, dw.tile, dw.slices).block >
                        plan_of(dx, dx.tile, dx.slices).block;
  const unsigned nx = blocks_of(dx), nw = blocks_of(dw);
  const dim3 grid(nx + nw), threads(kThreads<T, 128>);
  const int first = (int)(dw_first ? nw : nx);
  if constexpr (__is_same(T, float)) {
    gemm_two_kernel<T, 128, 128><<<grid, threads, 0, st>>>(dx, dw, first, dw_first);
  } else {
    if (dx.wide)
      gemm_two_kernel<T, kWide, kWide>
          <<<grid, dim3(kThreads<T, kWide>), 0, st>>>(dx, dw, first, dw_first);
    else if (dx.tile == 256 && dw.tile == 256)
      gemm_two_kernel<T, 256, 256><<<grid, threads, 0, st>>>(dx, dw, first, dw_first);
    else if (dx.tile == 256)
      gemm_two_kernel<T, 256, 128><<<grid, threads, 0, st>>>(dx, dw, first, dw_first);
    else if (dw.tile == 256)
      gemm_two_kernel<T, 128, 256><<<grid, threads, 0, st>>>(dx, dw, first, dw_first);
    else
      gemm_two_kernel<T, 128, 128><<<grid, threads, 0, st>>>(dx, dw, first, dw_first);
  }
  join_slices<T>(dx, st);
  join_slices<T>(dw, st);
}

// ---------------------------------------------------------------------------
// The activation's gradient and the sums of its columns
// ---------------------------------------------------------------------------

// A block has 64 vectors of columns and a slice of the rows, its four waves
// every fourth row of it.  The sums go over slices in a fixed order.  Bound by
// memory: 8192 x 16384 of bf16 (805 MB) take 175 us, 4.6 TB/s; with erff and
// expf of 32 bits they took 201.
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
          // (a NaN argument is not below zero: its gradient goes through, as it did)
          g[i] = a.act == Act::relu ? (z[i] <= 0.f ? 0.f : g[i])
                                    : g[i] * act_slope<T>(z[i], a.act);
      }
      if (a.dz && a.wide)
        store_some<float, VEC>(static_cast<float*>(a.dz) + (long)row * a.dz_ld + col,
                               left, g);
      else if (a.dz)
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
    for (int i = 0; i < VEC; ++i) {
      const float t = add[0][i * 64 + lane] + add[1][i * 64 + lane] +
                      add[2][i * 64 + lane] + add[3][i * 64 + lane];
      if (i >= left) continue;
      if (gridDim.y == 1)
        store_as(a.dbias, a.bias_dt, col + i, t);
      else
        a.partial[(long)blockIdx.y * a.n + col + i] = t;
    }
  }
}

// 32 columns a block, 32 strips of slices, each thread with four loads in
// flight.
__global__ __launch_bounds__(1024) void column_join_kernel(
    const float* __restrict__ partial, int slices, int n, void* out, Dt dt) {
  __shared__ float add[32][33];
  const int j = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const int col = (int)blockIdx.x * 32 + j;
  float t[4] = {};
  if (col < n) {
    const float* p = partial + col;
    int s = strip;
    for (; s + 96 < slices; s += 128)
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] += p[(long)(s + q * 32) * n];
    for (; s < slices; s += 32) t[0] += p[(long)s * n];
  }
  add[strip][j] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  // a half wave a column now
  float v = add[j][strip];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor(v, d, 32);
  const int to = (int)blockIdx.x * 32 + strip;
  if (j == 0 && to < n) store_as(out, dt, to, v);
}

}  // namespace

void gemm_fused(const GemmArgs& g, hipStream_t st) {
  if (g.m == 0 || g.n == 0) return;
  if (g.dt == Dt::f32)
    gemm_tiles<float>(g, st);
  else if (g.dt == Dt::bf16)
    gemm_tiles<bf16_t>(g, st);
  else
    gemm_tiles<f16_t>(g, st);
}

void gemm_two(const GemmArgs& dx, const GemmArgs& dw, hipStream_t st) {
  if (dx.dt == Dt::f32)
    gemm_two_tiles<float>(dx, dw, st);
  else if (dx.dt == Dt::bf16)
    gemm_two_tiles<bf16_t>(dx, dw, st);
  else
    gemm_two_tiles<f16_t>(dx, dw, st);
}

namespace {

void plan_tiles(GemmArgs& g) {
  double least = INFINITY;
  each_plan(g, false, [&](const Plan& p) {
    if (time_of(p) >= least) return;
    least = time_of(p);
    take(g, p);
  });
}

// A product for gemm_rows_kernel.
void plan_rows(GemmArgs& g) {
  // 16 rows of B a block, or 32 where A would be read too often (1 row with 134
  // MB and k 5000: 34 us, with 16 of B 43; with 34 MB 16 are faster)
  const long bytes = (long)g.n * g.k * dt_size(g.dt);
  g.way = Way::rows;
  g.tile = bytes > (48L << 20) ? 32 : 16;  // (at most 16 rows then)
  const long blocks = (g.n + g.tile - 1) / g.tile;
  const long lines = (long)g.k * dt_size(g.dt) / 128;
  long s = 512 / blocks;  // two blocks a CU, eight lines a wave at least
  if (s > lines / 64) s = lines / 64;
  g.slices = (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

// Floats with few rows or columns and with short sums; whether this is one.
bool plan_few(GemmArgs& g) {
  if (g.dt != Dt::f32) return false;
  // The gradients of a layer this small take one launch of tiles together (a whole
  // step of 3 x 16 to 19: 62 us, 67 with two launches, most of it the host's).
  if (g.b.across && g.m <= 128 && g.n <= 128 && g.k <= 128) return false;
  if (g.k <= kFew) {
    g.way = Way::brief;
    // rows of A that a wave goes down: eight waves a SIMD, if there are as many
    const long strips = (g.n + 63) / 64, groups = (g.m + 15L) / 16;
    long chunks = 8192 / strips;
    chunks = chunks < 1 ? 1 : chunks > groups ? groups : chunks;
    g.tile = (int)((groups + chunks - 1) / chunks) * 16;
    return true;
  }
  const bool a = g.m <= kFew, b = g.n <= kFew && (!a || g.n <= g.m);
  if (!a && !b) return false;
  const long many = b ? g.m : g.n;
  if (many > 1L << 27) return false;  // (a launch holds less than 2^32 threads)
  g.way = b ? Way::narrow_b : Way::narrow_a;
  // 32 rows of many a block; where it lies across those are 128 bytes of a row of
  // memory, so 128 if there are blocks enough (4000 x 10000 to 10: dW 35 us, with 32
  // 49; 2000 x 4096 to 32: 16 and 15, 512 x 2048 to 10 10 and 5)
  const bool across = b ? g.a.across : g.b.across;
  g.tile = across && many > 4608 ? 128 : 32;
  const long blocks = (many + g.tile - 1) / g.tile;
  const long tiles = ((long)g.k * g.tile + 4095) / 4096;
  // two blocks a CU, twelve tiles each at least: the joining kernel is another
  // launch and 4 us (512 x 2048 to 10 forward, 16 tiles: 11.3 us in one slice, 9.6 in
  // two; 3000 x 25 to 700 dW, 24 tiles: 33 in one, 17 in three)
  long s = 512 / blocks;
  if (s > tiles / 12) s = tiles / 12;
  g.slices = (int)(s < 1 ? 1 : s > 32 ? 32 : s);
  return true;
}

}  // namespace

void gemm_plan(GemmArgs& g) {
  g.way = Way::tiles;
  g.tile = 128;
  g.slices = 1;
  if (g.m < 1 || g.n < 1) return;  // nothing will be launched
  if (!g.a.across && !g.b.across && gemm_few_rows(g.m, g.n, g.k, g.dt))
    plan_rows(g);
  else if (!plan_few(g))
    plan_tiles(g);
}

bool gemm_plan_two(GemmArgs& a, GemmArgs& b) {
  gemm_plan(a);
  gemm_plan(b);
  if (a.way != Way::tiles || b.way != Way::tiles) return false;
  // (where both fill their rounds two launches are not slower: 2048^3 of bf16
  // took 45 us in two, 48 in one)
  double least = time_of(plan_of(a, a.tile, a.slices)) +
                 time_of(plan_of(b, b.tile, b.slices));
  bool together = false;
  each_plan(a, true, [&](const Plan& p) {
    each_plan(b, true, [&](const Plan& q) {
      const double time = time_of_two(p, q);
      // (a launch holds less than 2^32 threads)
      if (time >= least || p.blocks + q.blocks > 1L << 22) return;
      least = time;
      together = true;
      take(a, p);
      take(b, q);
    });
  });
  return together;
}

long gemm_work(const GemmArgs& g) {
  return g.slices > 1 ? (long)g.slices * g.m * g.n : 0;
}

// (dz rounded to 16 bits makes dx and dW 1.45 times as far from 64 bits as one
// rounding of theirs does, kept in floats 1.05.  The kernels of a backward pass
// in us, rounded and kept: 100 x 1000 by 1000 26 and 26, 128 x 1024 by 1024 20
// and 25, 1 x 4096 by 4096 37 and 49, while a pass is 75 of the host's time;
// beyond these sizes it costs more: 1 x 16384 by 4096 95 and 140, 1024 x 1024 by
// 1024 26 and 45, 2048^3 58 and 163.)
bool gemm_keeps_floats(long m, long n, long k, Dt dt, Act act) {
  return dt != Dt::f32 && (act == Act::gelu || act == Act::silu) &&
         m * n * k <= 1L << 28 && n * k <= 1L << 24;
}

bool gemm_takes(const Operand& o, long rows) {
  // (a tile's 256 rows are reached with 32-bit offsets)
  return (uintptr_t)o.p % 16 == 0 && o.ld % 8 == 0 && o.ld < kMostFeatures &&
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
  if (m <= 64) return 1;  // sixteen rows a wave: no second launch to join slices
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
  if (a.dbias && slices > 1)
    column_join_kernel<<<dim3((a.n + 31) / 32), dim3(1024), 0, st>>>(
        a.partial, slices, a.n, a.dbias, a.bias_dt);
}

}  // namespace cpd
