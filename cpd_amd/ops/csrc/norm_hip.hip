// Layer norm over the last axis for gfx950, with the residual sum in front.
//
//   s    = round(x + residual)            (only with a residual)
//   mean = sum(s) / C,  var = sum((s - mean)^2) / C,  r = 1/sqrt(var + eps)
//   y    = (s - mean) * r * weight + bias
//
// and backward, with h = (s - mean) * r and g = dy * weight:
//
//   dx      = r * (g - sum(g)/C - h * sum(g h)/C) + ds      (= dresidual)
//   dweight = sum over rows of dy * h,   dbias = sum over rows of dy
//
// Everything is bound by memory: each pass reads its inputs once and writes
// its outputs once.  A row stays in the registers of the threads that share
// it (16 threads, a wave, a block of 256 to 1024), so the variance is
// taken around the mean without a second read.  All sums are 32-bit floats.
//
// With bf16 rows of 4096 and the residual, 8192 of them take 60 us forward and
// 61 + 4 backward (268 MB each: 4.5 and 4.1 TB/s, where a copy of 1 GiB runs at
// 4.95); 20011 float rows of 257 take 12 and 18 + 4 (3.3 and 2.8 TB/s).
#include "fused_ops.h"

namespace cpd {
namespace {

// Threads that share a row, and 16-byte chunks each of them holds.  Longer rows
// go to the looping kernels below.  (us for 2^25 values:)
//  - Forward up to four chunks: bf16 rows of 8192 took 34, with two 47, floats of
//    4096 43 and 58; 512 threads where 256 are too few: floats of 5120 56, with
//    1024 threads 81, bf16 of 12288 42 and 49.
//  - Backward four of floats (1024: 81, with two 106), but two in 16 bits, whose
//    sums of columns take twice the registers (512: 46, with four 84; 8192: 50 and
//    107).
struct Shape {
  int tpr, ch;
};

Shape shape_for(int cols, Dt dt, int most, bool half) {
  const int vec = 16 / dt_size(dt);
  const int n = (cols + vec - 1) / vec;
  for (int t : {16, 64, 256, 512, 1024})
    if (n <= t * most && (t != 512 || half)) return {t, n <= t ? 1 : n <= 2 * t ? 2 : 4};
  return {0, 0};
}
Shape forward_shape(int cols, Dt dt) { return shape_for(cols, dt, 4, true); }
Shape backward_shape(int cols, Dt dt) {
  return shape_for(cols, dt, dt == Dt::f32 ? 4 : 2, false);
}

template <typename T, int TPR, int CH>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void norm_fwd_kernel(
    NormArgs a) {
  constexpr int VEC = Vec16<T>::N;
  constexpr int ROWS = TPR <= 64 ? 256 / TPR : 1;  // rows of a block
  __shared__ float smem[4 * (TPR <= 64 ? 1 : TPR / 64)];
  const int lane = threadIdx.x % TPR;
  for (long row0 = (long)blockIdx.x * ROWS; row0 < a.rows;
       row0 += (long)gridDim.x * ROWS) {
    const long row = row0 + threadIdx.x / TPR;
    if (row >= a.rows) break;  // a whole row's threads leave together
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    float v[CH][VEC];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
      load_vec<T>(x + at, a.cols - at, 0.f, v[c]);
    }
    if (a.res) {
      const T* r = static_cast<const T*>(a.res) + row * a.res_ld;
      T* s = static_cast<T*>(a.s) + row * a.cols;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int at = (c * TPR + lane) * VEC;
        float u[VEC];
        load_vec<T>(r + at, a.cols - at, 0.f, u);
        // the norm is of the sum as it is stored, which backward reads again
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] = (float)(T)(v[c][i] + u[i]);
        store_vec<T>(s + at, a.cols - at, v[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += v[c][i];
    const float mean = row_sum<TPR>(sum, smem, 0) / (float)a.cols;
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = v[c][i] - mean;
        sq += at + i < a.cols ? d * d : 0.f;
      }
    }
    const float var = row_sum<TPR>(sq, smem, 1) / (float)a.cols;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (a.stats && lane == 0) {
      a.stats[row * 2] = mean;
      a.stats[row * 2 + 1] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
      if (at >= a.cols) break;
      float w[VEC], b[VEC], o[VEC];
      if (a.weight) load_learned<VEC>(a.weight, a.wdt, at, a.cols - at, w);
      if (a.bias) load_learned<VEC>(a.bias, a.wdt, at, a.cols - at, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        o[i] = (v[c][i] - mean) * rstd;
        if (a.weight) o[i] *= w[i];
        if (a.bias) o[i] += b[i];
      }
      store_vec<T>(y + at, a.cols - at, o);
    }
  }
}

// Rows of any length: one block a row, the row read three times (the second
// and third time mostly from L2).
template <typename T>
__global__ __launch_bounds__(1024) void norm_fwd_loop_kernel(NormArgs a) {
  constexpr int VEC = Vec16<T>::N;
  __shared__ float smem[4 * 16];
  // (the launcher starts one block for every row)
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* src = x;
  float sum = 0.f;
  if (a.res) {
    const T* r = static_cast<const T*>(a.res) + row * a.res_ld;
    T* s = static_cast<T*>(a.s) + row * a.cols;
    src = s;  // a thread reads back only what it wrote itself
    for (long at = threadIdx.x * VEC; at < a.cols; at += 1024 * VEC) {
      const int left = (int)(a.cols - at);
      float v[VEC], u[VEC];
      load_vec<T>(x + at, left, 0.f, v);
      load_vec<T>(r + at, left, 0.f, u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[i] = (float)(T)(v[i] + u[i]);
        sum += v[i];
      }
      store_vec<T>(s + at, left, v);
    }
  } else {
    for (long at = threadIdx.x * VEC; at < a.cols; at += 1024 * VEC) {
      float v[VEC];
      load_vec<T>(x + at, (int)(a.cols - at), 0.f, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += v[i];
    }
  }
  const float mean = row_sum<1024>(sum, smem, 0) / (float)a.cols;
  float sq = 0.f;
  for (long at = threadIdx.x * VEC; at < a.cols; at += 1024 * VEC) {
    float v[VEC];
    load_vec<T>(src + at, (int)(a.cols - at), mean, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sq += (v[i] - mean) * (v[i] - mean);
  }
  const float var = row_sum<1024>(sq, smem, 1) / (float)a.cols;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  if (a.stats && threadIdx.x == 0) {
    a.stats[row * 2] = mean;
    a.stats[row * 2 + 1] = rstd;
  }
  T* y = static_cast<T*>(a.y) + row * a.cols;
  for (long at = threadIdx.x * VEC; at < a.cols; at += 1024 * VEC) {
    const int left = (int)(a.cols - at);
    float v[VEC], w[VEC], b[VEC];
    load_vec<T>(src + at, left, 0.f, v);
    if (a.weight) load_learned<VEC>(a.weight, a.wdt, at, left, w);
    if (a.bias) load_learned<VEC>(a.bias, a.wdt, at, left, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[i] = (v[i] - mean) * rstd;
      if (a.weight) v[i] *= w[i];
      if (a.bias) v[i] += b[i];
    }
    store_vec<T>(y + at, left, v);
  }
}

// Backward: each block walks rows gridDim.x apart and keeps its share of
// dweight and dbias in registers (a thread has the same columns in every
// row), so the data is read once for all three gradients; the next row is
// ordered before this one is worked on, since the two sums over the row leave
// memory idle otherwise (not in blocks of 1024, which have registers for one:
// 16384 bf16 took 221 us for 2^25 values with two, 83 with one).  The blocks'
// shares go to `partial` and are added in a fixed order: no atomics.
template <typename T, int TPR, int CH, bool DS>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void norm_bwd_kernel(
    NormGradArgs a) {
  constexpr int VEC = Vec16<T>::N;
  constexpr int ROWS = TPR <= 64 ? 256 / TPR : 1;
  __shared__ float smem[4 * (TPR <= 64 ? 1 : TPR / 64)];
  const int lane = threadIdx.x % TPR;
  const long stride = (long)gridDim.x * ROWS;
  struct Row {
    typename Vec16<T>::type s[CH], dy[CH], ds[DS ? CH : 1];
    float mean, rstd;
  };
  auto fetch = [&](long row, Row& r) {
    if (row >= a.rows) return;
    r.mean = a.stats[row * 2];
    r.rstd = a.stats[row * 2 + 1];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC, left = a.cols - at;
      r.s[c] = load_raw<T>(static_cast<const T*>(a.s) + row * a.s_ld + at, left);
      r.dy[c] = load_raw<T>(static_cast<const T*>(a.dy) + row * a.dy_ld + at, left);
      if constexpr (DS)
        r.ds[c] = load_raw<T>(static_cast<const T*>(a.ds) + row * a.ds_ld + at, left);
    }
  };
  float dw[CH][VEC] = {}, db[CH][VEC] = {};
  int turn = 0;
  auto work = [&](long row, const Row& r) {
    // (ROWS > 1: a row's threads are within a wave, and leave together)
    if (row >= a.rows) return;
    float h[CH][VEC], g[CH][VEC];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
      float w[VEC];
      if (a.weight) load_learned<VEC>(a.weight, a.wdt, at, a.cols - at, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[c][i] = ((float)r.s[c][i] - r.mean) * r.rstd;
        g[c][i] = (float)r.dy[c][i];
        dw[c][i] += g[c][i] * h[c][i];
        db[c][i] += g[c][i];
        if (a.weight) g[c][i] *= w[i];
        sg += g[c][i];
        sgh += g[c][i] * h[c][i];
      }
    }
    row_sums<TPR>(sg, sgh, smem, turn);
    turn ^= 1;
    sg /= (float)a.cols;
    sgh /= (float)a.cols;
    T* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
      if (at >= a.cols) break;
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        o[i] = r.rstd * (g[c][i] - sg - h[c][i] * sgh) +
               (DS ? (float)r.ds[DS ? c : 0][i] : 0.f);
      store_vec<T>(dx + at, a.cols - at, o);
    }
  };
  const long first = (long)blockIdx.x * ROWS;
  const int mine = threadIdx.x / TPR;
  if constexpr (TPR == 1024) {
    for (long row = first; row < a.rows; row += stride) {
      Row r;
      fetch(row + mine, r);
      work(row + mine, r);
    }
  } else {
    Row r0, r1;
    fetch(first + mine, r0);
    for (long row = first; row < a.rows; row += 2 * stride) {
      fetch(row + stride + mine, r1);
      work(row + mine, r0);
      if (row + stride >= a.rows) break;
      fetch(row + 2 * stride + mine, r0);
      work(row + stride + mine, r1);
    }
  }
  if (!a.partial) return;
  float* part = a.partial + (long)blockIdx.x * 2 * a.cols;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = (c * TPR + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (at + i < a.cols) {
          part[at + i] = dw[c][i];
          part[a.cols + at + i] = db[c][i];
        }
    }
  } else {
    // the block's rows share columns: add them up through LDS, in order
    __shared__ float add[ROWS][TPR * VEC + 1];
#pragma unroll
    for (int c = 0; c < 2 * CH; ++c) {
      const int base = (c >> 1) * TPR * VEC;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        add[mine][lane * VEC + i] = (c & 1) ? db[c >> 1][i] : dw[c >> 1][i];
      __syncthreads();
      for (int j = threadIdx.x; j < TPR * VEC; j += 256) {
        float t = 0.f;
        for (int r = 0; r < ROWS; ++r) t += add[r][j];
        if (base + j < a.cols) part[(c & 1) * a.cols + base + j] = t;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_loop_kernel(NormGradArgs a) {
  constexpr int VEC = Vec16<T>::N;
  __shared__ float smem[4 * 16];
  const long row = blockIdx.x;
  const T* s = static_cast<const T*>(a.s) + row * a.s_ld;
  const T* dy = static_cast<const T*>(a.dy) + row * a.dy_ld;
  const float mean = a.stats[row * 2], rstd = a.stats[row * 2 + 1];
  float sg = 0.f, sgh = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (long at = threadIdx.x * VEC; at < a.cols; at += 1024 * VEC) {
      const int left = (int)(a.cols - at);
      float h[VEC], g[VEC], w[VEC];
      load_vec<T>(s + at, left, mean, h);
      load_vec<T>(dy + at, left, 0.f, g);
      if (a.weight) load_learned<VEC>(a.weight, a.wdt, at, left, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[i] = (h[i] - mean) * rstd;
        if (a.weight) g[i] *= w[i];
      }
      if (pass == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          sg += g[i];
          sgh += g[i] * h[i];
        }
      } else {
        float o[VEC] = {};
        if (a.ds)
          load_vec<T>(static_cast<const T*>(a.ds) + row * a.ds_ld + at, left,
                      0.f, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] += rstd * (g[i] - sg - h[i] * sgh);
        store_vec<T>(static_cast<T*>(a.dx) + row * a.cols + at, left, o);
      }
    }
    if (pass == 0) {
      sg = row_sum<1024>(sg, smem, 0) / (float)a.cols;
      sgh = row_sum<1024>(sgh, smem, 1) / (float)a.cols;
    }
  }
}

// dweight and dbias of the looping kernels' rows: a thread a column, blocks
// of rows side by side.
template <typename T>
__global__ __launch_bounds__(256) void norm_bwd_cols_kernel(NormGradArgs a) {
  const long col = (long)blockIdx.x * 256 + threadIdx.x;
  if (col >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = (float)static_cast<const T*>(a.dy)[row * a.dy_ld + col];
    const float s = (float)static_cast<const T*>(a.s)[row * a.s_ld + col];
    dw += g * ((s - a.stats[row * 2]) * a.stats[row * 2 + 1]);
    db += g;
  }
  float* part = a.partial + (long)blockIdx.y * 2 * a.cols;
  part[col] = dw;
  part[a.cols + col] = db;
}

// Adds the blocks' shares: 32 columns a block, 32 strips of rows, each thread
// with four loads in flight.
__global__ __launch_bounds__(1024) void norm_bwd_join_kernel(
    const float* __restrict__ partial, int blocks, int cols, void* dweight,
    void* dbias, Dt wdt) {
  __shared__ float add[32][33];
  const int j = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const long all = 2L * cols;
  const long col = (long)blockIdx.x * 32 + j;  // over [2, cols] flattened
  float t[4] = {};
  if (col < all) {
    const float* p = partial + col;
    int b = strip;
    for (; b + 96 < blocks; b += 128)
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] += p[(b + q * 32) * all];
    for (; b < blocks; b += 32) t[0] += p[b * all];
  }
  add[strip][j] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  // a half wave a column now
  const int mine = threadIdx.x >> 5;
  float v = add[threadIdx.x & 31][mine];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor(v, d, 32);
  const long to = (long)blockIdx.x * 32 + mine;
  if ((threadIdx.x & 31) == 0 && to < all) {
    void* out = to < cols ? dweight : dbias;
    if (out) store_as(out, wdt, to < cols ? to : to - cols, v);
  }
}

template <typename T>
void forward_t(const NormArgs& a, hipStream_t st) {
  const Shape s = forward_shape(a.cols, a.dt);
  if (s.tpr == 0) {
    norm_fwd_loop_kernel<T><<<dim3(a.rows), dim3(1024), 0, st>>>(a);
    return;
  }
  const int rows = s.tpr <= 64 ? 256 / s.tpr : 1;
  // one group of rows a block, up to the most a launch may hold
  const long groups = (a.rows + rows - 1) / rows;
  const dim3 grid((unsigned)(groups < (1 << 20) ? groups : 1 << 20));
  const dim3 block(s.tpr <= 64 ? 256 : s.tpr);
#define CPD_NORM(TPR, CH)                                     \
  if (s.tpr == TPR && s.ch == CH) {                           \
    norm_fwd_kernel<T, TPR, CH><<<grid, block, 0, st>>>(a);   \
    return;                                                   \
  }
  CPD_NORM(16, 1) CPD_NORM(16, 2) CPD_NORM(16, 4)
  CPD_NORM(64, 2) CPD_NORM(64, 4)
  CPD_NORM(256, 2) CPD_NORM(256, 4)
  CPD_NORM(512, 4) CPD_NORM(1024, 4)
#undef CPD_NORM
}

template <typename T, bool DS>
void backward_t(const NormGradArgs& a, hipStream_t st) {
  const Shape s = backward_shape(a.cols, a.dt);
  const int blocks = norm_grad_blocks(a.rows, a.cols, a.dt);
  if (s.tpr == 0) {
    norm_bwd_loop_kernel<T><<<dim3(a.rows), dim3(1024), 0, st>>>(a);
    if (a.partial)
      norm_bwd_cols_kernel<T><<<dim3((a.cols + 255) / 256, blocks), dim3(256),
                                0, st>>>(a);
    return;
  }
  const dim3 grid(blocks), block(s.tpr <= 64 ? 256 : s.tpr);
#define CPD_NORM(TPR, CH)                                     \
  if (s.tpr == TPR && s.ch == CH) {                           \
    norm_bwd_kernel<T, TPR, CH, DS><<<grid, block, 0, st>>>(a); \
    return;                                                   \
  }
  if constexpr (sizeof(T) == 4) {
    CPD_NORM(16, 1) CPD_NORM(16, 2) CPD_NORM(16, 4)
    CPD_NORM(64, 2) CPD_NORM(64, 4)
    CPD_NORM(256, 2) CPD_NORM(256, 4)
    CPD_NORM(1024, 2) CPD_NORM(1024, 4)
  } else {
    CPD_NORM(16, 1) CPD_NORM(16, 2)
    CPD_NORM(64, 1) CPD_NORM(64, 2)
    CPD_NORM(256, 1) CPD_NORM(256, 2)
    CPD_NORM(1024, 1) CPD_NORM(1024, 2)
  }
#undef CPD_NORM
}

}  // namespace

void norm_forward(const NormArgs& a, hipStream_t st) {
  if (a.rows == 0) return;
  if (a.dt == Dt::f32)
    forward_t<float>(a, st);
  else if (a.dt == Dt::bf16)
    forward_t<bf16_t>(a, st);
  else
    forward_t<f16_t>(a, st);
}

int norm_grad_blocks(long rows, int cols, Dt dt) {
  const Shape s = backward_shape(cols, dt);
  if (s.tpr == 0) return (int)(rows < 64 ? rows : 64);
  const long per = s.tpr <= 64 ? 256 / s.tpr : 1;
  const long groups = (rows + per - 1) / per;
  // (us for 2^25 values of bf16, rows of 256, 2048 and 16384: 42, 50 and 66; with
  // half the blocks 54, 74 and 73; with twice as many 60, 55 and 94)
  const long most = s.tpr == 1024 ? 256 : 512;
  return (int)(groups < most ? groups : most);
}

void norm_backward(const NormGradArgs& a, hipStream_t st) {
  if (a.rows == 0) return;
  auto start = [&](auto zero) {
    if (a.ds)
      backward_t<decltype(zero), true>(a, st);
    else
      backward_t<decltype(zero), false>(a, st);
  };
  if (a.dt == Dt::f32)
    start(0.f);
  else if (a.dt == Dt::bf16)
    start((bf16_t)0.f);
  else
    start((f16_t)0.f);
  if (a.partial)
    norm_bwd_join_kernel<<<dim3((2L * a.cols + 31) / 32), dim3(1024), 0, st>>>(
        a.partial, norm_grad_blocks(a.rows, a.cols, a.dt), a.cols, a.dweight,
        a.dbias, a.wdt);
}

}  // namespace cpd
