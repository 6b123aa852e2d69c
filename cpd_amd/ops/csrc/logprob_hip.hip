// Log probabilities of given tokens, the entropy of each row of logits and
// its top alternatives, in one read of the logits (gfx950).
//
//   m = max x,  S = sum e^(x-m),  A = sum e^(x-m) (x-m)
//   logprob = (x_t - m) - log S
//   entropy = log S - A / S
//   top k   = the k largest, (value down, index up)
//
// and backward, with p = e^((x-m) - log S):
//
//   dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
//
// Both passes are bound by memory.  Forward keeps m, S and A running in
// 32-bit floats around the largest value seen so far; S and A are rescaled
// when that grows, so any logits' range is safe.
//
// The alternatives ride along: each wave holds the best 64 of what it has
// read as a sorted list, one entry a lane, and compares a whole vector of
// new values with the k-th entry before it does anything else.  For values in
// no order that test fails about k log(n / k) times in n values; values that
// keep rising pass one and all, which is slower but as right.
//
// Without alternatives 4096 rows of 50021 bf16 take 95 us (4.3 TB/s) forward and
// 149 backward (5.5 TB/s).  Alternatives add the work of inserting them: 2048
// rows of 131072 fp16 take 104 us, 123 with one, 154 with five, 195 with
// sixteen, 305 with 64.
//
// A row of -inf alone has log probability -inf, entropy 0 and no gradient.
// NaN or +inf in a row makes its log probabilities NaN; among the
// alternatives NaN counts as the largest.
#include "fused_ops.h"

namespace cpd {
namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp(float x) {  // e^x, e^-inf = 0
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// A distance from the maximum, kept finite: below this e^d is zero, and zero
// times an overflowed distance would be NaN.
__device__ __forceinline__ float near(float d) { return fmaxf(d, -1e4f); }

struct Soft {  // running maximum and sums
  float m, s, a;
};

// The sums of `o` and `v`, around the larger maximum.
__device__ __forceinline__ Soft join(Soft v, Soft o) {
  const float m = fmaxf(v.m, o.m);
  if (m == -INFINITY) return {m, v.s + o.s, 0.f};  // (NaN in a sum stays)
  const float dv = v.m == -INFINITY ? 0.f : near(v.m - m);
  const float dq = o.m == -INFINITY ? 0.f : near(o.m - m);
  const float fv = v.m == -INFINITY ? 0.f : fast_exp(dv);
  const float fo = o.m == -INFINITY ? 0.f : fast_exp(dq);
  return {m, v.s * fv + o.s * fo, fv * (v.a + dv * v.s) + fo * (o.a + dq * o.s)};
}

__device__ __forceinline__ Soft wave_join(Soft v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1)
    v = join(v, {__shfl_xor(v.m, d, 64), __shfl_xor(v.s, d, 64),
                 __shfl_xor(v.a, d, 64)});
  return v;
}

// Order of the alternatives as one number: larger value first, then smaller
// index; 0 is below every entry.
__device__ __forceinline__ u64 key_of(float x, int index) {
  u32 u = __float_as_uint(x);
  u = x != x     ? 0xFFFFFFFFu
      : x == 0.f ? 0x80000000u  // both zeros are one value
                 : (u >> 31 ? ~u : u | 0x80000000u);
  return ((u64)u << 32) | (u32)(0x7FFFFFFF - index);
}
__device__ __forceinline__ float key_value(u64 key) {
  const u32 u = (u32)(key >> 32);
  if (u == 0xFFFFFFFFu) return NAN;
  return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_index(u64 key) {
  return 0x7FFFFFFF - (int)(u32)key;
}

__device__ __forceinline__ u64 lane_key(u64 v, int lane) {
  const u32 lo = __builtin_amdgcn_readlane((u32)v, lane);
  const u32 hi = __builtin_amdgcn_readlane((u32)(v >> 32), lane);
  return ((u64)hi << 32) | lo;
}

__device__ __forceinline__ u64 key_across(u64 v, int d) {
  const u32 lo = __shfl_xor((u32)v, d, 64), hi = __shfl_xor((u32)(v >> 32), d, 64);
  return ((u64)hi << 32) | lo;
}

// The larger of two lanes' keys, or the smaller, to each its own.
__device__ __forceinline__ u64 exchange(u64 key, int d, bool larger) {
  const u64 other = key_across(key, d);
  return (other > key) == larger ? other : key;
}

// The wave's list: lane i holds the i-th entry.
struct Top {
  u64 mine, least;  // this lane's entry; the k-th entry
  int lane, k;

  __device__ __forceinline__ void start(int k_) {
    mine = least = 0;
    lane = threadIdx.x & 63;
    k = k_;
  }
  // what a value has to pass, NaN until there are k entries
  __device__ __forceinline__ float bar() const {
    return least ? key_value(least) : NAN;
  }
  // Joins a list in order, the largest first, one key a lane.
  __device__ __forceinline__ void join_list(u64 key) {
    // the larger of the i-th and the other's i-th from its end: the 64 best,
    // rising and falling once, which six exchanges put in order
    const u64 back = key_across(key, 63);
    mine = back > mine ? back : mine;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mine = exchange(mine, d, !(lane & d));
    least = lane_key(mine, k - 1);
  }
  __device__ __forceinline__ void insert(u64 key) {
    const int at = __popcll(__ballot(mine > key));
    // the entry of the lane below (wave_shr:1)
    const u32 lo = __builtin_amdgcn_update_dpp(0, (int)(u32)mine, 0x138, 0xf,
                                               0xf, false);
    const u32 hi = __builtin_amdgcn_update_dpp(0, (int)(u32)(mine >> 32),
                                               0x138, 0xf, 0xf, false);
    const u64 below = ((u64)hi << 32) | lo;
    mine = lane < at ? mine : lane == at ? key : below;
    least = lane_key(mine, k - 1);
  }
  // Every lane's key, the best ones kept: a few are inserted one by one, many
  // are put in order together (21 exchanges) and joined.  (For a list of one or
  // two few of the many would be inserted.)
  __device__ __forceinline__ void offer(u64 key) {
    u64 mask = __ballot(key > least);
    if (__popcll(mask) > 24 && k > 2) {
      key = key > least ? key : 0;
#pragma unroll 1
      for (int size = 2; size <= 64; size *= 2)
#pragma unroll 1
        for (int d = size / 2; d > 0; d >>= 1)
          key = exchange(key, d, !(lane & d) == !(lane & size));
      join_list(key);
      return;
    }
    while (mask) {
      const int from = __ffsll(mask) - 1;
      insert(lane_key(key, from));
      if (lane == from) key = 0;
      mask = __ballot(key > least);
    }
  }
};

// What one part of a row gives, for the joining kernel.
struct Part {
  float m, s, a, pad;
};

// How many blocks a row is cut into, and what each of them takes: with few
// rows a row is spread until about 512 blocks are running (two a CU); a part
// is at least one 16-byte load a thread.
struct Cut {
  int waves, parts, per;
};

Cut cut_for(long rows, int vocab, Dt dt) {
  const int vec = 16 / dt_size(dt);
  if (vocab <= 64 * vec * 4) return {1, 1, vocab};  // a wave a row
  const int step = 256 * vec;
  const int steps = (vocab + step - 1) / step;
  long want = rows >= 512 || rows < 1 ? 1 : (512 + rows - 1) / rows;
  if (want > 64) want = 64;
  if (want > steps) want = steps;
  const int per = (int)((steps + want - 1) / want) * step;
  return {4, (vocab + per - 1) / per, per};
}

template <int WAVES, bool TOP>
__device__ __forceinline__ void finish(const LogprobArgs& a, long row,
                                       int64_t target, Soft v, const Top& top) {
  const bool none = v.s == 0.f;
  const float logs = none ? -INFINITY : logf(v.s);
  if (top.lane == 0) {
    float lp;
    if (target < 0 || target >= a.vocab) {
      lp = NAN;  // neither a token nor the index to pass over
    } else {
      float x;
      const long at = row * a.ld + target;
      if (a.dt == Dt::f32)
        x = static_cast<const float*>(a.x)[at];
      else if (a.dt == Dt::bf16)
        x = (float)static_cast<const bf16_t*>(a.x)[at];
      else
        x = (float)static_cast<const f16_t*>(a.x)[at];
      lp = none ? -INFINITY : (x - v.m) - logs;
    }
    a.logprobs[row] = lp;
    a.entropy[row] = none ? 0.f : logs - v.a / v.s;
    a.stats[row * 2] = v.m;
    a.stats[row * 2 + 1] = logs;
  }
  if (TOP && top.lane < a.top) {
    a.top_ids[row * a.top + top.lane] = key_index(top.mine);
    a.top_logprobs[row * a.top + top.lane] =
        none ? -INFINITY : (key_value(top.mine) - v.m) - logs;
  }
}

// Joins the waves of a block: wave 0 leaves with everything.
template <int WAVES, bool TOP>
__device__ __forceinline__ void block_join(Soft& v, Top& top, Soft* softs,
                                           u64 (*lists)[kMostTop]) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // what the last row left there has been read
  if (top.lane == 0) softs[wave] = v;
  if (TOP) lists[wave][top.lane] = top.mine;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      v = join(v, softs[w]);
      if (TOP) top.join_list(lists[w][top.lane]);
    }
  }
}

struct Found {
  float value[64][4];  // 16 bytes of T
  int at[64], done[64];
};

// Offers a wave's vectors, one a lane, the first of them from index `from` on.
// (Rare, so it is kept small: it works through LDS and in loops, and hides its
// lane number from the compiler, which otherwise works out everything that
// depends on it ahead of the row and holds it in 80 registers.)
template <typename T>
__device__ __forceinline__ void search(Top& top,
                                       const typename Vec16<T>::type* seen,
                                       Found& found, bool odd, int from, int to) {
  constexpr int VEC = Vec16<T>::N;
  asm volatile("" : "+v"(top.lane));
  const typename Vec16<T>::type u = seen[top.lane];
  const int at = from + top.lane * VEC;
  // the largest value, where it is first, and the next one
  float most = -INFINITY, second = -INFINITY;
  int done = -1;
#pragma unroll
  for (int i = VEC - 1; i >= 0; --i) {
    const float y = (float)u[i];
    if (y >= most) {
      second = done >= 0 ? most : second;
      most = y;
      done = i;
    } else {
      second = fmaxf(second, y);
    }
  }
  bool mine = odd || !(most <= top.bar());
  u64 mask = __ballot(mine);
  if (!mask) return;
  if (__popcll(mask) > 8 && !__ballot(odd)) {
    // Many pass, as at a row's start: their largest values first, after which
    // most of the others do not.  (One that equals the bar may come before
    // what set it here.)
    top.offer(mine && at + done < to ? key_of(most, at + done) : 0);
    mine = mine && !(second < top.bar());
    mask = __ballot(mine);
    if (!mask) return;
  } else {
    done = -1;
  }
  // the vectors that are left side by side, and from there one value a lane
  const int rank = __popcll(mask & ((1ull << top.lane) - 1));
  if (mine) {
    *reinterpret_cast<typename Vec16<T>::type*>(found.value[rank]) = u;
    found.at[rank] = at;
    found.done[rank] = done;
  }
  __builtin_amdgcn_wave_barrier();
  const int many = __popcll(mask) * VEC;
  for (int i = top.lane; i - top.lane < many; i += 64) {
    const int slot = i / VEC & 63, index = found.at[slot] + i % VEC;
    const bool in = i < many && index < to && found.done[slot] != i % VEC;
    const float value = (float)reinterpret_cast<const T*>(found.value)[i & (64 * VEC - 1)];
    top.offer(in ? key_of(value, index) : 0);
  }
  __builtin_amdgcn_wave_barrier();
}

template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(256) void logprob_kernel(LogprobArgs a, int parts,
                                                      int per, Part* part,
                                                      u64* keys) {
  constexpr int VEC = Vec16<T>::N;
  constexpr int TPR = WAVES * 64;
  // (with alternatives 16-bit rows have registers for two: with four and 138
  // registers 16384 rows of 8192 with five of them took 225 us instead of 196)
  constexpr int LOADS = TOP && sizeof(T) == 2 ? 2 : 4;
  __shared__ Soft softs[WAVES];
  __shared__ u64 lists[TOP && WAVES > 1 ? WAVES : 1][kMostTop];
  __shared__ typename Vec16<T>::type seen[TOP ? 4 : 1][LOADS][64];
  __shared__ Found found[TOP ? 4 : 1];
  // (in a scalar register: what a row or a wave shares stays out of the others)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x % TPR;
  const long jobs = a.rows * parts;
  Top top;
  for (long job0 = (long)blockIdx.x * (256 / TPR); job0 < jobs;
       job0 += (long)gridDim.x * (256 / TPR)) {
    const long job = job0 + (WAVES == 1 ? wave : 0);
    if (job >= jobs) break;  // WAVES == 1 only: a whole wave leaves
    const long row = job / parts;
    const int64_t target = a.targets[row];
    top.start(TOP ? a.top : 1);
    if (target == a.ignore) {
      if (job == row * parts && tid < 64) {
        if (tid == 0) {
          a.logprobs[row] = 0.f;
          a.entropy[row] = 0.f;
          a.stats[row * 2] = 0.f;
          a.stats[row * 2 + 1] = 0.f;
        }
        if (TOP && tid < a.top) {
          a.top_ids[row * a.top + tid] = -1;
          a.top_logprobs[row * a.top + tid] = -INFINITY;
        }
      }
      continue;
    }
    const int from = (int)(job - row * parts) * per;
    const int to = a.vocab - from < per ? a.vocab : from + per;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    Soft v = {-INFINITY, 0.f, 0.f};
    // a few loads a thread at a time, one rescaling for all of them
    for (int base = from; base < to; base += TPR * VEC * LOADS) {
      typename Vec16<T>::type u[LOADS];
      if (base + TPR * VEC * LOADS <= to) {
#pragma unroll
        for (int c = 0; c < LOADS; ++c)
          u[c] = load_raw<T>(x + base + (c * TPR + tid) * VEC, VEC);
      } else {
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
          const int at = base + (c * TPR + tid) * VEC;
          u[c] = load_raw<T>(x + at, to - at, (T)-INFINITY);
        }
      }
      float big = (float)u[0][0];
#pragma unroll
      for (int c = 0; c < LOADS; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) big = fmaxf(big, (float)u[c][i]);
      if (big > v.m) {
        const float d = v.m == -INFINITY ? 0.f : near(v.m - big);
        const float f = v.m == -INFINITY ? 0.f : fast_exp(d);
        v.a = f * (v.a + d * v.s);
        v.s *= f;
        v.m = big;
      }
      const float about = v.m == -INFINITY ? 0.f : v.m;
#pragma unroll
      for (int c = 0; c < LOADS; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = (float)u[c][i] - about;
          const float e = fast_exp(d);
          v.s += e;
          v.a += e * near(d);
        }
      if (TOP) {
        // a NaN is passed over by the maximum, but it makes the sum one
        const bool odd = v.s != v.s;
        // Values equal to the bar come after what set it and do not pass.
        if (__ballot(odd || !(big <= top.bar()))) {
#pragma unroll
          for (int c = 0; c < LOADS; ++c) seen[wave][c][top.lane] = u[c];
#pragma unroll 1
          for (int c = 0; c < LOADS; ++c)
            search<T>(top, seen[wave][c], found[wave], odd,
                      base + (c * TPR + tid - top.lane) * VEC, to);
        }
      }
    }
    v = wave_join(v);
    if (WAVES > 1) block_join<WAVES, TOP>(v, top, softs, lists);
    if (tid < 64) {
      if (parts == 1) {
        finish<WAVES, TOP>(a, row, target, v, top);
      } else {
        if (tid == 0) part[job] = {v.m, v.s, v.a, 0.f};
        if (TOP && tid < a.top) keys[job * a.top + tid] = top.mine;
      }
    }
  }
}

// Joins a row's parts: one block a row, its waves take parts in turn.
template <bool TOP>
__global__ __launch_bounds__(256) void logprob_join_kernel(
    LogprobArgs a, int parts, const Part* part, const u64* keys) {
  __shared__ Soft softs[4];
  __shared__ u64 lists[4][kMostTop];
  const long row = blockIdx.x;
  const int64_t target = a.targets[row];
  if (target == a.ignore) return;  // written by the kernel before
  Top top;
  top.start(TOP ? a.top : 1);
  const int wave = threadIdx.x >> 6;
  Soft v = {-INFINITY, 0.f, 0.f};
  const int mine = wave + 4 * top.lane;  // this lane's part: at most 64 parts
  if (mine < parts) {
    const Part p = part[row * parts + mine];
    v = {p.m, p.s, p.a};
  }
  v = wave_join(v);
  if (TOP) {
    u64 key[16];  // all of them in flight
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int p = wave + 4 * i;
      key[i] = p < parts && top.lane < a.top
                   ? keys[(row * parts + p) * a.top + top.lane]
                   : 0;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (wave + 4 * i < parts) top.join_list(key[i]);
  }
  block_join<4, TOP>(v, top, softs, lists);
  if (wave == 0) finish<4, TOP>(a, row, target, v, top);
}

// WAVES = 1: a wave has a whole row; 4: a block has one of its `chunks`.  32768
// rows of 1000 take 38 us in 16 bits and 41 in 32 with a wave a row, 96 and 54
// with a block; longer rows than a wave takes at once have a block's bandwidth.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogprobGradArgs a,
                                                          int chunks) {
  constexpr int VEC = Vec16<T>::N;
  constexpr int TPR = WAVES * 64;
  constexpr int UNROLL = 4;
  const int tid = threadIdx.x % TPR;
  const long jobs = a.rows * chunks;
  // (in a scalar register, as everything that a row shares then is)
  const int mine =
      WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  for (long job = (long)blockIdx.x * (256 / TPR) + mine; job < jobs;
       job += (long)gridDim.x * (256 / TPR)) {
    const long row = WAVES == 1 ? job : job / chunks;
    const int base = (int)(job - row * chunks) * (TPR * VEC * UNROLL);
    const int64_t target = a.targets[row];
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    T* dx = static_cast<T*>(a.dx) + row * a.vocab;
    const float m = a.stats[row * 2], logs = a.stats[row * 2 + 1];
    const bool skip = target == a.ignore || logs == -INFINITY;
    float glp = a.glogprobs ? a.glogprobs[row] : 0.f;
    const float gent = a.gentropy ? a.gentropy[row] : 0.f;
    if (target < 0 || target >= a.vocab) glp = NAN;
    const float c0 = -(glp + gent * (a.gentropy ? a.entropy[row] : 0.f));
    // (all of a job's loads in flight at once: none under a condition but at a
    // row's end, and none across them)
    const bool whole = base + TPR * VEC * UNROLL <= a.vocab;
    typename Vec16<T>::type u[UNROLL] = {};
    if (!skip) {
      if (whole) {
#pragma unroll
        for (int c = 0; c < UNROLL; ++c)
          u[c] = load_raw<T>(x + base + (c * TPR + tid) * VEC, VEC);
      } else {
#pragma unroll
        for (int c = 0; c < UNROLL; ++c) {
          const int at = base + (c * TPR + tid) * VEC;
          u[c] = load_raw<T>(x + at, a.vocab - at);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < UNROLL; ++c) {
      const int at = base + (c * TPR + tid) * VEC;
      float d[VEC] = {};
      if (!skip) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float logp = ((float)u[c][i] - m) - logs;
          const float p = fast_exp(logp);
          d[i] = p == 0.f ? 0.f : p * (c0 - gent * logp);
          if (at + i == target) d[i] += glp;
        }
      }
      if (at < a.vocab) store_vec<T>(dx + at, whole ? VEC : a.vocab - at, d);
    }
  }
}

template <typename T>
void forward_t(const LogprobArgs& a, hipStream_t st) {
  const Cut c = cut_for(a.rows, a.vocab, a.dt);
  const long jobs = a.rows * c.parts;
  const long blocks = c.waves == 1 ? (jobs + 3) / 4 : jobs;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  Part* part = static_cast<Part*>(a.work);
  u64* keys = reinterpret_cast<u64*>(part + jobs);
  if (c.waves == 1) {
    if (a.top)
      logprob_kernel<T, 1, true><<<grid, dim3(256), 0, st>>>(a, 1, c.per, part, keys);
    else
      logprob_kernel<T, 1, false><<<grid, dim3(256), 0, st>>>(a, 1, c.per, part, keys);
    return;
  }
  if (a.top)
    logprob_kernel<T, 4, true><<<grid, dim3(256), 0, st>>>(a, c.parts, c.per, part, keys);
  else
    logprob_kernel<T, 4, false><<<grid, dim3(256), 0, st>>>(a, c.parts, c.per, part, keys);
  if (c.parts > 1) {  // fewer than 512 rows
    if (a.top)
      logprob_join_kernel<true><<<dim3(a.rows), dim3(256), 0, st>>>(a, c.parts, part, keys);
    else
      logprob_join_kernel<false><<<dim3(a.rows), dim3(256), 0, st>>>(a, c.parts, part, keys);
  }
}

template <typename T>
void backward_t(const LogprobGradArgs& a, hipStream_t st) {
  const int per = 256 * Vec16<T>::N * 4;
  const int chunks = (int)(((long)a.vocab + per - 1) / per);
  const bool wave = a.vocab <= per / 4;
  const long blocks = wave ? (a.rows + 3) / 4 : a.rows * chunks;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  if (wave)
    logprob_bwd_kernel<T, 1><<<grid, dim3(256), 0, st>>>(a, 1);
  else
    logprob_bwd_kernel<T, 4><<<grid, dim3(256), 0, st>>>(a, chunks);
}

}  // namespace

long logprob_work_bytes(long rows, int vocab, int top, Dt dt) {
  const Cut c = cut_for(rows, vocab, dt);
  if (c.parts == 1) return 0;
  return rows * c.parts * ((long)sizeof(Part) + 8L * top);
}

void logprob_forward(const LogprobArgs& a, hipStream_t st) {
  if (a.rows == 0) return;
  if (a.dt == Dt::f32)
    forward_t<float>(a, st);
  else if (a.dt == Dt::bf16)
    forward_t<bf16_t>(a, st);
  else
    forward_t<f16_t>(a, st);
}

void logprob_backward(const LogprobGradArgs& a, hipStream_t st) {
  if (a.rows == 0) return;
  if (a.dt == Dt::f32)
    backward_t<float>(a, st);
  else if (a.dt == Dt::bf16)
    backward_t<bf16_t>(a, st);
  else
    backward_t<f16_t>(a, st);
}

}  // namespace cpd
