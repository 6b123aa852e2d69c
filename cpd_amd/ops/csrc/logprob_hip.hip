// Log probabilities of given tokens, the entropy of each row of logits and
// its top alternatives, in one read of the logits (gfx950).
//
//   m = max x,  S = sum e^(x-m),  A = sum e^(x-m) (x-m)
//   logprob = (x_t - m) - log S
//   entropy = log S - A / S
//   top k   = the k largest, (value down, index up)
//
// and backward, with p = e^(x-m) / S:
//
//   dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
//
// Both passes are bound by memory.  Forward keeps m, S and A running in
// 32-bit floats around the largest value seen so far; S and A are rescaled
// when that grows, so any logits' range is safe.
//
// The alternatives ride along.  Each wave holds the best 64 of what it has read
// as a sorted list, one entry a lane, and a bar below which nothing need be
// kept: the k-th entry, and at a row's start the k-th largest of the lanes'
// maxima.  What passes is put aside in LDS, and a few of those at a time are
// sorted and joined.  For values in no order the bar is passed about
// k log(n / k) times in n values; values that keep rising pass often, which is
// slower but as right.
//
// Calls one after the other, three inputs in turn: without alternatives 4096 rows of
// 50021 bf16 take 93 us (4.4 TB/s) forward and 152 backward (5.4 TB/s); in a training
// step, behind each other's writes, 110 to 120 and 139 to 165.  Alternatives add
// work: 2048 rows of 131072 fp16 take 98 us, 121 with one, 144 with five, 171 with
// sixteen, 228 with 64 (inserted one by one 123, 154, 195 and 305).
//
// A row of -inf alone has log probability -inf, entropy 0 and no gradient.
// NaN or +inf in a row makes its log probabilities NaN; among the
// alternatives NaN counts as the largest.
#include <type_traits>

#include "fused_ops.h"

namespace cpd {
namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);

__device__ __forceinline__ float fast_exp(float x) {  // e^x, e^-inf = 0
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// The same for a probability beside logits of T.  Rounding x log2(e) puts e^x off
// by up to |x| half steps.  That is nothing to what is rounded to 16 bits; for
// floats what the product lost is put back (in the forward pass it evens out in
// the sums: 32768 rows of 1000 floats took 34 us with it, 31 without).
template <typename T>
__device__ __forceinline__ float entry_exp(float x) {
  if constexpr (sizeof(T) < 4) return fast_exp(x);
  const float t = x * kLog2e, e = __builtin_amdgcn_exp2f(t);
  const float low = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t));
  // (of -inf that is NaN, and the middle of the three a number)
  return fmaf(e, __builtin_amdgcn_fmed3f(low, -1.f, 1.f) * 0.69314718f, e);
}

// A distance from the maximum, kept finite: below this e^d is zero, and zero
// times an overflowed distance would be NaN.
__device__ __forceinline__ float near(float d) { return fmaxf(d, -1e4f); }

// (By its bits: of bf16 values taken as floats the compiler makes a maximum of
// bf16, which the machine does not have.)
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(f16_t x) { return (float)x; }
__device__ __forceinline__ float as_float(bf16_t x) {
  return __uint_as_float((u32)__builtin_bit_cast(unsigned short, x) << 16);
}

struct Soft {  // running maximum and sums
  float m, s, a;
};

// Two by two, so that no term is rounded more than log2 N times.
template <int N>
__device__ __forceinline__ float sum_of(const float* v) {
  if constexpr (N == 1) return v[0];
  else return sum_of<N / 2>(v) + sum_of<N / 2>(v + N / 2);
}

// Adds x to a sum that is the larger of the two; what that loses goes to `low`.
__device__ __forceinline__ void add_to(float& sum, float& low, float x) {
  const float t = sum + x;
  low += (sum - t) + x;
  sum = t;
}

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

// The same over a wave: the maximum first, so that each lane rescales once
// (32768 rows of 1000 floats: 32 us; pair by pair through LDS 4 more).
__device__ __forceinline__ Soft wave_join(Soft v) {
  const float m = group_max(v.m);
  const bool none = v.m == -INFINITY;
  const float d = none ? 0.f : near(v.m - m);
  const float f = none ? (m == -INFINITY ? 1.f : 0.f) : fast_exp(d);
  return {m, group_sum<64>(v.s * f), group_sum<64>(f * (v.a + d * v.s))};
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

// v of lane ^ D, within the instruction (a shuffle through LDS takes ten times
// as long).
template <int D>
__device__ __forceinline__ u32 across(u32 v) {
  auto dpp = [](u32 x, auto ctrl) {
    return (u32)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf,
                                            0xf, true);
  };
  using std::integral_constant;
  if constexpr (D == 1) return dpp(v, integral_constant<int, 0xB1>());
  if constexpr (D == 2) return dpp(v, integral_constant<int, 0x4E>());
  if constexpr (D == 4)  // 7, and 3 of it back
    return dpp(dpp(v, integral_constant<int, 0x141>()), integral_constant<int, 0x1B>());
  if constexpr (D == 8) return dpp(v, integral_constant<int, 0x128>());
  if constexpr (D == 15) return dpp(v, integral_constant<int, 0x140>());
  if constexpr (D == 16) {
    const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? both[0] : both[1];
  }
  if constexpr (D == 32) {
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? both[0] : both[1];
  }
  if constexpr (D == 63) return across<32>(across<16>(across<15>(v)));
}

template <int D>
__device__ __forceinline__ u64 key_across(u64 v) {
  return ((u64)across<D>((u32)(v >> 32)) << 32) | across<D>((u32)v);
}

// The larger of two lanes' keys, or the smaller, to each its own.
template <int D>
__device__ __forceinline__ u64 exchange(u64 key, bool larger) {
  const u64 other = key_across<D>(key);
  return (other > key) == larger ? other : key;
}

// Keys that rise and fall once (in groups of 2 D lanes) into order.
template <int D>
__device__ __forceinline__ u64 merge(u64 key, int lane, bool falling) {
  key = exchange<D>(key, !(lane & D) == falling);
  if constexpr (D > 1) key = merge<D / 2>(key, lane, falling);
  return key;
}

// A wave's keys in order, the largest first; those behind the n-th are 0.
template <int SIZE = 2>
__device__ __forceinline__ u64 sort(u64 key, int lane, int n) {
  key = merge<SIZE / 2>(key, lane, !(lane & SIZE));
  if constexpr (SIZE < 64)
    if (n > SIZE) key = sort<SIZE * 2>(key, lane, n);
  return key;
}

// The wave's list: lane i holds the i-th entry.
struct Top {
  u64 mine;
  int lane;

  __device__ __forceinline__ void start() {
    mine = 0;
    lane = threadIdx.x & 63;
  }
  // Joins a list in order, the largest first, one key a lane.
  __device__ __forceinline__ void join_list(u64 key) {
    // the larger of the i-th and the other's i-th from its end: the 64 best,
    // rising and falling once
    const u64 back = key_across<63>(key);
    mine = merge<32>(back > mine ? back : mine, lane, true);
  }
};

// The smallest float above x (infinity for infinity).
__device__ __forceinline__ float above(float x) {
  const u32 u = __float_as_uint(x);
  return x == INFINITY ? x
         : x == 0.f    ? __uint_as_float(1)
                       : __uint_as_float(u >> 31 ? u - 1 : u + 1);
}

__device__ __forceinline__ float uniform(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// Floats that rise and fall once into order, and any 64 into falling order.
template <int D>
__device__ __forceinline__ float merge_floats(float x, int lane, bool falling) {
  const float y = __uint_as_float(across<D>(__float_as_uint(x)));
  x = !(lane & D) == falling ? fmaxf(x, y) : fminf(x, y);
  if constexpr (D > 1) x = merge_floats<D / 2>(x, lane, falling);
  return x;
}
template <int SIZE = 2>
__device__ __forceinline__ float sort_floats(float x, int lane) {
  x = merge_floats<SIZE / 2>(x, lane, !(lane & SIZE));
  if constexpr (SIZE < 64) x = sort_floats<SIZE * 2>(x, lane);
  return x;
}

// What a wave has found for its list and not put there yet.  Less than 64 wait
// from one vector to the next, each of which may add all of its elements.
template <int VEC>
struct Pending {
  u64 key[64 + 64 * VEC];
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
    a.stats[row * 2 + 1] = v.s;
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

// Joins the `count` pending keys, 64 at a time.
template <int VEC>
__device__ __forceinline__ void settle(Top& top, Pending<VEC>& pending, int& count) {
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  while (count > 0) {
    const int n = count < 64 ? count : 64;
    count -= n;
    const u64 key = top.lane < n ? pending.key[count + top.lane] : 0;
    top.join_list(sort(key, top.lane, n));
  }
  __builtin_amdgcn_wave_barrier();
}

template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(256) void logprob_kernel(LogprobArgs a, int parts,
                                                      int per, Part* part,
                                                      u64* keys) {
  constexpr int VEC = Vec16<T>::N;
  constexpr int TPR = WAVES * 64;
  // vectors a lane that are worked on together (with alternatives 16-bit rows have
  // registers for two: with four 16384 rows of 8192 with five of them took 182 us
  // instead of 161)
  constexpr int LOADS = TOP && sizeof(T) == 2 ? 2 : 4;
  constexpr int STEP = TPR * VEC * LOADS;
  typedef typename Vec16<T>::type V;
  __shared__ Soft softs[WAVES];
  __shared__ u64 lists[TOP && WAVES > 1 ? WAVES : 1][kMostTop];
  __shared__ Pending<VEC> pendings[TOP ? 4 : 1];
  // (in a scalar register: what a row or a wave shares stays out of the others)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x % TPR;
  const long jobs = a.rows * parts;
  // (Pending keys do not raise the bar, and joining a few costs half of joining
  // 64: with one alternative 131072 fp16 took 125 us if four were waited for, 123
  // if two, 158 if 64; with sixteen 174, 169 and 171.)
  const int most = min(64, 2 * a.top);
  Top top;
  for (long job0 = (long)blockIdx.x * (256 / TPR); job0 < jobs;
       job0 += (long)gridDim.x * (256 / TPR)) {
    const long job = job0 + (WAVES == 1 ? wave : 0);
    if (job >= jobs) break;  // WAVES == 1 only: a whole wave leaves
    const long row = job / parts;
    const int64_t target = a.targets[row];
    top.start();
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
    // What the sums' roundings lost: a lane adds hundreds of small terms to the 1
    // that a row's maximum is (131072 floats, one of them at 0 and the rest at -12:
    // S was 1e-5 off without).
    float low_s = 0.f, low_a = 0.f;
    // Values below `bar` need not be kept.  (k of them are from it on, and those
    // of this wave's that equal it and come later come after them.)
    float bar = -INFINITY;
    int count = 0;  // of pending keys
    bool full = false;  // k of them are NaN: nothing comes before those
    // one rescaling for a few vectors
    auto work = [&](int base, const V (&u)[LOADS]) {
      float big = as_float(u[0][0]);
#pragma unroll
      for (int c = 0; c < LOADS; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) big = fmaxf(big, as_float(u[c][i]));
      if (big > v.m) {
        const float d = v.m == -INFINITY ? 0.f : near(v.m - big);
        const float f = v.m == -INFINITY ? 0.f : fast_exp(d);
        v.a = f * (v.a + d * v.s);
        v.s *= f;
        low_a = f * (low_a + d * low_s);
        low_s *= f;
        v.m = big;
      }
      const float about = v.m == -INFINITY ? 0.f : v.m;
      float some_s[LOADS], some_a[LOADS];
#pragma unroll
      for (int c = 0; c < LOADS; ++c) {
        some_s[c] = some_a[c] = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = as_float(u[c][i]) - about;
          const float e = fast_exp(d);
          some_s[c] += e;
          some_a[c] += e * near(d);
        }
      }
      add_to(v.s, low_s, sum_of<LOADS>(some_s));
      add_to(v.a, low_a, sum_of<LOADS>(some_a));
      if (!TOP) return;
      // a NaN is passed over by the maximum, but it makes the sum one
      const bool odd = v.s != v.s;
      const u64 some = __ballot(odd || !(big < bar));
      if (!some || full) return;
      // (What follows is rare.  The lane number and the values are hidden from the
      // compiler, which otherwise holds all that depends on them in registers
      // through the whole loop.)
      int lane = top.lane;
      asm volatile("" : "+v"(lane));
      Pending<VEC>& pending = pendings[wave];
      float now = bar;
      if (__popcll(some) > 16) {
        // Many pass, as at a row's start: the k-th of the lanes' maxima is a
        // better bar, and the next values have to be above it.
        const float kth = lane_value(sort_floats(fmaxf(big, -INFINITY), lane),
                                     a.top - 1);
        now = uniform(fmaxf(now, kth));
        bar = uniform(fmaxf(bar, above(kth)));
      }
#pragma unroll 1
      for (int c = 0; c < LOADS; ++c) {
        typedef u32 Raw __attribute__((ext_vector_type(4)));
        Raw raw = __builtin_bit_cast(Raw, u[0]);
#pragma unroll
        for (int j = 1; j < LOADS; ++j)
          if (c == j) raw = __builtin_bit_cast(Raw, u[j]);
        int at = base + (c * TPR + tid - top.lane + lane) * VEC;
        asm volatile("" : "+v"(raw), "+v"(at));
        const V w = __builtin_bit_cast(V, raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float y = as_float(w[i]);
          const bool in = !(y < now) && at + i < to;
          const u64 mask = __ballot(in);
          if (!mask) continue;
          if (in)
            pending.key[count + __builtin_amdgcn_mbcnt_hi(
                                    (u32)(mask >> 32),
                                    __builtin_amdgcn_mbcnt_lo((u32)mask, 0))] =
                key_of(y, at + i);
          count += __popcll(mask);
        }
        if (count < most) continue;
        settle(top, pending, count);
        const u64 least = lane_key(top.mine, a.top - 1);
        if (!least) continue;
        const float kth = key_value(least);
        full = kth != kth;
        now = uniform(fmaxf(now, kth));
        bar = uniform(fmaxf(bar, above(kth)));
      }
    };
    for (int base = from; base < to; base += STEP) {
      V u[LOADS];
      if (base + STEP <= to) {
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
      work(base, u);
    }
    if (TOP) settle(top, pendings[wave], count);
    v.s += low_s;
    v.a += low_a;
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
  top.start();
  const int wave = threadIdx.x >> 6;
  Soft v = {-INFINITY, 0.f, 0.f};
  const int mine = wave + 4 * top.lane;  // this lane's part: at most 64 parts
  if (mine < parts) {
    const Part p = part[row * parts + mine];
    v = {p.m, p.s, p.a};
  }
  v = wave_join(v);
  if (TOP && a.top < 16) {
    // Short lists 64 keys at a time: sorting and joining those is 28 exchanges,
    // joining a list is seven (one row of 128000 bf16 with eight: 4.6 us,
    // 7.4 list by list).
    const int many = parts * a.top;
    const u64* p = keys + row * many;
    u64 key[4];  // all of them in flight
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (wave + 4 * i) * 64 + top.lane;
      key[i] = at < many ? p[at] : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = many - (wave + 4 * i) * 64;
      if (left > 0) top.join_list(sort(key[i], top.lane, left));
    }
  } else if (TOP) {
    u64 key[16];
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
    const float m = a.stats[row * 2], sum = a.stats[row * 2 + 1];
    const bool skip = target == a.ignore || sum == 0.f;
    // (e^((x-m) - log S) would have the logarithm's rounding in it, and the
    // difference's: three to four times as far off with 131072 floats)
    const float logs = logf(sum), one = 1.f / sum;
    float glp = a.glogprobs ? a.glogprobs[row] : 0.f;
    const float gent = a.gentropy ? a.gentropy[row] : 0.f;
    // (the entropy does not ask for the target)
    if ((target < 0 || target >= a.vocab) && a.glogprobs) glp = NAN;
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
          const float x = (float)u[c][i] - m;
          const float p = entry_exp<T>(x) * one;
          d[i] = p == 0.f ? 0.f : p * (c0 - gent * (x - logs));
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
