// Matrix-core products of 16-bit operands for gfx950, the part of
// linear_hip.hip that its time goes to.
//
//   C[m, n] = sum over k of A(m, k) B(n, k)
//
// An operand lies with k innermost ("along") or outermost ("across").  Tiles
// of 64 k go from memory straight into LDS (16 bytes a lane, no registers)
// and from there to v_mfma_f32_16x16x32 in the order that the instruction
// wants: along, a lane's eight k are adjacent and are one 16-byte read;
// across, ds_read_b64_tr_b16 transposes 4 k by 16 rows on the way.
//
// LDS holds a half tile of 128 rows (16 KB) as
//   along:   row r, 128 bytes;  its 16-byte chunk c at place c ^ (r/2 % 8)
//   across:  k, 256 bytes;      its 16-byte chunk c at place c ^ f(k),
//            f(k) = 2 (k % 4 + 4 (k/8 % 2))
// Both orders make the lanes that read together touch every bank once.  The
// copy into LDS is linear in the lane, so the order is made on the other
// side: each lane asks memory for the chunk that belongs at its place.
//
// The matrix instruction takes B's rows first, so that a lane holds four
// neighbouring n of one m.  Results go through LDS once more, 64 by 64 of a
// wave at a time, and leave as whole 128-byte lines.
#pragma once

#include "fused_ops.h"

namespace cpd {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using u32 = uint32_t;

constexpr int kTileK = 64;
constexpr int kHalf = 16384;  // bytes of a half tile: 128 rows by 64 k

typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ u32 lds_address(const void* p) {
  return (u32)(uintptr_t)(const lds_char*)p;
}

// 16 bytes a lane from base + off to LDS at `lds` + 16 * lane.  Counted by
// vmcnt; the compiler does not know of it, the callers wait.
__device__ __forceinline__ void copy_to_lds(const void* base, u32 off, u32 lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(off), "s"(base), "s"(lds)
      : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_copies() {  // all but the newest N, and LDS reads
  // lgkmcnt(0) alone, in the form that the compiler takes note of
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <typename T>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (__is_same(T, bf16_t))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ int swizzle_along(int r) { return r >> 1 & 7; }

__device__ __forceinline__ int swizzle_across(int k) {
  return 2 * ((k & 3) | ((k >> 3) & 1) << 2);
}

// What a lane copies of half tiles: WAVES waves, 16 / WAVES copies a half.
// The halves are rows 0-127 and 128-255, or, WOVEN, the even and the odd 32
// rows of 256.
template <bool ACROSS, int WAVES, bool WOVEN>
struct Copier {
  static constexpr int PASSES = 16 / WAVES;
  const char* base;   // of the first tile; uniform
  long step;          // bytes from a tile to the next
  u32 off[2][PASSES]; // of this lane's chunks, in half 0 and 1
  int at[PASSES];     // along: this lane's first k in a tile; across: its k
  u32 place;          // LDS offset of this wave's first copy in a half

  static __device__ __forceinline__ int row_of(int r, int h) {
    return WOVEN ? (r >> 5) * 64 + h * 32 + (r & 31) : h * 128 + r;
  }

  __device__ __forceinline__ void start(const Operand& o, int row0, int rows,
                                        int wave, int lane) {
    const char* p = static_cast<const char*>(o.p);
    place = wave * 1024;
    if constexpr (!ACROSS) {
      base = p + (long)row0 * o.ld * 2;
      step = kTileK * 2;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = (i * WAVES + wave) * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ swizzle_along(r);
        at[i] = chunk * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // rows behind the last one repeat it: their results are not stored
          const int row = min(row_of(r, h), rows - 1 - row0);
          off[h][i] = (u32)row * (u32)(o.ld * 2) + chunk * 16;
        }
      }
    } else {
      base = p;
      step = (long)kTileK * o.ld * 2;
      const int last = (rows + 7) / 8 * 8 - 8;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int k = (i * WAVES + wave) * 4 + (lane >> 4);
        const int chunk = (lane & 15) ^ swizzle_across(k);
        at[i] = k;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = min(row0 + row_of(chunk * 8, h), last);
          off[h][i] = (u32)k * (u32)(o.ld * 2) + (u32)c * 2;
        }
      }
    }
  }

  __device__ __forceinline__ void half(int tile, int h, u32 lds) const {
    const char* b = base + (long)tile * step;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
      copy_to_lds(b, off[h][i], lds + place + i * (WAVES * 1024));
  }

  // The last tile, of `left` < 64 k: through registers, zeros behind its end.
  __device__ __forceinline__ void rest(int tile, int h, char* lds, int left,
                                       int lane) const {
    const char* b = base + (long)tile * step;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      s16x8 v = {};
      const short* p = reinterpret_cast<const short*>(b + off[h][i]);
      if (ACROSS) {
        if (at[i] < left) v = *reinterpret_cast<const s16x8*>(p);
      } else if (at[i] + 8 <= left) {
        v = *reinterpret_cast<const s16x8*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at[i] + j < left) v[j] = p[j];
      }
      *reinterpret_cast<s16x8*>(lds + place + i * (WAVES * 1024) + lane * 16) = v;
    }
  }
};

// A lane's part of 16 rows by 32 k of a half tile: rows from `row`, the kk-th
// 32 k.
template <bool ACROSS>
__device__ __forceinline__ s16x8 fragment(const char* half, int row, int kk,
                                          int lane) {
  if constexpr (!ACROSS) {
    const int r = row + (lane & 15);
    const int place = (kk * 4 + (lane >> 4)) ^ swizzle_along(r);
    return *reinterpret_cast<const s16x8*>(half + r * 128 + place * 16);
  } else {
    const int s = lane & 15;
    const int k = kk * 32 + 8 * (lane >> 4) + (s >> 2);
    const int place = (row / 8 + ((s & 3) >> 1)) ^ swizzle_across(k);
    const char* p = half + k * 256 + place * 16 + (s & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds_vec;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec*)(p + 1024));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// ---------------------------------------------------------------------------
// Floats on the 16-bit matrix cores.
//
// A float is the sum of three bf16, exactly: each takes the next eight bits of
// its significand (cut off, not rounded, so that nothing overflows).  Of the
// nine products of two floats' parts the six largest are kept,
//   a1 b1 + (a1 b2 + a2 b1) + (a1 b3 + a2 b2 + a3 b1),
// the rest is below 2^-24 of a b.  A sixth of the 16-bit rate is 0.42 PFLOP/s
// against the float matrix instructions' 0.157; 0.21 are measured at 8192 x 2048
// by 8192, where the library's float product has 0.15.
//
// Where a 16-bit product gets one operand in floats (dz), both are cut into two
// parts, which is exact for the 16-bit one and leaves 16 bits of the other, and
// three products are kept.
//
// What is not finite becomes (+-1, 0, x): the last part meets first parts
// only, which are zero for zeros alone, so inf times 0 is NaN, inf times
// anything else inf, and no part of a finite number makes a NaN of it.
//
// bf16 ends at 2^-133: what a float has below that is cut off (of floats under
// 2^-109, 1.5e-33; at 1e-36 that is 1e-4 of the value), and a float that is all
// below it counts as 2^-133, so that its first part is not zero.  So each operand
// is off by 2^-133 at most.
//
// Tiles are of 32 k and three planes of 8 KB: along, row r of 64 bytes with
// its chunk c at place c ^ r/2 % 4; across, as above.
__device__ __forceinline__ int swizzle_float(int r) { return r >> 1 & 3; }

constexpr int kFloatK = 32;
constexpr int kPlane = 8192;

// One thread's share of 128 rows by 32 k: eight floats (or what T has for them),
// cut into P parts.
template <typename T, int P, bool ACROSS>
struct FloatStager {
  const T* p;      // of this thread's eight, in the first tile
  long step;       // elements from a tile to the next
  int at;          // along: its first k; across: its k
  int rows_left;   // across: rows from its first on
  u32 place;       // where its 16 bytes of a plane belong

  __device__ __forceinline__ void start(const Operand& o, int row0, int rows,
                                        int tid) {  // of 512
    const T* base = static_cast<const T*>(o.p);
    if constexpr (!ACROSS) {
      const int r = tid >> 2, chunk = tid & 3;
      at = chunk * 8;
      rows_left = 8;
      p = base + (long)min(row0 + r, rows - 1) * o.ld + at;
      step = kFloatK;
      place = r * 64 + ((chunk ^ swizzle_float(r)) << 4);
    } else {
      const int chunk = tid & 15;
      at = tid >> 4;
      rows_left = rows - (row0 + chunk * 8);
      p = base + (long)at * o.ld + row0 + chunk * 8;
      step = kFloatK * o.ld;
      place = at * 256 + ((chunk ^ swizzle_across(at)) << 4);
    }
  }

  // `left`: k from this tile's first on
  __device__ __forceinline__ void load(int tile, int left, float (&v)[8]) const {
    const T* q = p + tile * step;
    const int n = ACROSS ? (at < left ? rows_left : 0) : left - at;
    load_some<T, 8>(q, n, v);
  }

  __device__ __forceinline__ void store(char* lds, const float (&v)[8]) const {
    u32 part[P][4];
    // NaN, infinities and what is below the normal range: one instruction each
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) odd |= __builtin_amdgcn_classf(v[i], 0x297);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32 first[2], second[2], third[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = v[2 * i + j];
        first[j] = __float_as_uint(x) & 0xFFFF0000u;
        const float r = x - __uint_as_float(first[j]);
        second[j] = __float_as_uint(r) & 0xFFFF0000u;
        third[j] = __float_as_uint(r - __uint_as_float(second[j]));
      }
      // the upper halves of two, side by side
      part[0][i] = __builtin_amdgcn_perm(first[1], first[0], 0x07060302u);
      part[1][i] = __builtin_amdgcn_perm(second[1], second[0], 0x07060302u);
      if (P > 2)
        part[P - 1][i] = __builtin_amdgcn_perm(third[1], third[0], 0x07060302u);
    }
    if (odd) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const u32 u = __float_as_uint(v[i]);
        const u32 sh = (i & 1) * 16, keep = i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        if ((u << 1) >= 0xFF000000u) {
          // (a NaN whose bits are all in the lower half must stay one)
          const u32 top = (u >> 16) | (u << 9 ? 0x40u : 0u);
          part[0][i / 2] = (part[0][i / 2] & keep) |
                           ((0x3F80u | (u >> 16 & 0x8000u)) << sh);
          if (P > 2) part[1][i / 2] = part[1][i / 2] & keep;
          part[P - 1][i / 2] = (part[P - 1][i / 2] & keep) | (top << sh);
        } else if ((u << 1) - 1 < 0x1FFFFu) {
          part[0][i / 2] |= 1u << sh;  // 2^-133; its parts are zeros, with its sign
        }
      }
    }
#pragma unroll
    for (int q = 0; q < P; ++q) {
      typedef u32 V __attribute__((ext_vector_type(4)));
      *reinterpret_cast<V*>(lds + q * kPlane + place) =
          V{part[q][0], part[q][1], part[q][2], part[q][3]};
    }
  }
};

template <bool ACROSS>
__device__ __forceinline__ s16x8 float_fragment(const char* plane, int row,
                                                int lane) {
  if constexpr (!ACROSS) {
    const int r = row + (lane & 15);
    const int place = (lane >> 4) ^ swizzle_float(r);
    return *reinterpret_cast<const s16x8*>(plane + r * 64 + place * 16);
  } else {
    return fragment<true>(plane, row, 0, lane);
  }
}

// A wave's results, 16 F rows by 64, v[i][j] for rows 16 i + lane % 16 and
// columns 16 j + 4 (lane / 16), through 4 F KB of LDS of its own (a row's
// 16-byte chunks in the order chunk ^ row % 16, which keeps both sides off
// each other's banks).  `put(row, col, v)` then gets eight neighbouring
// results; eight lanes have a row's 64.
template <int F, typename P>
__device__ __forceinline__ void leave(char* lds, const f32x4 (*v)[4], int lane,
                                      P put) {
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = i * 16 + (lane & 15), chunk = j * 4 + (lane >> 4);
      *reinterpret_cast<f32x4*>(lds + row * 256 + ((chunk ^ (row & 15)) << 4)) =
          v[i][j];
    }
#pragma unroll 1
  for (int pass = 0; pass < 2 * F; ++pass) {
    const int row = pass * 8 + (lane >> 3), chunk = (lane & 7) * 2;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(
        lds + row * 256 + ((chunk ^ (row & 15)) << 4));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(
        lds + row * 256 + (((chunk + 1) ^ (row & 15)) << 4));
    float out[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    put(row, (lane & 7) * 8, out);
  }
}

}  // namespace
}  // namespace cpd
