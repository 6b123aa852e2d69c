// Launchers of the layer-norm, linear and log-probability kernels.  Plain
// pointers and sizes: the checks on tensors are in hip_bindings.cpp.  Each
// enqueues on `stream` and returns; none allocates.
#pragma once

#include "fused_common.h"

namespace cpd {

struct NormArgs {
  const void* x;          // [rows, cols], row stride x_ld
  const void* res;        // or null
  const void* weight;     // [cols] or null
  const void* bias;       // [cols] or null
  void* y;                // [rows, cols] contiguous
  void* s;                // [rows, cols] contiguous, with res
  float* stats;           // [rows, 2]: mean, 1/std; or null
  long rows;
  int cols;
  long x_ld, res_ld;
  float eps;
  Dt dt, wdt;
};
void norm_forward(const NormArgs& a, hipStream_t stream);

struct NormGradArgs {
  const void* s;          // what was normalised [rows, cols], row stride s_ld
  const void* dy;         // [rows, cols], row stride dy_ld
  const void* ds;         // added to the result, or null
  const void* weight;     // or null
  const float* stats;     // [rows, 2]
  void* dx;               // [rows, cols] contiguous
  void* dweight;          // [cols] or null
  void* dbias;            // [cols] or null
  float* partial;         // [norm_grad_blocks(), 2, cols]
  long rows;
  int cols;
  long s_ld, dy_ld, ds_ld;
  Dt dt, wdt;
};
// How many rows of `partial` the backward pass writes for these sizes.
int norm_grad_blocks(long rows, int cols, Dt dt);
void norm_backward(const NormGradArgs& a, hipStream_t stream);

constexpr int kMostTop = 64;  // alternatives: one lane of a wave each

struct LogprobArgs {
  const void* x;            // logits [rows, vocab], row stride ld
  const int64_t* targets;   // [rows]
  float* logprobs;          // [rows]
  float* entropy;           // [rows]
  float* stats;             // [rows, 2]: maximum, sum around it
  int64_t* top_ids;         // [rows, top] or null
  float* top_logprobs;      // [rows, top] or null
  void* work;               // logprob_work_bytes(), 8-byte aligned
  long rows, ld;
  int vocab, top;
  int64_t ignore;
  Dt dt;
};
long logprob_work_bytes(long rows, int vocab, int top, Dt dt);
void logprob_forward(const LogprobArgs& a, hipStream_t stream);

struct LogprobGradArgs {
  const void* x;
  const int64_t* targets;
  const float* stats;       // of the forward pass
  const float* entropy;
  const float* glogprobs;   // [rows] or null
  const float* gentropy;    // [rows] or null
  void* dx;                 // [rows, vocab] contiguous
  long rows, ld;
  int vocab;
  int64_t ignore;
  Dt dt;
};
void logprob_backward(const LogprobGradArgs& a, hipStream_t stream);

enum class Act : int { none = 0, relu = 1, gelu = 2, silu = 3 };
// Which kernel makes a product: tiles; few rows of A, both operands along, straight
// from memory; floats with few rows of B or of A; short sums of floats (`tile`: the
// rows that a wave goes down).
enum class Way : int { tiles = 0, rows = 1, narrow_b = 2, narrow_a = 3, brief = 4 };

// C[m, n] = sum over k of A(m, k) B(n, k), and what becomes of it.  An operand
// lies with k innermost (A[m * ld + k]) or, `across`, with k outermost
// (A[k * ld + m]).
struct Operand {
  const void* p;
  long ld;
  bool across;
  bool padded;  // across: a row's last 8 elements may be read past its end
};
struct GemmArgs {
  Operand a, b;
  int m, n, k;
  Dt dt;              // of A, B, y, z, residual
  bool wide;          // A is float, whatever dt is
  void* y;            // [m, n], row stride y_ld: act(C + bias) + residual
  long y_ld;
  void* z;            // [m, n] contiguous: C + bias, or null
  const void* bias;   // [n] or null
  Dt bias_dt;
  const void* res;    // [m, n], row stride res_ld, or null
  long res_ld;
  Act act;
  float* work;        // gemm_work() floats
  Way way;            // how it is cut up, by gemm_plan
  int tile, slices;
};
// Sets how a product is cut up, from its sizes and layouts.
void gemm_plan(GemmArgs& g);
// The same for dx and dW of one layer (A of dx lies along, the rest across);
// whether one launch for both takes less time than two.
bool gemm_plan_two(GemmArgs& dx, GemmArgs& dw);
// The workspace that a planned product needs.
long gemm_work(const GemmArgs& g);
constexpr long kMostFeatures = 1L << 22;
// Whether a 16-bit product takes the operand as it lies (`rows` by k), 16
// bytes at a time; if not, pad_rows makes a copy that it takes.  Floats are
// taken as they lie, and so is everything along with gemm_few_rows.
bool gemm_takes(const Operand& o, long rows);
// Whether dz is kept in floats behind an activation that makes new numbers of it:
// where the products' time is the launch's.
bool gemm_keeps_floats(long m, long n, long k, Dt dt, Act act);
bool gemm_few_rows(long m, long n, long k, Dt dt);
void pad_rows(const void* from, long ld, void* to, long to_ld, int rows,
              int cols, Dt dt, hipStream_t stream);
void gemm_fused(const GemmArgs& a, hipStream_t stream);
void gemm_two(const GemmArgs& dx, const GemmArgs& dw, hipStream_t stream);

// dz = dy * act'(z) and the sums of its columns.
struct ActGradArgs {
  const void* dy;     // [m, n], row stride dy_ld
  long dy_ld;
  const void* z;      // [m, n], row stride z_ld; for relu the output may stand in
  long z_ld;
  void* dz;           // [m, n], row stride dz_ld, or null
  bool wide;          // dz is float, whatever dt is
  long dz_ld;
  void* dbias;        // [n] or null
  Dt bias_dt;
  float* partial;     // [act_grad_slices(), n], with dbias
  int m, n;
  Dt dt;
  Act act;
};
int act_grad_slices(int m, int n, Dt dt);
void act_grad(const ActGradArgs& a, hipStream_t stream);

}  // namespace cpd
