// Tensors in, tensors out: checks, allocation and streams of the layer-norm,
// linear and log-probability kernels.  Everything is enqueued on the current
// stream of the tensors' device, whichever device is current; workspaces come
// from torch's allocator in every call, so that two streams or two captured
// graphs never share one.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>
#include <torch/extension.h>

#include <optional>
#include <vector>

#include "fused_ops.h"

namespace {

using at::Tensor;
using cpd::Dt;
using OptTensor = std::optional<Tensor>;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

Dt dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return Dt::f32;
    case at::kBFloat16:
      return Dt::bf16;
    case at::kHalf:
      return Dt::f16;
    default:
      TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, got ",
                       t.scalar_type());
  }
}

// The memory that a kernel reads or writes.  Tensors without any (of a wrapper
// class, of a mode that only follows shapes, zeros known without being stored)
// have address 0, which a kernel would go to.
void check_memory(const void* p, const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(p || t.numel() == 0, name, " has no memory of its own");
}
void check_memory(const Tensor& t, const char* name) {
  check_memory(t.const_data_ptr(), t, name);
}
template <typename T = void>
T* made(const Tensor& t) {
  void* p = t.mutable_data_ptr();
  check_memory(p, t, "a tensor made for the result");
  return static_cast<T*>(p);
}

void check_on(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(),
                    ", the input on ", x.device());
  check_memory(t, name);
}

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  check_on(t, x, name);
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " is ",
                   t.scalar_type(), ", the input ", x.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == x.sizes(), name, " has shape ", t.sizes(),
                    ", wanted ", x.sizes());
}

// A learned vector: contiguous, of the input's type or float32.
std::optional<Tensor> learned(const OptTensor& t, const Tensor& x, int64_t n,
                              const char* name) {
  if (!t.has_value() || !t->defined()) return std::nullopt;
  check_on(*t, x, name);
  TORCH_CHECK_TYPE(
      t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat,
      name, " must be ", x.scalar_type(), " like the input, or float32, got ",
      t->scalar_type());
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == n, name, " has shape ",
                    t->sizes(), ", wanted [", n, "]");
  return t->resolve_neg().contiguous();
}

// A tensor as rows of its last axis: itself where the rows are evenly apart
// and their elements adjacent, a contiguous copy otherwise, and of a view that
// stands for the negative of what its memory holds (.imag of a conjugate).
struct Rows {
  Tensor keep;
  const void* p = nullptr;
  long rows = 0, cols = 0, ld = 0;
};

Rows rows_of(const Tensor& any) {
  const Tensor t = any.resolve_neg();
  Rows r;
  r.cols = t.size(-1);
  r.rows = r.cols ? t.numel() / r.cols : 0;
  // Stride of the leading axes joined into one.  Axes that do not join, and
  // rows that overlap (an expanded axis has stride 0), are copied.
  long ld = r.cols, next = 0;
  bool even = r.cols <= 1 || t.stride(-1) == 1, first = true;
  for (int64_t d = t.dim() - 2; d >= 0 && even; --d) {
    if (t.size(d) == 1) continue;
    even = t.stride(d) >= r.cols && (first || t.stride(d) == next);
    if (first) ld = t.stride(d);
    next = t.stride(d) * t.size(d);
    first = false;
  }
  if (!even) {
    r.keep = t.contiguous();
    ld = r.cols;
  } else {
    r.keep = t;
  }
  r.ld = ld;
  r.p = r.keep.const_data_ptr();
  check_memory(r.p, r.keep, "a tensor");
  return r;
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

void check_input(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.is_cuda(), name, " must be on the GPU");
  check_memory(x, name);
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------

// y, s (with a residual), stats [rows, 2]
std::vector<Tensor> norm_fwd(const Tensor& x, const OptTensor& weight,
                             const OptTensor& bias, double eps,
                             const OptTensor& residual) {
  check_input(x, "layer norm's input");
  cpd::NormArgs a{};
  a.dt = dtype_of(x, "layer norm's input");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1,
                    "layer norm needs a last axis of one element or more");
  TORCH_CHECK_VALUE(x.size(-1) < (1L << 30), "layer norm's last axis is too long");
  const Guard guard(x.device());
  const auto w = learned(weight, x, x.size(-1), "weight");
  const auto b = learned(bias, x, x.size(-1), "bias");
  TORCH_CHECK_TYPE(!w || !b || w->scalar_type() == b->scalar_type(),
                   "weight and bias must have one type");
  const Rows r = rows_of(x);
  Rows q;
  Tensor s;
  if (residual.has_value()) {
    check_like(*residual, x, "residual");
    q = rows_of(*residual);
    s = at::empty(x.sizes(), x.options());
    a.res = q.p;
    a.res_ld = q.ld;
    a.s = made(s);
  }
  TORCH_CHECK_VALUE(r.rows < (1L << 31), "layer norm takes less than 2^31 rows");
  TORCH_CHECK_VALUE(r.cols <= 16384 || r.rows < (1L << 22),
                    "layer norm takes less than 2^22 rows of this length");
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor stats = at::empty({r.rows, 2}, x.options().dtype(at::kFloat));
  a.x = r.p;
  a.x_ld = r.ld;
  a.weight = w ? w->const_data_ptr() : nullptr;
  a.bias = b ? b->const_data_ptr() : nullptr;
  a.wdt = w ? dtype_of(*w, "weight") : b ? dtype_of(*b, "bias") : a.dt;
  a.y = made(y);
  a.stats = made<float>(stats);
  a.rows = r.rows;
  a.cols = (int)r.cols;
  a.eps = (float)eps;
  cpd::norm_forward(a, stream_of(x));
  check_launch("layer norm");
  return {y, s, stats};
}

// dx, dweight, dbias
std::vector<Tensor> norm_bwd(const Tensor& s, const Tensor& dy,
                             const OptTensor& ds, const OptTensor& weight,
                             const Tensor& stats, bool need_w, bool need_b,
                             at::ScalarType bias_type) {
  check_input(s, "layer norm's input");
  const Guard guard(s.device());
  cpd::NormGradArgs a{};
  a.dt = dtype_of(s, "layer norm's input");
  const Rows r = rows_of(s);
  const auto w = learned(weight, s, r.cols, "weight");
  TORCH_CHECK_VALUE(stats.is_contiguous() && stats.numel() == 2 * r.rows &&
                        stats.scalar_type() == at::kFloat,
                    "stats are not this input's");
  check_on(stats, s, "stats");
  check_like(dy, s, "the output's gradient");
  const Rows g = rows_of(dy);
  a.dy = g.p;
  a.dy_ld = g.ld;
  Rows h;
  if (ds.has_value() && ds->defined()) {
    check_like(*ds, s, "the sum's gradient");
    h = rows_of(*ds);
    a.ds = h.p;
    a.ds_ld = h.ld;
  }
  const auto wtype = w ? w->scalar_type() : bias_type;
  const auto wopt = s.options().dtype(wtype);
  Tensor dx = at::empty(s.sizes(), s.options());
  Tensor dw, db, partial;
  if (need_w || need_b) {
    // no rows: the sums over them are zero
    if (need_w) dw = r.rows ? at::empty({r.cols}, wopt) : at::zeros({r.cols}, wopt);
    if (need_b) db = r.rows ? at::empty({r.cols}, wopt) : at::zeros({r.cols}, wopt);
    partial = at::empty(
        {cpd::norm_grad_blocks(r.rows, (int)r.cols, a.dt), 2, r.cols},
        s.options().dtype(at::kFloat));
    a.partial = made<float>(partial);
  }
  a.s = r.p;
  a.s_ld = r.ld;
  a.weight = w ? w->const_data_ptr() : nullptr;
  a.stats = stats.data_ptr<float>();
  a.dx = made(dx);
  a.dweight = need_w ? made(dw) : nullptr;
  a.dbias = need_b ? made(db) : nullptr;
  a.rows = r.rows;
  a.cols = (int)r.cols;
  a.wdt = wtype == at::kFloat      ? Dt::f32
          : wtype == at::kBFloat16 ? Dt::bf16
                                   : Dt::f16;
  cpd::norm_backward(a, stream_of(s));
  check_launch("layer norm backward");
  return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// log probabilities
// ---------------------------------------------------------------------------

// logprobs, entropy, stats, top_ids, top_logprobs
std::vector<Tensor> logprob_fwd(const Tensor& x, const Tensor& targets,
                                int64_t top, int64_t ignore) {
  check_input(x, "logits");
  cpd::LogprobArgs a{};
  a.dt = dtype_of(x, "logits");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1L << 30),
                    "logits need a last axis of 1 to 2^30 - 1 entries");
  check_on(targets, x, "targets");
  TORCH_CHECK_TYPE(targets.scalar_type() == at::kLong, "targets must be int64, got ",
                   targets.scalar_type());
  TORCH_CHECK_VALUE(targets.sizes() == x.sizes().slice(0, x.dim() - 1),
                    "targets have shape ", targets.sizes(), ", logits ", x.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= cpd::kMostTop && top <= x.size(-1),
                    "top_k must be 0 to ", cpd::kMostTop,
                    " and at most the number of logits, got ", top);
  const Guard guard(x.device());
  const Rows r = rows_of(x);
  const Tensor t = targets.contiguous();
  const auto f = x.options().dtype(at::kFloat);
  Tensor lp = at::empty(t.sizes(), f), ent = at::empty(t.sizes(), f);
  Tensor stats = at::empty({r.rows, 2}, f);
  Tensor ids, tops, work;
  if (top) {
    auto shape = t.sizes().vec();
    shape.push_back(top);
    ids = at::empty(shape, t.options());
    tops = at::empty(shape, f);
  }
  const long bytes = cpd::logprob_work_bytes(r.rows, (int)r.cols, (int)top, a.dt);
  if (bytes) work = at::empty({bytes}, x.options().dtype(at::kByte));
  a.x = r.p;
  a.ld = r.ld;
  a.targets = t.data_ptr<int64_t>();
  a.logprobs = made<float>(lp);
  a.entropy = made<float>(ent);
  a.stats = made<float>(stats);
  a.top_ids = top ? made<int64_t>(ids) : nullptr;
  a.top_logprobs = top ? made<float>(tops) : nullptr;
  a.work = bytes ? made(work) : nullptr;
  a.rows = r.rows;
  a.vocab = (int)r.cols;
  a.top = (int)top;
  a.ignore = ignore;
  cpd::logprob_forward(a, stream_of(x));
  check_launch("token log probabilities");
  return {lp, ent, stats, ids, tops};
}

Tensor logprob_bwd(const Tensor& x, const Tensor& targets, const Tensor& stats,
                   const Tensor& entropy, const OptTensor& glp,
                   const OptTensor& gent, int64_t ignore) {
  check_input(x, "logits");
  const Guard guard(x.device());
  cpd::LogprobGradArgs a{};
  a.dt = dtype_of(x, "logits");
  const Rows r = rows_of(x);
  const Tensor t = targets.contiguous(), e = entropy.contiguous();
  TORCH_CHECK_VALUE(t.numel() == r.rows && e.numel() == r.rows &&
                        stats.numel() == 2 * r.rows && stats.is_contiguous(),
                    "saved tensors are not these logits'");
  Tensor g, h;
  if (glp.has_value() && glp->defined()) g = glp->to(at::kFloat).resolve_neg().contiguous();
  if (gent.has_value() && gent->defined()) h = gent->to(at::kFloat).resolve_neg().contiguous();
  for (const Tensor* v : {&g, &h}) {
    if (v->defined()) check_memory(*v, "a gradient");
    TORCH_CHECK_VALUE(!v->defined() || (v->device() == x.device() &&
                                        v->numel() == r.rows),
                      "a gradient does not fit the logits");
  }
  Tensor dx = at::empty(x.sizes(), x.options());
  a.x = r.p;
  a.ld = r.ld;
  a.targets = t.data_ptr<int64_t>();
  a.stats = stats.data_ptr<float>();
  a.entropy = e.data_ptr<float>();
  a.glogprobs = g.defined() ? g.data_ptr<float>() : nullptr;
  a.gentropy = h.defined() ? h.data_ptr<float>() : nullptr;
  a.dx = made(dx);
  a.rows = r.rows;
  a.vocab = (int)r.cols;
  a.ignore = ignore;
  cpd::logprob_backward(a, stream_of(x));
  check_launch("token log probabilities backward");
  return dx;
}

// ---------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------

cpd::Act act_of(int64_t act) {
  TORCH_CHECK_VALUE(act >= 0 && act <= 3, "unknown activation");
  return static_cast<cpd::Act>(act);
}

// m rows of k features in, n out: what the kernels count in 32 bits, for the
// product and for both of its gradients.
void check_sizes(int64_t m, int64_t n, int64_t k) {
  TORCH_CHECK_VALUE(m < (1L << 31) - 8192, "linear takes less than 2^31 - 8192 rows");
  TORCH_CHECK_VALUE(n < cpd::kMostFeatures && k < cpd::kMostFeatures,
                    "linear takes less than 2^22 features");
  auto tiles = [](int64_t a, int64_t b) { return ((a + 127) / 128) * ((b + 127) / 128); };
  TORCH_CHECK_VALUE(tiles(m, n) < (1L << 22) && tiles(m, k) < (1L << 22) &&
                        tiles(n, k) < (1L << 22),
                    "linear's tensors are too large");
}

// Where rows are laid out here, they begin on a 128-byte line: a tile's 64 k of
// a row are one line then and not parts of two (38 us instead of 56 for 1023 x
// 5000 by 2050).
int64_t whole_lines(int64_t cols) { return (cols + 63) / 64 * 64; }

// The products of a call: operands as the kernels read them, and workspaces,
// kept until all is enqueued.
struct Products {
  Dt dt;
  hipStream_t st;
  std::vector<Tensor> keep;

  // `any`: the kernel takes it as it lies
  cpd::Operand operand(const Rows& r, bool across, bool padded, bool any,
                       const Tensor& like) {
    cpd::Operand o{r.p, r.ld, across, padded};
    if (any || dt == Dt::f32 || r.rows == 0 ||
        cpd::gemm_takes(o, across ? r.cols : r.rows))
      return o;
    const int64_t ld = whole_lines(r.cols);
    keep.push_back(at::empty({r.rows, ld}, like.options()));
    cpd::pad_rows(r.p, r.ld, made(keep.back()), ld, (int)r.rows,
                  (int)r.cols, dt, st);
    return {keep.back().const_data_ptr(), ld, across, true};
  }

  // The workspace of a planned product.
  void give_work(cpd::GemmArgs& g, const Tensor& like) {
    const long floats = cpd::gemm_work(g);
    if (!floats) return;
    keep.push_back(at::empty({floats}, like.options().dtype(at::kFloat)));
    g.work = made<float>(keep.back());
  }

  void run(cpd::GemmArgs& g, const Tensor& like) {
    cpd::gemm_plan(g);
    give_work(g, like);
    cpd::gemm_fused(g, st);
  }

  void run_two(cpd::GemmArgs& dx, cpd::GemmArgs& dw, const Tensor& like) {
    const bool together = cpd::gemm_plan_two(dx, dw);
    give_work(dx, like);
    give_work(dw, like);
    if (together) {
      cpd::gemm_two(dx, dw, st);
    } else {
      cpd::gemm_fused(dx, st);
      cpd::gemm_fused(dw, st);
    }
  }
};

// y, z (with want_z: act's argument, in the input's type)
std::vector<Tensor> linear_fwd(const Tensor& x, const Tensor& weight,
                               const OptTensor& bias, int64_t act,
                               const OptTensor& residual, bool want_z) {
  check_input(x, "linear's input");
  cpd::GemmArgs g{};
  g.dt = dtype_of(x, "linear's input");
  g.act = act_of(act);
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1),
                    "linear's input has shape ", x.sizes(), ", its weight ",
                    weight.sizes());
  check_on(weight, x, "weight");
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "weight is ",
                   weight.scalar_type(), ", the input ", x.scalar_type());
  TORCH_CHECK_VALUE(weight.size(1) >= 1, "linear needs one input feature or more");
  const Guard guard(x.device());
  const auto b = learned(bias, x, weight.size(0), "bias");
  const Rows r = rows_of(x), w = rows_of(weight);
  check_sizes(r.rows, weight.size(0), r.cols);
  auto shape = x.sizes().vec();
  shape.back() = weight.size(0);
  Tensor y = at::empty(shape, x.options()), z;
  Rows q;
  if (residual.has_value()) {
    check_like(*residual, y, "residual");
    q = rows_of(*residual);
    g.res = q.p;
    g.res_ld = q.ld;
  }
  if (want_z) {
    z = at::empty(shape, x.options());
    g.z = made(z);
  }
  Products products{g.dt, stream_of(x), {}};
  const bool few = cpd::gemm_few_rows(r.rows, w.rows, r.cols, g.dt);
  g.a = products.operand(r, false, false, few, x);
  g.b = products.operand(w, false, false, few, x);
  g.m = (int)r.rows;
  g.n = (int)weight.size(0);
  g.k = (int)r.cols;
  g.y = made(y);
  g.y_ld = g.n;
  g.bias = b ? b->const_data_ptr() : nullptr;
  g.bias_dt = b ? dtype_of(*b, "bias") : g.dt;
  products.run(g, x);
  check_launch("linear");
  return {y, z};
}

// dx, dweight, dbias
std::vector<Tensor> linear_bwd(const Tensor& dy, const Tensor& x,
                               const Tensor& weight, const OptTensor& z,
                               int64_t act, bool need_x, bool need_w,
                               bool need_b, at::ScalarType bias_type) {
  check_input(x, "linear's input");
  const Guard guard(x.device());
  const hipStream_t st = stream_of(x);
  const Dt dt = dtype_of(x, "linear's input");
  const int64_t n = weight.size(0), k = weight.size(1);
  const Rows r = rows_of(x), w = rows_of(weight);
  check_on(dy, x, "the output's gradient");
  TORCH_CHECK_TYPE(dy.scalar_type() == x.scalar_type(), "the output's gradient is ",
                   dy.scalar_type(), ", the input ", x.scalar_type());
  TORCH_CHECK_VALUE(dy.size(-1) == n && dy.numel() == r.rows * n,
                    "the output's gradient has shape ", dy.sizes());
  const int64_t m = r.rows;
  check_sizes(m, n, k);
  Rows g = rows_of(dy);
  g.rows = m;
  Tensor dx, dw, db, dz, partial;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_w) dw = m ? at::empty({n, k}, x.options()) : at::zeros({n, k}, x.options());
  const auto bopt = x.options().dtype(bias_type);
  if (need_b) db = m ? at::empty({n}, bopt) : at::zeros({n}, bopt);
  if (m == 0 || n == 0) {
    if (need_x && n == 0) dx.zero_();
    return {dx, dw, db};
  }
  cpd::ActGradArgs p{};
  p.act = act_of(act);
  p.dt = dt;
  p.m = (int)m;
  p.n = (int)n;
  p.dy = g.p;
  p.dy_ld = g.ld;
  Rows zr;
  if (p.act != cpd::Act::none) {
    TORCH_CHECK_VALUE(z.has_value() && z->numel() == m * n, "linear kept no z");
    zr = rows_of(*z);
    p.z = zr.p;
    p.z_ld = zr.ld;
  }
  // dz, or a copy of a dy that the products do not take as it lies
  const bool fits =
      dt == Dt::f32 || ((!need_x || cpd::gemm_takes({g.p, g.ld, false, false}, m)) &&
                        (!need_w || cpd::gemm_takes({g.p, g.ld, true, false}, n)));
  const bool wide = cpd::gemm_keeps_floats(m, n, k, dt, p.act);
  if ((need_x || need_w) && (p.act != cpd::Act::none || !fits)) {
    g.ld = whole_lines(n);
    dz = at::empty({m, g.ld}, wide ? x.options().dtype(at::kFloat) : x.options());
    p.wide = wide;
    p.dz = made(dz);
    p.dz_ld = g.ld;
    g.p = p.dz;
    g.keep = dz;
  }
  if (need_b) {
    p.dbias = made(db);
    p.bias_dt = bias_type == at::kFloat ? Dt::f32 : dt;
    partial = at::empty({cpd::act_grad_slices(p.m, p.n, dt), n},
                        x.options().dtype(at::kFloat));
    p.partial = made<float>(partial);
  }
  if (need_b || p.dz) cpd::act_grad(p, st);
  // dx: dz [m, n] with W [n, k], the sum runs over n;
  // dW: dz^T x, the sum runs over m
  Products products{dt, st, {}};
  const bool padded = p.dz != nullptr;
  cpd::GemmArgs q{}, v{};
  q.dt = q.bias_dt = v.dt = v.bias_dt = dt;
  q.wide = v.wide = wide;
  q.n = v.n = (int)k;
  q.y_ld = v.y_ld = k;
  if (need_x) {
    q.a = products.operand(g, false, padded, wide, x);
    q.b = products.operand(w, true, false, wide, x);
    q.m = (int)m;
    q.k = (int)n;
    q.y = made(dx);
  }
  if (need_w) {
    v.a = products.operand(g, true, padded, wide, x);
    v.b = products.operand(r, true, false, wide, x);
    v.m = (int)n;
    v.k = (int)m;
    v.y = made(dw);
  }
  if (need_x && need_w)
    products.run_two(q, v, x);
  else if (need_x)
    products.run(q, x);
  else if (need_w)
    products.run(v, x);
  check_launch("linear backward");
  return {dx, dw, db};
}

// How the products of m rows, n features out and k in are cut up (without an
// activation): tile and slices of forward, of dx and of dW, whether a call for
// both gradients takes one launch, and the three products' way.  Which kernels run
// is not seen in the results, and tests have to reach every one.
std::vector<int64_t> linear_plan(int64_t m, int64_t n, int64_t k,
                                 at::ScalarType type, bool need_x, bool need_w) {
  check_sizes(m, n, k);
  const Dt dt = type == at::kFloat      ? Dt::f32
                : type == at::kBFloat16 ? Dt::bf16
                                        : Dt::f16;
  auto product = [&](int64_t rows, int64_t cols, int64_t sum, bool ax, bool bx) {
    cpd::GemmArgs g{};
    g.dt = dt;
    g.m = (int)rows;
    g.n = (int)cols;
    g.k = (int)sum;
    g.a.across = ax;
    g.b.across = bx;
    return g;
  };
  auto y = product(m, n, k, false, false), dx = product(m, k, n, false, true),
       dw = product(n, k, m, true, true);
  cpd::gemm_plan(y);
  bool together = false;
  if (need_x && need_w) {
    together = cpd::gemm_plan_two(dx, dw);
  } else {
    cpd::gemm_plan(dx);
    cpd::gemm_plan(dw);
  }
  return {y.tile,    y.slices,   dx.tile,     dx.slices,   dw.tile,
          dw.slices, together, (int)y.way, (int)dx.way, (int)dw.way};
}

// ---------------------------------------------------------------------------
// The operators with their gradients.  The graph's nodes are C++: a backward
// pass through Python's own function class costs about 50 us of waiting for
// the interpreter, more than most of these kernels take.
// ---------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Whether a node has to stand for this call: for a gradient, or for a tangent
// of forward mode, which the node refuses and a bare call would lose.
bool wants_grad(const Tensor& t) {
  return (t.requires_grad() && at::GradMode::is_enabled()) ||
         t._fw_grad(0).defined();
}
bool wants_grad(const OptTensor& t) {
  return t.has_value() && t->defined() && wants_grad(*t);
}

bool present(const OptTensor& t) { return t.has_value() && t->defined(); }

OptTensor some(const Tensor& t) {
  return t.defined() ? OptTensor(t) : std::nullopt;
}

// (an edge for every tensor that forward was given, in its order)
bool needs(const AutogradContext* ctx, const char* name) {
  const auto edge = ctx->saved_data.at(name).toInt();
  return edge >= 0 && ctx->needs_input_grad(edge);
}
void name_edges(AutogradContext* ctx,
                std::initializer_list<std::pair<const char*, bool>> inputs) {
  int64_t edge = 0;
  for (const auto& in : inputs) ctx->saved_data[in.first] = in.second ? edge++ : -1;
}

void check_once(const char* what) {
  // gradients are asked for with their own graph only to differentiate again
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " cannot be differentiated twice (create_graph=True)");
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const OptTensor& weight, const OptTensor& bias,
                               double eps, const OptTensor& residual) {
    auto out = norm_fwd(x, weight, bias, eps, residual);
    ctx->set_materialize_grads(false);
    name_edges(ctx, {{"x", true}, {"weight", present(weight)},
                     {"bias", present(bias)}, {"residual", present(residual)}});
    ctx->saved_data["type"] = bias ? bias->scalar_type() : x.scalar_type();
    ctx->save_for_backward({residual ? out[1] : x, weight.value_or(Tensor()),
                            out[2]});
    if (residual) return {out[0], out[1]};
    return {out[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("layer norm");
    const Tensor ds = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined() && !ds.defined()) return variable_list(5);
    const bool x = needs(ctx, "x"), w = needs(ctx, "weight"),
               b = needs(ctx, "bias"), res = needs(ctx, "residual");
    const auto type = ctx->saved_data["type"].toScalarType();
    if (!g[0].defined()) {
      // Only the sum was used: its gradient is x's and the residual's as it is,
      // also in rows whose norm is not finite.
      const auto none = [&](bool need) {
        return need ? at::zeros({ds.size(-1)}, ds.options().dtype(type)) : Tensor();
      };
      return {x ? ds : Tensor(), none(w), none(b), Tensor(), res ? ds : Tensor()};
    }
    const auto saved = ctx->get_saved_variables();
    auto d = norm_bwd(saved[0], g[0], some(ds), some(saved[1]), saved[2], w, b, type);
    return {x ? d[0] : Tensor(), d[1], d[2], Tensor(), res ? d[0] : Tensor()};
  }
};

std::vector<Tensor> layer_norm(const Tensor& x, const OptTensor& weight,
                               const OptTensor& bias, double eps,
                               const OptTensor& residual) {
  if (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))
    return LayerNorm::apply(x, weight, bias, eps, residual);
  auto out = norm_fwd(x, weight, bias, eps, residual);
  out.resize(residual ? 2 : 1);
  return out;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& weight, const OptTensor& bias, int64_t act,
                        const OptTensor& residual) {
    // relu's slope can be read off its own output, unless a residual was added
    // to that
    const bool from_y = act_of(act) == cpd::Act::relu && !residual;
    auto out = linear_fwd(x, weight, bias, act, residual, act != 0 && !from_y);
    ctx->set_materialize_grads(false);
    name_edges(ctx, {{"x", true}, {"weight", true}, {"bias", present(bias)},
                     {"residual", present(residual)}});
    ctx->saved_data["act"] = act;
    ctx->saved_data["type"] = bias ? bias->scalar_type() : x.scalar_type();
    ctx->save_for_backward({x, weight, from_y ? out[0] : out[1]});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("linear");
    const Tensor dy = g[0];
    if (!dy.defined()) return variable_list(5);
    const bool x = needs(ctx, "x"), w = needs(ctx, "weight"), b = needs(ctx, "bias");
    std::vector<Tensor> d(3);
    if (x || w || b) {
      const auto saved = ctx->get_saved_variables();
      d = linear_bwd(dy, saved[0], saved[1], some(saved[2]),
                     ctx->saved_data["act"].toInt(), x, w, b,
                     ctx->saved_data["type"].toScalarType());
    }
    return {d[0], d[1], d[2], Tensor(), needs(ctx, "residual") ? dy : Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias,
              int64_t act, const OptTensor& residual) {
  if (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))
    return Linear::apply(x, weight, bias, act, residual);
  return linear_fwd(x, weight, bias, act, residual, false)[0];
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const Tensor& targets, int64_t top, int64_t ignore) {
    auto out = logprob_fwd(x, targets, top, ignore);
    ctx->set_materialize_grads(false);
    ctx->saved_data["ignore"] = ignore;
    ctx->save_for_backward({x, targets, out[2], out[1]});
    if (!top) return {out[0], out[1]};
    ctx->mark_non_differentiable({out[3], out[4]});
    return {out[0], out[1], out[3], out[4]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("token log probabilities");
    if (!g[0].defined() && !g[1].defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    return {logprob_bwd(saved[0], saved[1], saved[2], saved[3], some(g[0]),
                        some(g[1]), ctx->saved_data["ignore"].toInt()),
            Tensor(), Tensor(), Tensor()};
  }
};

// logprobs, entropy, and with top > 0 ids and log probabilities
std::vector<Tensor> token_logprobs(const Tensor& x, const Tensor& targets,
                                   int64_t top, int64_t ignore) {
  if (wants_grad(x))
    return TokenLogprobs::apply(x, targets, top, ignore);
  auto out = logprob_fwd(x, targets, top, ignore);
  if (!top) return {out[0], out[1]};
  return {out[0], out[1], out[3], out[4]};
}

}  // namespace

void cpd_register_fused(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm, "layer norm (+residual): [y] or [y, s]");
  m.def("linear", &linear, "act(x W^T + bias) + residual");
  m.def("linear_plan", &linear_plan,
        "[tile, slices] of y, dx and dW, whether the last two share a launch, "
        "and the way of each");
  m.def("token_logprobs", &token_logprobs,
        "[logprobs, entropy] or [logprobs, entropy, top_ids, top_logprobs]");
}
