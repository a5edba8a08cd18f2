// Bindings and autograd of the training operators: layer norm, GELU and
// linear with 8-bit checkpoints, and the cross entropy. Checks of arguments
// are here; the kernels (norm.cu, act8.cu, wgrad8.cu, xent.cu) trust them.

#include <ATen/ATen.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <tuple>
#include <vector>

#include "train.hpp"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

train::Type type_of(const Tensor& x, const char* who, const char* what) {
  switch (x.scalar_type()) {
    case at::kFloat:
      return train::Type::f32;
    case at::kBFloat16:
      return train::Type::bf16;
    case at::kHalf:
      return train::Type::f16;
    default:
      TORCH_CHECK(false, who, ": ", what, " must be float32, bfloat16 or float16, got ", x.scalar_type());
  }
}

void check_dtype(at::ScalarType t, const char* who, const char* what) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, who, ": ", what,
              " must be float32, bfloat16 or float16, got ", t);
}

// Rows of a tensor whose last dimension is a row: adjacent elements, one
// distance between rows. Other orders are copied into this form.
struct Mat {
  Tensor t;  // keeps a copy alive
  train::Rows rows;
  std::int64_t n = 0, cols = 0;
};

Mat matrix(const Tensor& x, const char* who, const char* what) {
  TORCH_CHECK(x.is_cuda(), who, ": ", what, " must be a CUDA tensor");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, who, ": ", what, " needs rows of one element at least");
  Mat m;
  m.rows.t = type_of(x, who, what);
  m.cols = x.size(-1);
  m.n = x.numel() / m.cols;
  bool ok = m.cols == 1 || x.stride(-1) == 1;
  std::int64_t ld = m.cols;
  bool first = true;
  std::int64_t span = 0;  // distance that the next outer dimension has to have
  for (std::int64_t d = x.dim() - 2; ok && d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (first)
      ld = x.stride(d), first = false;
    else
      ok = x.stride(d) == span;
    span = x.stride(d) * x.size(d);
  }
  if (m.n == 0) ok = true;
  m.t = ok ? x : x.contiguous();
  m.rows.ld = ok ? ld : m.cols;
  m.rows.p = m.t.data_ptr();
  return m;
}

void same_device(const Tensor& a, const Tensor& b, const char* who, const char* what) {
  TORCH_CHECK(b.is_cuda() && a.device() == b.device(), who, ": ", what, " must be on ", a.device(), ", got ",
              b.device());
}

// A vector over the columns, contiguous.
Tensor column_vector(const Tensor& v, const Tensor& x, std::int64_t cols, const char* who, const char* what) {
  same_device(x, v, who, what);
  TORCH_CHECK(v.dim() == 1 && v.size(0) == cols, who, ": ", what, " must have shape [", cols, "], got ", v.sizes());
  check_dtype(v.scalar_type(), who, what);
  return v.contiguous();
}

Tensor defined_or(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Held {  // the two tensors of an 8-bit form
  Tensor q, scale;
};

Held new_held(const Tensor& like, std::int64_t rows, std::int64_t cols) {
  const auto ng = train::groups(cols);
  return {at::empty({rows, ng * train::kGroup}, like.options().dtype(at::kChar)),
          at::empty({rows, ng}, like.options().dtype(at::kByte))};
}

void check_held(const Tensor& q, const Tensor& scale, std::int64_t rows, std::int64_t cols, const char* who) {
  TORCH_CHECK(q.is_cuda() && scale.is_cuda() && q.device() == scale.device(), who,
              ": the 8-bit form must be CUDA tensors on one device");
  TORCH_CHECK(q.scalar_type() == at::kChar && scale.scalar_type() == at::kByte && q.is_contiguous() &&
                  scale.is_contiguous(),
              who, ": the 8-bit form is contiguous int8 values and uint8 scales");
  const auto ng = train::groups(cols);
  TORCH_CHECK(q.dim() == 2 && q.size(0) == rows && q.size(1) == ng * train::kGroup && scale.dim() == 2 &&
                  scale.size(0) == rows && scale.size(1) == ng,
              who, ": the 8-bit form of ", rows, " rows of ", cols, " has shapes [", rows, ", ", ng * train::kGroup,
              "] and [", rows, ", ", ng, "], got ", q.sizes(), " and ", scale.sizes());
  TORCH_CHECK(reinterpret_cast<std::uintptr_t>(q.data_ptr()) % 16 == 0, who,
              ": the 8-bit values must start on a 16-byte boundary");
}

std::int8_t* q_ptr(const Tensor& q) { return q.defined() ? q.data_ptr<std::int8_t>() : nullptr; }
std::uint8_t* s_ptr(const Tensor& s) { return s.defined() ? s.data_ptr<std::uint8_t>() : nullptr; }

// A kernel whose wait ran out has left NaN. Its call has returned long before, so
// the next one says it; the word is in host memory and nothing waits for the GPU.
void check_waits(const char* who) {
  TORCH_CHECK(!commux_ops::wait_gave_up(), who,
              ": a kernel's wait has run out (COMMUX_KERNEL_WAIT_MS), and results since then may "
              "be NaN; commux_b200.ops.kernel_status(reset=True) clears this");
}

void no_second_order(const char* who) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who, ": the backward pass has no derivative (create_graph=True)");
}

// Whether autograd will ask for a gradient of x (inside a Function's forward
// the grad mode is off, so this is asked before).
bool graph(const Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }
bool graph(const optional<Tensor>& x) { return x.has_value() && graph(*x); }

// --- layer norm ----------------------------------------------------------------

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  // returns y, then s (if a residual is given), then q and scale (if packed)
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual,
                               const Tensor& weight, const optional<Tensor>& bias, double eps, at::ScalarType out,
                               bool pack, bool train) {
    const char* who = "layer_norm";
    check_waits(who);
    const Mat m = matrix(x, who, "x");
    check_dtype(out, who, "out_dtype");
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor w = column_vector(weight, x, m.cols, who, "weight");
    Tensor b = defined_or(bias);
    if (b.defined()) {
      b = column_vector(b, x, m.cols, who, "bias");
      TORCH_CHECK(b.scalar_type() == w.scalar_type(), who, ": weight and bias must have one dtype");
    }
    Mat r;
    if (residual.has_value()) {
      TORCH_CHECK(residual->sizes() == x.sizes(), who, ": residual must have x's shape ", x.sizes(), ", got ",
                  residual->sizes());
      r = matrix(*residual, who, "residual");
      same_device(x, *residual, who, "residual");
    }
    const Tensor y = at::empty(x.sizes(), x.options().dtype(out));
    const Tensor s = r.t.defined() ? at::empty(x.sizes(), x.options()) : Tensor();
    Held held;
    if (pack) held = new_held(x, m.n, m.cols);
    Tensor stats;  // rstd and, unless packed, mean
    if (train) stats = at::empty({pack ? 1 : 2, m.n}, x.options().dtype(at::kFloat));
    if (m.n > 0) {
      train::NormFwd a{};
      a.x = m.rows;
      a.r = r.rows;
      a.w = w.data_ptr();
      a.b = ptr(b);
      a.wt = type_of(w, who, "weight");
      a.s = out_ptr(s);
      a.y = y.data_ptr();
      a.yt = type_of(y, who, "out_dtype");
      a.q = q_ptr(held.q);
      a.scale = s_ptr(held.scale);
      a.rstd = train ? stats.data_ptr<float>() : nullptr;
      a.mean = train && !pack ? a.rstd + m.n : nullptr;
      a.rows = m.n;
      a.cols = m.cols;
      a.eps = static_cast<float>(eps);
      C10_CUDA_CHECK(train::norm_forward(a, stream_of(x)));
    }
    ctx->set_materialize_grads(false);
    variable_list outs{y};
    if (s.defined()) outs.push_back(s);
    if (pack) {
      outs.push_back(held.q);
      outs.push_back(held.scale);
      ctx->mark_non_differentiable({held.q, held.scale});
    }
    if (train) {
      // the packed form replaces the stream itself in what is kept
      ctx->save_for_backward({pack ? Tensor() : s.defined() ? s : m.t, held.q, held.scale, stats, weight});
      // dtypes of x and of the residual, and whether there is a bias, in one number: every entry costs host time
      ctx->saved_data["kinds"] = static_cast<int64_t>(x.scalar_type()) |
                                 (r.t.defined() ? static_cast<int64_t>(residual->scalar_type()) : int64_t{0xff}) << 8 |
                                 static_cast<int64_t>(b.defined()) << 16;
    }
    return outs;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "layer_norm";
    check_waits(who);
    no_second_order(who);
    const auto saved = ctx->get_saved_variables();
    const Tensor &kept = saved[0], &q = saved[1], &scale = saved[2], &stats = saved[3], &weight = saved[4];
    const int64_t kinds = ctx->saved_data["kinds"].toInt();
    const auto xt = static_cast<at::ScalarType>(kinds & 0xff), rt = static_cast<at::ScalarType>(kinds >> 8 & 0xff);
    const bool has_bias = kinds >> 16 != 0, has_residual = (kinds >> 8 & 0xff) != 0xff;
    const Tensor dy = grads[0], ds = has_residual ? grads[1] : Tensor();
    variable_list out(8);
    const auto opts = stats.options();
    if (!dy.defined()) {  // only the stream was used
      if (ds.defined()) {
        out[0] = ds;
        if (has_residual) out[1] = ds.to(rt);
      }
      return out;
    }
    c10::cuda::CUDAGuard guard(stats.device());
    const Tensor w = weight.contiguous();
    const Mat mdy = matrix(dy, who, "gradient");
    Mat mds, ms;
    if (ds.defined()) mds = matrix(ds, who, "gradient");
    train::NormBwd a{};
    a.rows = stats.size(1);
    a.cols = w.size(0);
    const auto sizes = dy.sizes();
    const Tensor dx = at::empty(sizes, opts.dtype(xt));
    Tensor dr;
    // graph edges are counted over the tensors that were given
    const bool need_r = has_residual && ctx->needs_input_grad(1);
    if (need_r && rt != xt) dr = at::empty(sizes, opts.dtype(rt));
    const size_t w_edge = has_residual ? 2 : 1;
    const bool need_w = ctx->needs_input_grad(w_edge), need_b = has_bias && ctx->needs_input_grad(w_edge + 1);
    const Tensor dw = need_w ? at::empty_like(w) : Tensor(), db = need_b ? at::empty_like(w) : Tensor();
    if (a.rows > 0) {
      a.dy = mdy.rows;
      a.ds = mds.rows;
      if (q.defined()) {
        a.q = q_ptr(q);
        a.scale = s_ptr(scale);
      } else {
        ms = matrix(kept, who, "x");
        a.s = ms.rows;
        a.mean = stats.data_ptr<float>() + a.rows;
      }
      a.rstd = stats.data_ptr<float>();
      a.w = w.data_ptr();
      a.wt = type_of(w, who, "weight");
      a.dx = dx.data_ptr();
      a.xt = type_of(dx, who, "x");
      a.dr = out_ptr(dr);
      a.rt = dr.defined() ? type_of(dr, who, "residual") : a.xt;
      a.dw = out_ptr(dw);
      a.db = out_ptr(db);
      const Tensor work = at::empty({train::norm_backward_work(a)}, opts);
      a.work = work.data_ptr<float>();
      C10_CUDA_CHECK(train::norm_backward(a, stream_of(dx)));
    } else {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
    }
    if (ctx->needs_input_grad(0)) out[0] = dx;
    if (need_r) out[1] = dr.defined() ? dr : dx;
    out[2] = dw;
    out[3] = db;
    return out;
  }
};

variable_list layer_norm(const Tensor& x, const optional<Tensor>& residual, const Tensor& weight,
                         const optional<Tensor>& bias, double eps, at::ScalarType out, bool pack) {
  return LayerNorm::apply(x, residual, weight, bias, eps, out, pack,
                          graph(x) || graph(weight) || graph(residual) || graph(bias));
}

// --- 8-bit form ------------------------------------------------------------------

std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  check_waits("pack8");
  const Mat m = matrix(x, "pack8", "x");
  c10::cuda::CUDAGuard guard(x.device());
  const Held h = new_held(x, m.n, m.cols);
  if (m.n > 0)
    C10_CUDA_CHECK(train::pack8(m.rows, q_ptr(h.q), s_ptr(h.scale), m.n, m.cols, stream_of(x)));
  return {h.q, h.scale};
}

Tensor unpack8(const Tensor& q, const Tensor& scale, std::vector<int64_t> sizes, at::ScalarType dtype,
               const optional<Tensor>& weight, const optional<Tensor>& bias) {
  const char* who = "unpack8";
  check_waits(who);
  check_dtype(dtype, who, "dtype");
  TORCH_CHECK(!sizes.empty() && sizes.back() >= 1, who, ": shape needs rows of one element at least");
  const int64_t cols = sizes.back(), rows = c10::multiply_integers(sizes) / cols;
  check_held(q, scale, rows, cols, who);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor w = defined_or(weight), b = defined_or(bias);
  if (w.defined()) w = column_vector(w, q, cols, who, "weight");
  if (b.defined()) b = column_vector(b, q, cols, who, "bias");
  TORCH_CHECK(!b.defined() || (w.defined() && w.scalar_type() == b.scalar_type()), who,
              ": a bias comes with a weight of its dtype");
  const Tensor out = at::empty(sizes, q.options().dtype(dtype));
  if (rows > 0)
    C10_CUDA_CHECK(train::unpack8(q_ptr(q), s_ptr(scale), ptr(w), ptr(b),
                                  w.defined() ? type_of(w, who, "weight") : train::Type::f32, out.data_ptr(),
                                  type_of(out, who, "dtype"), rows, cols, stream_of(q)));
  return out;
}

// --- GELU ------------------------------------------------------------------------

template <bool kTanh>
struct Gelu8 : torch::autograd::Function<Gelu8<kTanh>> {
  // returns y, then its 8-bit form (if packed)
  static variable_list forward(AutogradContext* ctx, const Tensor& x, bool pack, bool train) {
    const char* who = "gelu8";
    check_waits(who);
    const Mat m = matrix(x, who, "x");
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = at::empty(x.sizes(), x.options());
    Held h, hy;
    if (train) h = new_held(x, m.n, m.cols);
    if (pack) hy = new_held(x, m.n, m.cols);
    if (m.n > 0) {
      train::GeluFwd a{};
      a.x = m.rows;
      a.y = y.data_ptr();
      a.q = q_ptr(h.q);
      a.scale = s_ptr(h.scale);
      a.yq = q_ptr(hy.q);
      a.yscale = s_ptr(hy.scale);
      a.rows = m.n;
      a.cols = m.cols;
      a.tanh_form = kTanh;
      C10_CUDA_CHECK(train::gelu8_forward(a, stream_of(x)));
    }
    if (train) ctx->save_for_backward({h.q, h.scale});
    variable_list outs{y};
    if (pack) {
      outs.push_back(hy.q);
      outs.push_back(hy.scale);
      ctx->mark_non_differentiable({hy.q, hy.scale});
    }
    ctx->set_materialize_grads(false);
    return outs;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "gelu8";
    check_waits(who);
    no_second_order(who);
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Mat m = matrix(grads[0], who, "gradient");
    c10::cuda::CUDAGuard guard(grads[0].device());
    const Tensor dx = at::empty(grads[0].sizes(), grads[0].options());
    if (m.n > 0) {
      train::GeluBwd a{};
      a.dy = m.rows;
      a.q = q_ptr(saved[0]);
      a.scale = s_ptr(saved[1]);
      a.dx = dx.data_ptr();
      a.rows = m.n;
      a.cols = m.cols;
      a.tanh_form = kTanh;
      C10_CUDA_CHECK(train::gelu8_backward(a, stream_of(dx)));
    }
    out[0] = dx;
    return out;
  }
};

variable_list gelu8(const Tensor& x, bool tanh_form, bool pack) {
  return tanh_form ? Gelu8<true>::apply(x, pack, graph(x)) : Gelu8<false>::apply(x, pack, graph(x));
}

// --- linear ----------------------------------------------------------------------

// Coordinates of the tiles' copies are 32-bit.
void check_extent(std::int64_t rows, std::int64_t cols, std::int64_t outs, const char* who) {
  constexpr std::int64_t most = (1ll << 31) - 1024;
  TORCH_CHECK(rows <= most && cols <= most && outs <= most, who, ": at most ", most,
              " rows, columns and outputs, got ", rows, ", ", cols, " and ", outs);
}

std::tuple<Tensor, Tensor> weight_grad8(const Tensor& dy, const Tensor& q, const Tensor& scale, int64_t cols,
                                        const optional<Tensor>& weight, const optional<Tensor>& bias,
                                        optional<at::ScalarType> db_out, at::ScalarType out) {
  const char* who = "weight_grad8";
  check_waits(who);
  check_dtype(out, who, "out_dtype");
  const Mat m = matrix(dy, who, "dy");
  same_device(dy, q, who, "the 8-bit form");
  check_held(q, scale, m.n, cols, who);
  check_extent(m.n, cols, m.cols, who);
  c10::cuda::CUDAGuard guard(dy.device());
  Tensor w = defined_or(weight), b = defined_or(bias);
  if (w.defined()) w = column_vector(w, dy, cols, who, "weight");
  if (b.defined()) b = column_vector(b, dy, cols, who, "bias");
  TORCH_CHECK(!b.defined() || (w.defined() && w.scalar_type() == b.scalar_type()), who,
              ": a bias comes with a weight of its dtype");
  const Tensor dw = at::empty({m.cols, cols}, dy.options().dtype(out));
  const Tensor db = db_out.has_value() ? at::empty({m.cols}, dy.options().dtype(*db_out)) : Tensor();
  train::Wgrad8 a{};
  a.dy = m.rows;
  a.q = q_ptr(q);
  a.scale = s_ptr(scale);
  a.w = ptr(w);
  a.b = ptr(b);
  a.wt = w.defined() ? type_of(w, who, "weight") : train::Type::f32;
  a.dw = dw.data_ptr();
  a.db = out_ptr(db);
  a.dwt = type_of(dw, who, "out_dtype");
  a.dbt = db.defined() ? type_of(db, who, "bias") : a.dwt;
  a.rows = m.n;
  a.cols = cols;
  a.outs = m.cols;
  if (m.n == 0) {
    dw.zero_();
    if (db.defined()) db.zero_();
  } else {
    const Tensor work = at::empty({train::wgrad8_work(a)}, dy.options().dtype(at::kByte));
    a.work = work.data_ptr();
    C10_CUDA_CHECK(train::wgrad8(a, stream_of(dy)));
  }
  return {dw, db};
}

struct Linear8 : torch::autograd::Function<Linear8> {
  // q, scale: the 8-bit form of x, or of h where x = h * nw + nb
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                        const optional<Tensor>& q, const optional<Tensor>& scale, const optional<Tensor>& nw,
                        const optional<Tensor>& nb, bool keep) {
    const char* who = "linear8";
    check_waits(who);
    const Mat m = matrix(x, who, "x");
    c10::cuda::CUDAGuard guard(x.device());
    same_device(x, weight, who, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == m.cols, who, ": weight must have shape [outputs, ", m.cols,
                "], got ", weight.sizes());
    check_dtype(weight.scalar_type(), who, "weight");
    if (keep) check_extent(m.n, m.cols, weight.size(0), who);
    if (bias.has_value()) {
      same_device(x, *bias, who, "bias");
      TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), who, ": bias must have shape [",
                  weight.size(0), "], got ", bias->sizes());
      check_dtype(bias->scalar_type(), who, "bias");
    }
    const Tensor w = weight.to(x.scalar_type());
    const Tensor y = at::linear(x, w, bias.has_value() ? optional<Tensor>(bias->to(x.scalar_type())) : bias);
    Held h;
    if (keep) {
      if (q.has_value()) {
        TORCH_CHECK(scale.has_value(), who, ": an 8-bit form has scales");
        h = {*q, *scale};
        check_held(h.q, h.scale, m.n, m.cols, who);
        same_device(x, h.q, who, "the 8-bit form");
      } else {
        const auto p = pack8(x);
        h = {std::get<0>(p), std::get<1>(p)};
      }
    }
    ctx->save_for_backward({h.q, h.scale, w, defined_or(nw), defined_or(nb)});
    ctx->saved_data["wt"] = static_cast<int64_t>(weight.scalar_type());
    ctx->saved_data["bt"] = bias.has_value() ? static_cast<int64_t>(bias->scalar_type()) : int64_t{-1};
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_waits("linear8");
    no_second_order("linear8");
    variable_list out(8);
    const Tensor& dy = grads[0];
    const auto saved = ctx->get_saved_variables();
    const auto wt = static_cast<at::ScalarType>(ctx->saved_data["wt"].toInt());
    const int64_t bt = ctx->saved_data["bt"].toInt();
    const bool need_b = bt >= 0 && ctx->needs_input_grad(2);
    c10::cuda::CUDAGuard guard(dy.device());
    if (ctx->needs_input_grad(0)) out[0] = at::matmul(dy, saved[2]);
    if (ctx->needs_input_grad(1)) {
      const auto opt = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); };
      const auto g = weight_grad8(dy, saved[0], saved[1], saved[2].size(1), opt(saved[3]), opt(saved[4]),
                                  need_b ? optional<at::ScalarType>(static_cast<at::ScalarType>(bt)) : c10::nullopt,
                                  wt);
      out[1] = std::get<0>(g);
      if (need_b) out[2] = std::get<1>(g);
    } else if (need_b) {
      out[2] = dy.reshape({-1, dy.size(-1)}).sum(0, false, static_cast<at::ScalarType>(bt));
    }
    return out;
  }
};

Tensor linear8(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& q,
               const optional<Tensor>& scale, const optional<Tensor>& nw, const optional<Tensor>& nb) {
  return Linear8::apply(x, weight, bias, q, scale, nw, nb, graph(weight));
}

// --- cross entropy -----------------------------------------------------------------

train::Xent xent_args(const Mat& m, const Tensor& target, int64_t ignore, int64_t reduction, const Tensor& stats,
                      const Tensor& work) {
  train::Xent a{};
  a.x = m.rows;
  a.target = target.data_ptr<int64_t>();
  a.ignore = ignore;
  a.reduction = static_cast<int>(reduction);
  a.stats = stats.data_ptr<float>();
  a.work = work.data_ptr<float>();
  a.rows = m.n;
  a.cols = m.cols;
  return a;
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& target, int64_t ignore,
                        int64_t reduction, bool train) {
    const char* who = "cross_entropy";
    check_waits(who);
    const Mat m = matrix(logits, who, "logits");
    same_device(logits, target, who, "targets");
    TORCH_CHECK(target.scalar_type() == at::kLong, who, ": targets must be int64, got ", target.scalar_type());
    TORCH_CHECK(target.sizes() == logits.sizes().slice(0, logits.dim() - 1), who, ": targets must have shape ",
                logits.sizes().slice(0, logits.dim() - 1), ", got ", target.sizes());
    c10::cuda::CUDAGuard guard(logits.device());
    const Tensor t = target.contiguous();
    const auto f32 = logits.options().dtype(at::kFloat);
    const Tensor loss = reduction == 0 ? at::empty(target.sizes(), f32) : at::empty({}, f32);
    const Tensor stats = at::empty({2, m.n}, f32), work = at::empty({train::xent_work(m.n)}, f32);
    const bool now = train && reduction != 0;
    const Tensor dx = now ? at::empty(logits.sizes(), logits.options()) : Tensor();
    train::Xent a = xent_args(m, t, ignore, reduction, stats, work);
    a.loss = loss.data_ptr<float>();
    a.dx = out_ptr(dx);
    C10_CUDA_CHECK(train::xent_forward(a, stream_of(logits)));
    if (train) {
      ctx->save_for_backward({m.t, t, stats, work});  // a copy that was made serves both passes
      // the gradient for an upstream gradient of one, handed out by the first backward pass
      if (now) ctx->saved_data["unit"] = dx;
      ctx->saved_data["ignore"] = ignore;
      ctx->saved_data["reduction"] = reduction;
    }
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "cross_entropy";
    check_waits(who);
    no_second_order(who);
    const auto saved = ctx->get_saved_variables();
    const int64_t reduction = ctx->saved_data["reduction"].toInt();
    const Mat m = matrix(saved[0], who, "logits");
    c10::cuda::CUDAGuard guard(saved[0].device());
    train::Xent a = xent_args(m, saved[1], ctx->saved_data["ignore"].toInt(), reduction, saved[2], saved[3]);
    const auto unit = ctx->saved_data.find("unit");
    const bool have = unit != ctx->saved_data.end();
    // handed out once: a second pass over a kept graph fills a tensor of its own
    const Tensor dx = have ? unit->second.toTensor() : at::empty(saved[0].sizes(), saved[0].options());
    if (have) ctx->saved_data.erase(unit);
    a.dx = dx.data_ptr();
    const Tensor g = grads[0].to(at::kFloat).contiguous();
    if (m.n > 0) C10_CUDA_CHECK(train::xent_backward(a, g.data_ptr<float>(), have, stream_of(dx)));
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor cross_entropy(const Tensor& logits, const Tensor& target, int64_t ignore, int64_t reduction) {
  return CrossEntropy::apply(logits, target, ignore, reduction, graph(logits));
}

at::ScalarType dtype_of(const py::object& o) { return torch::python::detail::py_object_to_dtype(o); }

}  // namespace

void bind_train(py::module& m) {
  m.def("layer_norm", [](const Tensor& x, const optional<Tensor>& residual, const Tensor& weight,
                         const optional<Tensor>& bias, double eps, const py::object& out, bool pack) {
    return layer_norm(x, residual, weight, bias, eps, dtype_of(out), pack);
  });
  m.def("pack8", &pack8);
  m.def("unpack8", [](const Tensor& q, const Tensor& scale, std::vector<int64_t> sizes, const py::object& dtype,
                      const optional<Tensor>& weight, const optional<Tensor>& bias) {
    return unpack8(q, scale, std::move(sizes), dtype_of(dtype), weight, bias);
  });
  m.def("gelu8", &gelu8);
  m.def("weight_grad8", [](const Tensor& dy, const Tensor& q, const Tensor& scale, int64_t cols,
                           const optional<Tensor>& weight, const optional<Tensor>& bias, bool need_db,
                           const py::object& out) {
    const at::ScalarType t = dtype_of(out);
    return weight_grad8(dy, q, scale, cols, weight, bias, need_db ? optional<at::ScalarType>(t) : c10::nullopt, t);
  });
  m.def("linear8", &linear8);
  m.def("cross_entropy", &cross_entropy);
}
