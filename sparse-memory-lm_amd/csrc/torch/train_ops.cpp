// The dense operators of a training step as autograd nodes (smlm_hip.kernels.linear_cross_entropy, gated_ffn and
// add_rmsnorm_train): argument checks, outputs and workspaces from torch's allocator, and the C entry points of
// include/smlm_pkm.h on torch's current stream of the inputs' device.
//
// In C++ because a backward runs on a thread of autograd's own, often far from the caller's core, where a node written in
// Python takes 60 to 90 us before its kernels: forward and gradient of a norm took 112 us there, of an FFN block of 48
// tokens 146, against 40 us for a node that does nothing.
//
// A backward that is itself recorded (create_graph) runs as PyTorch ops, so that it can be differentiated again.
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "smlm_pkm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxRowStride = 1 << 21;   // elements (csrc/lm_mm.h)
constexpr int64_t kNormMaxCols = 16384;      // csrc/lm_rmsnorm.hip

int64_t ceil8(int64_t n) { return (n + 7) / 8 * 8; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int dtype_of(at::ScalarType t) { return t == at::kFloat ? SMLM_F32 : SMLM_BF16; }
bool is_float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

void check(int rc, const char *what) {
  TORCH_CHECK(rc == SMLM_OK, what, " failed with status ", rc, ": ", smlm_pkm_last_error());
}

// t with its values in memory as they are (a view may hold a sign that is yet to be applied).
Tensor plain(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void check_device(const char *name, const Tensor &first, std::initializer_list<const Tensor *> others) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be traced: a trace would hold its outputs as they were");
  TORCH_CHECK_VALUE(first.is_cuda(), name, ": all tensors must be on a HIP (cuda) device, got ", first.device());
  for (const Tensor *t : others)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == first.device(), name, ": all tensors must be on one device, got ",
                      first.device(), " and ", t->device());
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor workspace(const Tensor &like, int64_t bytes) { return at::empty({bytes}, like.options().dtype(at::kByte)); }

// t, `blocks` groups of rows, with zeros behind each group's rows and behind the columns.  (Fill and copy, as constant_pad_nd
// does it, are two launches: forward and gradient of an FFN block of 48 x 65, hidden 130, took 85 us instead of 68.)
Tensor padded(const Tensor &t, int64_t blocks, int64_t rows, int64_t cols) {
  // (contiguous() would leave a single row its stride, which may be any)
  const Tensor s = t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.clone(at::MemoryFormat::Contiguous);
  const Tensor out = at::empty({blocks * rows, cols}, t.options());
  check(smlm_pad_rows(s.data_ptr(), s.stride(0), blocks, s.size(0) / blocks, s.size(1), out.data_ptr(), rows, cols, stream_of(t)),
        "smlm_pad_rows");
  return out;
}

// t (rows', cols') as the products read it: rows of 16-byte aligned 8-element pieces, zeros from rows' and cols' on up to
// rows and cols.  t itself where it is so already.
Tensor mm_rows(const Tensor &t, int64_t rows, int64_t cols) {
  if (t.size(0) != rows || t.size(1) != cols) return padded(t, 1, rows, cols);
  if (t.stride(1) != 1 || t.stride(0) % 8 || t.stride(0) < cols || t.stride(0) > kMaxRowStride ||
      (uintptr_t)t.data_ptr() % 16)
    return t.clone(at::MemoryFormat::Contiguous);
  return t;
}

Tensor narrowed(const Tensor &t, int64_t rows, int64_t cols) {
  return t.size(0) == rows && t.size(1) == cols ? t : t.narrow(0, 0, rows).narrow(1, 0, cols);
}

// What a backward gets back need not be what forward saved (a saved-tensor hook gives what it likes, and a leaf's .data can be
// replaced meanwhile): the kernels read only tensors of the type, device and sizes that they take them for.
void check_saved(const char *name, const Tensor &t, at::ScalarType type, at::Device device, at::IntArrayRef sizes) {
  TORCH_CHECK(t.defined() && t.scalar_type() == type && t.device() == device && t.sizes() == sizes && !t.is_neg(), name,
              ": a saved tensor came back changed, expected ", type, " ", sizes, " on ", device);
}

// Within it the ops of a recorded backward keep their fp32 where autocast is on.
struct NoAutocast {
  c10::impl::ExcludeDispatchKeyGuard guard{c10::autocast_dispatch_keyset};
};

// The inputs as a recorded backward differentiates them: aliases, so that the gradient of one is not also what reaches it by
// way of another that was computed from it (tied embeddings), which the graph around this node adds by itself.
variable_list aliases(const variable_list &inputs) {
  variable_list out;
  for (const Tensor &t : inputs) out.push_back(t.view_as(t));
  return out;
}

// The gradients of `y` with respect to the wanted inputs (aliases), recorded.
variable_list recorded(const Tensor &y, const Tensor &dy, const variable_list &inputs, const std::vector<bool> &wants) {
  variable_list asked;
  for (size_t i = 0; i < inputs.size(); ++i)
    if (wants[i]) asked.push_back(inputs[i]);
  auto got = torch::autograd::grad({y}, asked, {dy}, std::nullopt, /*create_graph=*/true, /*allow_unused=*/true);
  variable_list out(inputs.size());
  for (size_t i = 0, k = 0; i < inputs.size(); ++i)
    if (wants[i]) out[i] = got[k++];
  return out;
}

// ---- the loss ----------------------------------------------------------------------------------------------------------
struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Tensor &targets, int64_t ignore,
                        int64_t reduction) {
    const int64_t d = x.size(-1), V = weight.size(0), M = x.numel() / d, d8 = ceil8(d);
    const auto f32 = x.options().dtype(at::kFloat);
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    const bool none = reduction == SMLM_REDUCE_NONE;
    if (M == 0) {
      ctx->save_for_backward({x, weight, targets, Tensor(), Tensor(), Tensor(), Tensor()});
      if (none) return at::empty(targets.sizes(), f32);
      return at::full({}, reduction == SMLM_REDUCE_MEAN ? std::numeric_limits<float>::quiet_NaN() : 0.f, f32);
    }
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = x.reshape({M, d}), xr = mm_rows(x2, M, d8), wr = mm_rows(weight, V, d8), t = targets.reshape({M}).contiguous();
    Tensor loss = none ? at::empty(targets.sizes(), f32) : at::empty({}, f32);
    Tensor lse = at::empty({M}, f32), count = none ? Tensor() : at::empty({}, f32);
    const Tensor ws = workspace(x, smlm_linear_ce_workspace(M, V, d8, 0));
    check(smlm_linear_ce(xr.data_ptr(), xr.stride(0), wr.data_ptr(), wr.stride(0), t.data_ptr<int64_t>(), ignore,
                         (int)reduction, M, V, d8, loss.data_ptr<float>(), (float *)ptr(count), lse.data_ptr<float>(),
                         ws.data_ptr(), ws.numel(), stream_of(x)),
          "smlm_linear_ce");
    // copies that the kernels needed serve the gradient too
    ctx->save_for_backward({x, weight, targets, lse, count, xr.is_same(x2) ? Tensor() : xr,
                            wr.is_same(weight) ? Tensor() : wr});
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &targets = saved[2];
    const int64_t ignore = ctx->saved_data["ignore"].toInt(), reduction = ctx->saved_data["reduction"].toInt();
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), none = reduction == SMLM_REDUCE_NONE;
    Tensor g = plain(grads[0]);
    const char *name = "linear_cross_entropy's gradient";
    const auto device = g.device();
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && weight.dim() == 2, name, ": a saved tensor came back changed");
    const int64_t d = x.size(-1), V = weight.size(0), M = x.numel() / d, d8 = ceil8(d);
    check_saved(name, x, at::kBFloat16, device, x.sizes());
    check_saved(name, weight, at::kBFloat16, device, {V, d});
    check_saved(name, targets, at::kLong, device, x.sizes().slice(0, x.dim() - 1));
    TORCH_CHECK(V > 0 && (!none || g.sizes() == targets.sizes()), name, ": a saved tensor came back changed");
    if (M > 0) {
      check_saved(name, saved[3], at::kFloat, device, {M});
      if (reduction == SMLM_REDUCE_MEAN) check_saved(name, saved[4], at::kFloat, device, {});
      if (saved[5].defined()) check_saved(name, saved[5], at::kBFloat16, device, {M, d8});
      if (saved[6].defined()) check_saved(name, saved[6], at::kBFloat16, device, {V, d8});
    }
    if (at::GradMode::is_enabled()) {
      const NoAutocast fp32;
      // an index outside the vocabulary, which the loss would stop the device for: any other, and NaN
      const Tensor t = targets.reshape({M}), bad = t.ne(ignore).logical_and(t.lt(0).logical_or(t.ge(V)));
      const Tensor one = at::ones({}, x.options().dtype(at::kFloat));
      const Tensor poison = at::where(bad, one * std::numeric_limits<float>::quiet_NaN(), one).unsqueeze(1);
      const auto in = aliases({x, weight});
      const Tensor logits = at::matmul(in[0].reshape({M, d}).to(at::kFloat), in[1].to(at::kFloat).t()) * poison;
      const Tensor y = at::cross_entropy_loss(logits, t.masked_fill(bad, ignore == 0 && V > 1 ? 1 : 0), {}, reduction, ignore);
      const auto got = recorded(y, g.reshape(y.sizes()), in, {want_x, want_w});
      return {got[0], got[1], Tensor(), Tensor(), Tensor()};
    }
    if (M == 0) return {at::zeros_like(x), at::zeros_like(weight), Tensor(), Tensor(), Tensor()};
    const c10::DeviceGuard guard(x.device());
    const Tensor xr = mm_rows(saved[5].defined() ? saved[5] : x.reshape({M, d}), M, d8);
    const Tensor wr = mm_rows(saved[6].defined() ? saved[6] : weight, V, d8);
    const Tensor t = targets.reshape({M}).contiguous(), lse = saved[3].contiguous();
    g = g.reshape({-1}).contiguous();
    const Tensor dx = want_x ? at::empty({M, d8}, x.options()) : Tensor(), dw = want_w ? at::empty({V, d8}, x.options()) : Tensor();
    const Tensor ws = workspace(x, smlm_linear_ce_workspace(M, V, d8, 1));
    check(smlm_linear_ce_backward(g.data_ptr<float>(), reduction == SMLM_REDUCE_MEAN ? saved[4].data_ptr<float>() : nullptr,
                                  none, xr.data_ptr(), xr.stride(0), wr.data_ptr(), wr.stride(0),
                                  t.data_ptr<int64_t>(), ignore, lse.data_ptr<float>(), M, V, d8, ptr(dx), ptr(dw),
                                  ws.data_ptr(), ws.numel(), stream_of(x)),
          "smlm_linear_ce_backward");
    return {want_x ? narrowed(dx, M, d).view(x.sizes()) : Tensor(), want_w ? narrowed(dw, V, d) : Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

Tensor linear_cross_entropy(const Tensor &x, const Tensor &weight, const Tensor &targets, int64_t ignore,
                            const std::string &reduction) {
  check_device("linear_cross_entropy", x, {&weight, &targets});
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && weight.scalar_type() == at::kBFloat16,
                    "linear_cross_entropy: x and weight must be bf16, got ", x.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.numel() > 0,
                    "linear_cross_entropy: expected x (..., d) and weight (V, d), got ", x.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(targets.scalar_type() == at::kLong && targets.sizes() == x.sizes().slice(0, x.dim() - 1),
                    "linear_cross_entropy: targets must be int64 of the shape ", x.sizes().slice(0, x.dim() - 1), ", got ",
                    targets.scalar_type(), " ", targets.sizes());
  const int64_t how = reduction == "mean" ? SMLM_REDUCE_MEAN : reduction == "sum" ? SMLM_REDUCE_SUM
                      : reduction == "none" ? SMLM_REDUCE_NONE : -1;
  TORCH_CHECK_VALUE(how >= 0, "linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got '", reduction, "'");
  return LinearCrossEntropy::apply(plain(x), plain(weight), targets, ignore, how);
}

// ---- the feed-forward block --------------------------------------------------------------------------------------------
// w13 with halves that end on whole pieces.
Tensor halves(const Tensor &w13, int64_t h, int64_t h8, int64_t d8) {
  return h8 == h ? mm_rows(w13, 2 * h, d8) : padded(w13, 2, h8, d8);
}

struct GatedFFN : torch::autograd::Function<GatedFFN> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w13, const Tensor &w2) {
    const int64_t d = x.size(-1), o = w2.size(0), h = w2.size(1), M = x.numel() / d, d8 = ceil8(d), h8 = ceil8(h), o8 = ceil8(o);
    auto shape = x.sizes().vec();
    shape.back() = o;
    if (M == 0) {
      ctx->save_for_backward({x, w13, w2, Tensor(), Tensor(), Tensor()});
      return at::empty(shape, x.options());
    }
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = x.reshape({M, d}), a = mm_rows(x2, M, d8), b = halves(w13, h, h8, d8), c = mm_rows(w2, o8, h8);
    const Tensor ws = workspace(x, smlm_gated_ffn_workspace(M, d8, h8, o8, 0));
    const Tensor y = at::empty({M, o8}, x.options());
    check(smlm_gated_ffn(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), c.data_ptr(), c.stride(0), M, d8, h8, o8,
                         y.data_ptr(), ws.data_ptr(), ws.numel(), stream_of(x)),
          "smlm_gated_ffn");
    ctx->save_for_backward({x, w13, w2, a.is_same(x2) ? Tensor() : a, b.is_same(w13) ? Tensor() : b, c.is_same(w2) ? Tensor() : c});
    return o8 == o ? y.view(shape) : y.narrow(1, 0, o).contiguous().view(shape);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w13 = saved[1], &w2 = saved[2], dy = plain(grads[0]);
    const bool want_x = ctx->needs_input_grad(0), want_w13 = ctx->needs_input_grad(1), want_w2 = ctx->needs_input_grad(2);
    const char *name = "gated_ffn's gradient";
    const auto device = dy.device();
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && w2.dim() == 2 && w2.numel() > 0, name, ": a saved tensor came back changed");
    const int64_t d = x.size(-1), o = w2.size(0), h = w2.size(1), M = x.numel() / d, d8 = ceil8(d), h8 = ceil8(h), o8 = ceil8(o);
    auto shape = x.sizes().vec();
    shape.back() = o;
    check_saved(name, x, at::kBFloat16, device, x.sizes());
    check_saved(name, w13, at::kBFloat16, device, {2 * h, d});
    check_saved(name, w2, at::kBFloat16, device, {o, h});
    TORCH_CHECK(dy.sizes() == at::IntArrayRef(shape), name, ": a saved tensor came back changed");
    if (saved[3].defined()) check_saved(name, saved[3], at::kBFloat16, device, {M, d8});
    if (saved[4].defined()) check_saved(name, saved[4], at::kBFloat16, device, {2 * h8, d8});
    if (saved[5].defined()) check_saved(name, saved[5], at::kBFloat16, device, {o8, h8});
    if (at::GradMode::is_enabled()) {
      const NoAutocast fp32;
      const auto in = aliases({x, w13, w2});
      const auto ab = at::matmul(in[0].to(at::kFloat), in[1].to(at::kFloat).t()).chunk(2, -1);
      const Tensor y = at::matmul(at::silu(ab[0]) * ab[1], in[2].to(at::kFloat).t()).to(dy.scalar_type());
      return recorded(y, dy, in, {want_x, want_w13, want_w2});
    }
    if (M == 0) return {at::zeros_like(x), at::zeros_like(w13), at::zeros_like(w2)};
    const c10::DeviceGuard guard(x.device());
    const Tensor a = mm_rows(saved[3].defined() ? saved[3] : x.reshape({M, d}), M, d8);
    const Tensor b = saved[4].defined() ? mm_rows(saved[4], 2 * h8, d8) : halves(w13, h, h8, d8);
    const Tensor c = mm_rows(saved[5].defined() ? saved[5] : w2, o8, h8), g = mm_rows(dy.reshape({M, o}), M, o8);
    const Tensor dx = want_x ? at::empty({M, d8}, x.options()) : Tensor();
    const Tensor dw13 = want_w13 ? at::empty({2 * h8, d8}, x.options()) : Tensor();
    const Tensor dw2 = want_w2 ? at::empty({o8, h8}, x.options()) : Tensor();
    const Tensor ws = workspace(x, smlm_gated_ffn_workspace(M, d8, h8, o8, 1));
    check(smlm_gated_ffn_backward(g.data_ptr(), g.stride(0), a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), c.data_ptr(),
                                  c.stride(0), M, d8, h8, o8, ptr(dx), ptr(dw13), ptr(dw2), ws.data_ptr(), ws.numel(),
                                  stream_of(x)),
          "smlm_gated_ffn_backward");
    Tensor r13 = dw13;
    if (want_w13 && h8 != h) r13 = dw13.view({2, h8, d8}).narrow(1, 0, h).narrow(2, 0, d).reshape({2 * h, d});
    else if (want_w13) r13 = narrowed(dw13, 2 * h, d);
    return {want_x ? narrowed(dx, M, d).view(x.sizes()) : Tensor(), r13, want_w2 ? narrowed(dw2, o, h) : Tensor()};
  }
};

Tensor gated_ffn(const Tensor &x, const Tensor &w13, const Tensor &w2) {
  check_device("gated_ffn", x, {&w13, &w2});
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && w13.scalar_type() == at::kBFloat16 && w2.scalar_type() == at::kBFloat16,
                    "gated_ffn: x, w13 and w2 must be bf16, got ", x.scalar_type(), ", ", w13.scalar_type(), " and ",
                    w2.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && w13.dim() == 2 && w2.dim() == 2 && w13.size(0) == 2 * w2.size(1) &&
                        w13.size(1) == x.size(-1) && w13.numel() > 0 && w2.numel() > 0,
                    "gated_ffn: expected x (..., d), w13 (2 * hidden, d) and w2 (n_out, hidden), got ", x.sizes(), ", ",
                    w13.sizes(), " and ", w2.sizes());
  return GatedFFN::apply(plain(x), plain(w13), plain(w2));
}

// ---- the norm ----------------------------------------------------------------------------------------------------------
struct AddRMSNorm : torch::autograd::Function<AddRMSNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &delta, const Tensor &weight,
                               double eps, at::ScalarType out_dtype) {
    ctx->set_materialize_grads(false);
    const int64_t C = x.size(-1), M = x.numel() / C;
    const bool add = delta.has_value();
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["delta"] = add ? (int64_t)delta->scalar_type() : -1;
    const c10::DeviceGuard guard(x.device());
    const Tensor a = x.contiguous(), w = weight.contiguous(), e = add ? delta->contiguous() : Tensor();
    const Tensor xs = add ? at::empty(x.sizes(), x.options()) : x;   // nothing to add: x itself, as an output of this node
    const Tensor h = at::empty(x.sizes(), x.options().dtype(out_dtype)), rstd = at::empty({M}, x.options().dtype(at::kFloat));
    if (M > 0)
      check(smlm_rmsnorm_train(a.data_ptr(), dtype_of(a.scalar_type()), ptr(e), dtype_of(add ? e.scalar_type() : at::kBFloat16),
                               w.data_ptr(), dtype_of(w.scalar_type()), (float)eps, M, C, add ? xs.data_ptr() : nullptr,
                               h.data_ptr(), dtype_of(out_dtype), rstd.data_ptr<float>(), stream_of(x)),
            "smlm_rmsnorm_train");
    ctx->save_for_backward({xs, weight, rstd});
    return {xs, h};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &xs = saved[0], &weight = saved[1], &rstd = saved[2], dxs = plain(grads[0]), dh = plain(grads[1]);
    const int64_t kind = ctx->saved_data["delta"].toInt();
    const bool add = kind >= 0;
    const auto delta_dtype = add ? (at::ScalarType)kind : xs.scalar_type();
    const bool want_x = ctx->needs_input_grad(0), want_delta = add && ctx->needs_input_grad(1),
               want_w = ctx->needs_input_grad(add ? 2 : 1);
    variable_list out(5);
    if (!dh.defined()) {
      if (!dxs.defined()) return out;
      if (want_x) out[0] = dxs;
      if (want_delta) out[1] = dxs.to(delta_dtype);
      if (want_w) out[2] = at::zeros_like(weight);
      return out;
    }
    const char *name = "add_rmsnorm_train's gradient";
    const auto device = dh.device();
    check_saved(name, xs, xs.scalar_type(), device, dh.sizes());
    const int64_t C = xs.size(-1), M = xs.numel() / C;
    check_saved(name, weight, weight.scalar_type(), device, {C});
    check_saved(name, rstd, at::kFloat, device, {M});
    TORCH_CHECK(is_float_type(xs.scalar_type()) && is_float_type(weight.scalar_type()), name, ": a saved tensor came back changed");
    if (dxs.defined()) check_saved(name, dxs, xs.scalar_type(), device, xs.sizes());
    if (at::GradMode::is_enabled()) {                            // in terms of xs, an output of this node
      const Tensor x = xs.to(at::kFloat), g = dh.to(at::kFloat);
      const Tensor r = (x.square().mean(-1, true) + ctx->saved_data["eps"].toDouble()).rsqrt(), hat = x * r;
      const Tensor gw = g * weight.to(at::kFloat);
      Tensor dx = (gw - hat * (gw * hat).mean(-1, true)) * r;
      if (dxs.defined()) dx = dx + dxs.to(at::kFloat);
      dx = dx.to(xs.scalar_type());
      if (want_x) out[0] = dx;
      if (want_delta) out[1] = dx.to(delta_dtype);
      if (want_w) out[2] = (g * hat).reshape({-1, xs.size(-1)}).sum(0).to(weight.scalar_type());
      return out;
    }
    const c10::DeviceGuard guard(device);
    const Tensor s = xs.contiguous(), w = weight.contiguous(), gh = dh.contiguous(), gx = dxs.defined() ? dxs.contiguous() : dxs;
    const Tensor r = rstd.contiguous();
    const Tensor dx = at::empty(xs.sizes(), xs.options());
    const bool cast = want_delta && delta_dtype != xs.scalar_type();
    const Tensor ddelta = cast ? at::empty(xs.sizes(), xs.options().dtype(delta_dtype)) : Tensor();
    Tensor dw, parts;
    if (want_w) {
      dw = M > 0 ? at::empty({C}, w.options()) : at::zeros({C}, w.options());
      parts = at::empty({smlm_rmsnorm_parts(M, C)}, w.options().dtype(at::kFloat));
    }
    if (M > 0)
      check(smlm_rmsnorm_train_backward(ptr(gx), gh.data_ptr(), dtype_of(gh.scalar_type()), s.data_ptr(),
                                        dtype_of(s.scalar_type()), w.data_ptr(), dtype_of(w.scalar_type()),
                                        r.data_ptr<float>(), M, C, dx.data_ptr(), ptr(ddelta), dtype_of(delta_dtype),
                                        ptr(dw), (float *)ptr(parts), stream_of(xs)),
            "smlm_rmsnorm_train_backward");
    if (want_x) out[0] = dx;
    if (want_delta) out[1] = cast ? ddelta : dx;
    if (want_w) out[2] = dw;
    return out;
  }
};

std::tuple<Tensor, Tensor> add_rmsnorm_train(const Tensor &x, const std::optional<Tensor> &delta, const Tensor &weight,
                                             std::optional<double> eps, std::optional<at::ScalarType> out_dtype) {
  const char *name = "add_rmsnorm_train";
  const Tensor none;
  check_device(name, x, {delta.has_value() ? &*delta : &none, &weight});
  const auto out = out_dtype.value_or(x.scalar_type());
  TORCH_CHECK_VALUE(is_float_type(x.scalar_type()) && is_float_type(weight.scalar_type()) && is_float_type(out), name,
                    ": x, the norm's weight and out_dtype must be fp32 or bf16, got ", x.scalar_type(), ", ",
                    weight.scalar_type(), " and ", out);
  TORCH_CHECK_VALUE(!delta.has_value() || (delta->sizes() == x.sizes() && (delta->scalar_type() == at::kBFloat16 ||
                                                                            delta->scalar_type() == x.scalar_type())),
                    name, ": delta must be ", x.sizes(), " in bf16 or x's type, got ",
                    delta.has_value() ? delta->sizes() : x.sizes(), " ", delta.has_value() ? delta->scalar_type() : out);
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1) && x.size(-1) > 0 &&
                        x.size(-1) <= kNormMaxCols,
                    name, ": x ", x.sizes(), " must end with the norm's ", weight.sizes(), ", at most ", kNormMaxCols, " columns");
  const double e = eps.value_or(0x1p-23);   // nn.RMSNorm's default: of fp32, which it computes in, whatever x's type
  TORCH_CHECK_VALUE(e >= 0, name, ": the norm's eps must not be negative, got ", e);
  const auto added = delta.has_value() ? std::optional<Tensor>(plain(*delta)) : delta;
  const auto got = AddRMSNorm::apply(plain(x), added, plain(weight), e, out);
  return {got[0], got[1]};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("gated_ffn", &gated_ffn);
  m.def("add_rmsnorm_train", &add_rmsnorm_train);
}
