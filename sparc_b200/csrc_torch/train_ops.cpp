// The gated linear recurrence, the layer norm and the gradient norm and clipping as PyTorch
// operators (torch.ops.sparc_b200.gated_scan, gated_scan_step, layer_norm, grad_clip): argument
// checks, output allocation and autograd around the C ABI, in C++ because these calls are short
// (a decode step, a norm) next to what a Python autograd function costs. No arithmetic here.
//
// Checks come in the order of the package's Python functions: shapes (ValueError), dtypes
// (TypeError), forward-mode derivatives (NotImplementedError), then the device (RuntimeError: there
// is no CPU path).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <atomic>
#include <cmath>
#include <optional>
#include <vector>

#include "sparc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SPARC_OK, what, " failed (", rc, "): ", sparc_last_error());
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return SPARC_DTYPE_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "sparc_b200 supports float32 and bfloat16 activations, got ",
                   t.scalar_type());
  return SPARC_DTYPE_BF16;
}

void require_device(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), "sparc_b200: ", name, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(t.device() == like.device(), "sparc_b200: ", name, " is on ", t.device(), ", not on ", like.device());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// t as a dense float32 array (itself where it is one).
Tensor f32(const Tensor& t) {
  if (t.scalar_type() == at::kFloat && t.is_contiguous() && !t.is_neg()) return t;
  return t.detach().to(at::kFloat).contiguous().resolve_neg();
}
const float* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
float* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// No operator here carries a forward-mode derivative on; a result without it would pass for one that is zero.
void refuse_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
                              what, " has no forward-mode derivative (its inputs may hold no tangent)");
}

// t as the kernels read it: any strides but adjacent values in the last dimension.
Tensor adjacent(const Tensor& t) {
  return (t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous()).resolve_neg();
}

// The gradients of a first-order backward; where a graph of them is asked for, it ends in an error.
variable_list once(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& g : grads)
    if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " is differentiable once: its gradients have no gradient", (int64_t)in.size());
  const variable_list out = (*error)(std::move(in));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// The library's status words, or'ed by kernels whose bounded waits ran out, of the devices that such kernels have
// been launched on.
constexpr int kDevices = 64;
std::atomic<unsigned*> g_status[kDevices];

unsigned* status_word(const Tensor& like) {  // (of the current device, like's)
  const int d = like.get_device();
  TORCH_CHECK(d < kDevices, "sparc_b200: device ", d, " is beyond the ", kDevices, " that are supported");
  unsigned* word = g_status[d].load(std::memory_order_acquire);
  if (word == nullptr) {
    check(sparc_gated_status_word(&word), "sparc_gated_status_word");
    g_status[d].store(word, std::memory_order_release);
  }
  return word;
}
std::vector<Tensor> wait_status() {
  std::vector<Tensor> out;
  for (int d = 0; d < kDevices; ++d)
    if (unsigned* word = g_status[d].load(std::memory_order_acquire))
      out.push_back(at::from_blob(word, {1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, d)));
  return out;
}

// ------------------------------------------------------------------ gated linear recurrence
void gated_check(const char* what, const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& nu, const OptTensor& state,
                 const OptTensor& pos, int64_t dim) {
  TORCH_CHECK_VALUE(x.dim() == dim && r.sizes() == x.sizes() && w.sizes() == x.sizes(), what,
                    " expects x, retention_gate and write_gate of one shape ",
                    dim == 3 ? "[batch, length, channels]" : "[batch, channels]");
  const int64_t B = x.size(0), D = x.size(-1);
  TORCH_CHECK_VALUE(nu.dim() == 1 && nu.size(0) == D, "nu_log must have shape [channels]");
  TORCH_CHECK_VALUE(!state || (state->dim() == 2 && state->size(0) == B && state->size(1) == D),
                    "state must have shape [batch, channels]");
  TORCH_CHECK_VALUE(!pos || pos->sizes() == x.sizes().slice(0, dim - 1), "segment_pos must have shape ",
                    x.sizes().slice(0, dim - 1));
  TORCH_CHECK_VALUE(x.numel() > 0, what, " expects at least one row, token and channel, got ", x.sizes());
  dtype_code(x);
  TORCH_CHECK_TYPE(r.scalar_type() == x.scalar_type() && w.scalar_type() == x.scalar_type(), what,
                   " expects x and its gates in one dtype, got ", x.scalar_type(), ", ", r.scalar_type(), ", ",
                   w.scalar_type());
  TORCH_CHECK_TYPE(nu.is_floating_point() && (!state || state->is_floating_point()),
                   "nu_log and state must be floating-point tensors");
  TORCH_CHECK_TYPE(!pos || (at::isIntegralType(pos->scalar_type(), true) && pos->element_size() <= 8),
                   "segment_pos must be an integer tensor, got ", pos ? pos->scalar_type() : at::kLong);
  for (const Tensor* t : {&x, &r, &w, &nu}) refuse_tangent(what, *t);
  if (state) refuse_tangent(what, *state);
  require_device(x, "x", x);
  require_device(r, "retention_gate", x);
  require_device(w, "write_gate", x);
  require_device(nu, "nu_log", x);
  if (state) require_device(*state, "state", x);
  if (pos) require_device(*pos, "segment_pos", x);
}

// The kernel call on checked tensors: y, last (where wanted), carry (where wanted).
struct GatedOut {
  Tensor y, last, carry;
};
GatedOut gated_forward(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& nu, const Tensor& h0, const Tensor& pos,
                       bool want_last, bool want_carry) {
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
  const auto fo = x.options().dtype(at::kFloat).requires_grad(false);
  GatedOut o;
  o.y = at::empty({B, T, D}, x.options().requires_grad(false));
  if (want_last) o.last = at::empty({B, D}, fo);
  if (want_carry) o.carry = at::empty({B, sparc_gated_carry_chunks(T), D}, fo);
  SparcGatedFwdArgs a = {};
  a.x = x.const_data_ptr();
  a.retention_gate = r.const_data_ptr();
  a.write_gate = w.const_data_ptr();
  a.nu_log = ptr(nu);
  a.h0 = ptr(h0);
  a.segment_pos = pos.defined() ? pos.const_data_ptr() : nullptr;
  a.segment_pos_bytes = pos.defined() ? (int)pos.element_size() : 0;
  a.y = o.y.mutable_data_ptr();
  a.last = out_ptr(o.last);
  a.carry = out_ptr(o.carry);
  a.x_batch_stride = x.stride(0);
  a.x_token_stride = x.stride(1);
  a.retention_batch_stride = r.stride(0);
  a.retention_token_stride = r.stride(1);
  a.write_batch_stride = w.stride(0);
  a.write_token_stride = w.stride(1);
  a.batch = B;
  a.length = T;
  a.channels = D;
  a.dtype = dtype_code(x);
  a.status = status_word(x);
  check(sparc_gated_scan_forward(&a, stream_of(x)), "sparc_gated_scan_forward");
  return o;
}

class GatedScan : public torch::autograd::Function<GatedScan> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& r_in, const Tensor& w_in,
                               const Tensor& nu_in, const OptTensor& state, const OptTensor& pos_in, bool want_last) {
    const Tensor x = adjacent(x_in), r = adjacent(r_in), w = adjacent(w_in), nu = f32(nu_in);
    const Tensor h0 = state ? f32(*state) : Tensor(), pos = pos_in ? pos_in->contiguous() : Tensor();
    GatedOut o = gated_forward(x, r, w, nu, h0, pos, want_last, true);
    ctx->save_for_backward({x, r, w, nu, pos, o.carry});
    ctx->saved_data["nu_dtype"] = (int64_t)nu_in.scalar_type();
    ctx->saved_data["state_dtype"] = state ? (int64_t)state->scalar_type() : (int64_t)-1;
    ctx->set_materialize_grads(false);
    return want_last ? variable_list{o.y, o.last} : variable_list{o.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) { return once(gradients(ctx, g), "gated scan"); }

 private:
  static variable_list gradients(AutogradContext* ctx, const variable_list& g) {
    const Tensor dy_in = g[0], dlast_in = g.size() > 1 ? g[1] : Tensor();
    if (!dy_in.defined() && !dlast_in.defined()) return variable_list(7);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &r = saved[1], &w = saved[2], &nu = saved[3], &pos = saved[4], &carry = saved[5];
    const c10::cuda::CUDAGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
    const auto xo = x.options().requires_grad(false), fo = xo.dtype(at::kFloat);
    const Tensor dy = dy_in.defined() ? adjacent(dy_in.to(x.scalar_type())) : at::zeros({B, T, D}, xo);
    const Tensor dlast = dlast_in.defined() ? f32(dlast_in) : Tensor();
    const Tensor dx = at::empty({B, T, D}, xo), dr = at::empty({B, T, D}, xo), dw = at::empty({B, T, D}, xo);
    const Tensor dnu = at::empty({D}, fo);
    const int64_t state_dtype = ctx->saved_data["state_dtype"].toInt();
    const Tensor dh0 = state_dtype >= 0 ? at::empty({B, D}, fo) : Tensor();
    const size_t bytes = sparc_gated_workspace_bytes(B, T, D);
    const Tensor ws = at::empty({(int64_t)bytes}, xo.dtype(at::kByte));
    SparcGatedBwdArgs a = {};
    a.x = x.const_data_ptr();
    a.retention_gate = r.const_data_ptr();
    a.write_gate = w.const_data_ptr();
    a.nu_log = ptr(nu);
    a.dy = dy.const_data_ptr();
    a.carry = ptr(carry);
    a.grad_last = ptr(dlast);
    a.segment_pos = pos.defined() ? pos.const_data_ptr() : nullptr;
    a.segment_pos_bytes = pos.defined() ? (int)pos.element_size() : 0;
    a.grad_x = dx.mutable_data_ptr();
    a.grad_retention_gate = dr.mutable_data_ptr();
    a.grad_write_gate = dw.mutable_data_ptr();
    a.grad_nu_log = out_ptr(dnu);
    a.grad_h0 = out_ptr(dh0);
    a.workspace = ws.mutable_data_ptr();
    a.workspace_bytes = bytes;
    a.x_batch_stride = x.stride(0);
    a.x_token_stride = x.stride(1);
    a.retention_batch_stride = r.stride(0);
    a.retention_token_stride = r.stride(1);
    a.write_batch_stride = w.stride(0);
    a.write_token_stride = w.stride(1);
    a.dy_batch_stride = dy.stride(0);
    a.dy_token_stride = dy.stride(1);
    a.batch = B;
    a.length = T;
    a.channels = D;
    a.dtype = dtype_code(x);
    a.status = status_word(x);
    check(sparc_gated_scan_backward(&a, stream_of(x)), "sparc_gated_scan_backward");
    const auto nu_dtype = (at::ScalarType)ctx->saved_data["nu_dtype"].toInt();
    return {dx, dr, dw, dnu.to(nu_dtype), dh0.defined() ? dh0.to((at::ScalarType)state_dtype) : Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> gated_scan(const Tensor& x, const Tensor& retention_gate, const Tensor& write_gate, const Tensor& nu_log,
                               const OptTensor& state, const OptTensor& segment_pos, bool return_last) {
  gated_check("gated scan", x, retention_gate, write_gate, nu_log, state, segment_pos, 3);
  const c10::cuda::CUDAGuard guard(x.device());
  if (c10::GradMode::is_enabled() &&
      (wants(x) || wants(retention_gate) || wants(write_gate) || wants(nu_log) || (state && wants(*state))))
    return GatedScan::apply(x, retention_gate, write_gate, nu_log, state, segment_pos, return_last);
  const at::NoGradGuard no_grad;  // no gradient can be asked for: no carries are kept
  GatedOut o = gated_forward(adjacent(x), adjacent(retention_gate), adjacent(write_gate), f32(nu_log),
                             state ? f32(*state) : Tensor(), segment_pos ? segment_pos->contiguous() : Tensor(), return_last,
                             false);
  return return_last ? std::vector<Tensor>{o.y, o.last} : std::vector<Tensor>{o.y};
}

std::tuple<Tensor, Tensor> gated_scan_step(const Tensor& x_in, const Tensor& r_in, const Tensor& w_in, const Tensor& nu_log,
                                           const Tensor& state, const OptTensor& segment_pos) {
  gated_check("gated scan step", x_in, r_in, w_in, nu_log, state, segment_pos, 2);
  const c10::cuda::CUDAGuard guard(x_in.device());
  const at::NoGradGuard no_grad;
  const Tensor x = adjacent(x_in.detach()), r = adjacent(r_in), w = adjacent(w_in), nu = f32(nu_log), h0 = f32(state);
  const Tensor pos = segment_pos ? segment_pos->contiguous() : Tensor();
  const Tensor y = at::empty(x.sizes(), x.options()), next = at::empty(x.sizes(), x.options().dtype(at::kFloat));
  SparcGatedStepArgs a = {};
  a.x = x.const_data_ptr();
  a.retention_gate = r.const_data_ptr();
  a.write_gate = w.const_data_ptr();
  a.nu_log = ptr(nu);
  a.state = ptr(h0);
  a.segment_pos = pos.defined() ? pos.const_data_ptr() : nullptr;
  a.segment_pos_bytes = pos.defined() ? (int)pos.element_size() : 0;
  a.y = y.mutable_data_ptr();
  a.new_state = out_ptr(next);
  a.x_stride = x.stride(0);
  a.retention_stride = r.stride(0);
  a.write_stride = w.stride(0);
  a.batch = x.size(0);
  a.channels = x.size(1);
  a.dtype = dtype_code(x);
  check(sparc_gated_step(&a, stream_of(x)), "sparc_gated_step");
  return {y, next};
}

// ------------------------------------------------------------------ layer norm
// t as [rows, width] with adjacent columns (a view where its strides allow one).
Tensor as_rows(const Tensor& t) { return adjacent(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

Tensor ln_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, at::IntArrayRef shape, Tensor* stats) {
  const int64_t R = x.size(0), W = x.size(1);
  const Tensor y = at::empty(shape, x.options().requires_grad(false));
  if (stats != nullptr) *stats = at::empty({2, R}, x.options().dtype(at::kFloat).requires_grad(false));
  if (R == 0) return y;
  SparcLayerNormFwdArgs a = {};
  a.x = x.const_data_ptr();
  a.weight = ptr(weight);
  a.bias = ptr(bias);
  a.y = y.mutable_data_ptr();
  if (stats != nullptr) {
    a.mean = out_ptr(*stats);
    a.rstd = a.mean + R;
  }
  a.x_row_stride = x.stride(0);
  a.rows = R;
  a.width = W;
  a.eps = (float)eps;
  a.dtype = dtype_code(x);
  check(sparc_layer_norm_forward(&a, stream_of(x)), "sparc_layer_norm_forward");
  return y;
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight, const OptTensor& bias, double eps) {
    const Tensor x = as_rows(x_in), w = f32(weight);
    Tensor stats;
    Tensor y = ln_forward(x, w, bias ? f32(*bias) : Tensor(), eps, x_in.sizes(), &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["weight_dtype"] = (int64_t)weight.scalar_type();
    ctx->saved_data["bias_dtype"] = bias ? (int64_t)bias->scalar_type() : (int64_t)-1;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) { return once(gradients(ctx, g), "layer norm"); }

 private:
  static variable_list gradients(AutogradContext* ctx, const variable_list& g) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2], &dy_in = g[0];
    const c10::cuda::CUDAGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const int64_t R = x.size(0), W = x.size(1), bias_dtype = ctx->saved_data["bias_dtype"].toInt();
    const bool need_w = ctx->needs_input_grad(1), need_b = bias_dtype >= 0 && ctx->needs_input_grad(2);
    const auto xo = x.options().requires_grad(false), fo = xo.dtype(at::kFloat);
    const Tensor dx = at::empty(dy_in.sizes(), xo);
    Tensor dw = need_w ? at::empty({W}, fo) : Tensor(), db = need_b ? at::empty({W}, fo) : Tensor();
    if (R > 0) {
      const Tensor dy = as_rows(dy_in.to(x.scalar_type()));
      const size_t bytes = need_w || need_b ? sparc_layer_norm_workspace_bytes(R, W) : 0;
      const Tensor ws = at::empty({(int64_t)bytes}, xo.dtype(at::kByte));
      SparcLayerNormBwdArgs a = {};
      a.x = x.const_data_ptr();
      a.dy = dy.const_data_ptr();
      a.weight = ptr(w);
      a.mean = ptr(stats);
      a.rstd = a.mean + R;
      a.dx = dx.mutable_data_ptr();
      a.grad_weight = out_ptr(dw);
      a.grad_bias = out_ptr(db);
      a.workspace = ws.mutable_data_ptr();
      a.workspace_bytes = bytes;
      a.x_row_stride = x.stride(0);
      a.dy_row_stride = dy.stride(0);
      a.rows = R;
      a.width = W;
      a.dtype = dtype_code(x);
      check(sparc_layer_norm_backward(&a, stream_of(x)), "sparc_layer_norm_backward");
    } else {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
    }
    if (dw.defined()) dw = dw.to((at::ScalarType)ctx->saved_data["weight_dtype"].toInt());
    if (db.defined()) db = db.to((at::ScalarType)bias_dtype);
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1),
                    "layer norm expects x [..., width] and weight [width]");
  TORCH_CHECK_VALUE(!bias || bias->sizes() == weight.sizes(), "layer norm expects bias [width]");
  TORCH_CHECK_VALUE(x.size(-1) > 0, "layer norm expects at least one column");
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative");
  dtype_code(x);
  TORCH_CHECK_TYPE(weight.is_floating_point() && (!bias || bias->is_floating_point()),
                   "layer norm expects floating-point parameters");
  for (const Tensor* t : {&x, &weight}) refuse_tangent("layer norm", *t);
  if (bias) refuse_tangent("layer norm", *bias);
  require_device(x, "x", x);
  require_device(weight, "weight", x);
  if (bias) require_device(*bias, "bias", x);
  const c10::cuda::CUDAGuard guard(x.device());
  if (c10::GradMode::is_enabled() && (wants(x) || wants(weight) || (bias && wants(*bias))))
    return LayerNorm::apply(x, weight, bias, eps);
  const at::NoGradGuard no_grad;
  return ln_forward(as_rows(x), f32(weight), bias ? f32(*bias) : Tensor(), eps, x.sizes(), nullptr);
}

// ------------------------------------------------------------------ gradient norm and clipping
void grads_check(const char* what, const std::vector<Tensor>& tensors) {
  for (const Tensor& t : tensors) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, " expects dense tensors, got ", t.layout());
    dtype_code(t);
    refuse_tangent(what, t);
  }
}
void grads_check_device(const char* what, const std::vector<Tensor>& tensors) {
  for (const Tensor& t : tensors) {
    TORCH_CHECK(t.is_cuda(), "sparc_b200: every gradient must be a CUDA tensor (there is no CPU path)");
    TORCH_CHECK(t.device() == tensors[0].device(), what, " expects tensors of one device, got ", tensors[0].device(), " and ",
                t.device());
  }
}

// A tensor's values as one dense array (any order of its dimensions), or a dense copy.
Tensor dense(const Tensor& t) { return (t.is_non_overlapping_and_dense() ? t : t.contiguous()).resolve_neg(); }

bool same_view(const Tensor& a, const Tensor& b) {
  return a.const_data_ptr() == b.const_data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides() && a.is_neg() == b.is_neg();
}
// Whether a and b share memory, as far as that shows without a search: strided ones where they are the same view.
bool overlaps(const Tensor& a, const Tensor& b) {
  const auto status = at::get_overlap_status(a, b);
  return status == at::MemOverlapStatus::TooHard ? same_view(a, b) : status != at::MemOverlapStatus::No;
}

// Outputs that are written through a copy, whose memory the kernels' own check does not see: not from several
// places of themselves, and apart from every other tensor. (An output may be its own gradient.)
void check_copied_outputs(const std::vector<Tensor>& grads, const std::vector<Tensor>& out) {
  const std::vector<Tensor>& target = out.empty() ? grads : out;
  for (size_t i = 0; i < target.size(); ++i) {
    const Tensor& t = target[i];
    if (t.numel() == 0 || (t.is_non_overlapping_and_dense() && !t.is_neg() && t.strides() == grads[i].strides())) continue;
    TORCH_CHECK(at::has_internal_overlap(t) != at::MemOverlap::Yes, "clip grads: an output overlaps itself (it is expanded)");
    for (size_t j = 0; j < target.size(); ++j)
      TORCH_CHECK((j == i || !overlaps(t, target[j])) && (out.empty() || !overlaps(t, grads[j]) || (j == i && same_view(t, grads[j]))),
                  "clip grads: an output overlaps another tensor");
  }
}

// The norm of `grads`, and with `clip` the gradients scaled into `out` (in place where it is empty).
Tensor grad_clip(const std::vector<Tensor>& grads, const std::vector<Tensor>& out, bool clip, double max_norm, double eps) {
  const char* what = clip ? "clip grads" : "grad norm";
  TORCH_CHECK_VALUE(!grads.empty(), what, " expects at least one tensor");
  TORCH_CHECK_VALUE(!clip || (max_norm >= 0.0 && eps >= 0.0), "max_norm and eps must not be negative");
  TORCH_CHECK_VALUE(out.empty() || out.size() == grads.size(), "clip grads expects one output for each gradient");
  for (size_t i = 0; i < out.size(); ++i)
    TORCH_CHECK_VALUE(out[i].sizes() == grads[i].sizes() && out[i].scalar_type() == grads[i].scalar_type(),
                      "clip grads expects out to match the gradients' shapes and dtypes");
  grads_check(what, grads);
  grads_check(what, out);
  if (clip) check_copied_outputs(grads, out);
  grads_check_device(what, grads);
  if (!out.empty()) {
    grads_check_device(what, out);
    TORCH_CHECK(out[0].device() == grads[0].device(), "clip grads expects out on the gradients' device");
  }
  const c10::cuda::CUDAGuard guard(grads[0].device());
  const at::NoGradGuard no_grad;
  const size_t n = grads.size();
  const std::vector<Tensor>& target = out.empty() ? grads : out;
  std::vector<Tensor> src(n), dst(n);
  std::vector<const void*> in_ptrs(n);
  std::vector<void*> out_ptrs(n);
  std::vector<long long> counts(n);
  std::vector<int> dtypes(n);
  for (size_t i = 0; i < n; ++i) {
    src[i] = dense(grads[i]);
    if (clip) {
      // in place: the gradient's own array or the copy of it; else an array in the source's order
      dst[i] = out.empty() ? src[i]
               : out[i].strides() == src[i].strides() && out[i].is_non_overlapping_and_dense() && !out[i].is_neg() ? out[i]
                                                                                               : at::empty_like(src[i]);
      out_ptrs[i] = dst[i].mutable_data_ptr();
    }
    in_ptrs[i] = src[i].const_data_ptr();
    counts[i] = src[i].numel();
    dtypes[i] = dtype_code(src[i]);
  }
  const auto fo = grads[0].options().dtype(at::kFloat).requires_grad(false);
  const Tensor norm = at::empty({}, fo);
  const size_t bytes = sparc_grad_clip_workspace_bytes((int)n);
  const Tensor ws = at::empty({(int64_t)bytes}, fo.dtype(at::kByte));
  SparcGradClipArgs a = {};
  a.grads = in_ptrs.data();
  a.out = clip ? out_ptrs.data() : nullptr;
  a.counts = counts.data();
  a.dtypes = dtypes.data();
  a.tensors = (int)n;
  a.max_norm = (float)max_norm;
  a.eps = (float)eps;
  a.norm = out_ptr(norm);
  a.workspace = ws.mutable_data_ptr();
  a.workspace_bytes = bytes;
  check(sparc_grad_clip(&a, stream_of(grads[0])), "sparc_grad_clip");
  if (clip) {
    for (size_t i = 0; i < n; ++i) {
      Tensor t = target[i];
      if (!t.is_same(dst[i])) t.copy_(dst[i]);
      else if (!t.is_inference()) torch::autograd::impl::bump_version(t);
    }
  }
  return norm;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sparc_b200, m) {
  m.def("gated_scan(Tensor x, Tensor retention_gate, Tensor write_gate, Tensor nu_log, Tensor? state, Tensor? segment_pos, "
        "bool return_last) -> Tensor[]", &gated_scan);
  m.def("gated_scan_step(Tensor x, Tensor retention_gate, Tensor write_gate, Tensor nu_log, Tensor state, "
        "Tensor? segment_pos) -> (Tensor, Tensor)", &gated_scan_step);
  m.def("layer_norm(Tensor x, Tensor weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("grad_clip(Tensor(a!)[] grads, Tensor(b!)[] out, bool clip, float max_norm, float eps) -> Tensor", &grad_clip);
  m.def("wait_status() -> Tensor[]", &wait_status);
}
