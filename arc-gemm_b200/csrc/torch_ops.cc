// torch_ops.cc — the linear and grouped operators as PyTorch sees them: argument checks, output
// and workspace tensors, the current stream, autograd. Host C++ over the C ABI (arc_b200.h).
//
// Why here and not in Python: for a small call the GPU is done in a few microseconds, and the
// Python form of the same steps took 13 us per forward call and 127 us per training step of a
// tiny layer (64 x 64), of which the launches themselves are 4 and 12.
//
// The library's functions come in by address (bind), so that the one the package has loaded, the
// probe build included, is the one that is called.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <optional>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "arc_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
namespace py = pybind11;

// ---------------------------------------------------------------------------------
// The C ABI by address, errors
// ---------------------------------------------------------------------------------
struct Api {
  decltype(&arc_last_error) last_error = nullptr;
  decltype(&arc_status_string) status_string = nullptr;
  decltype(&arc_linear_bf16) linear = nullptr;
  decltype(&arc_linear_backward_workspace_bytes) linear_backward_ws = nullptr;
  decltype(&arc_linear_backward) linear_backward = nullptr;
  decltype(&arc_grouped_matmul) grouped = nullptr;
  decltype(&arc_grouped_matmul_dx) grouped_dx = nullptr;
  decltype(&arc_grouped_matmul_dw) grouped_dw = nullptr;
  decltype(&arc_a8w4_grouped_workspace_bytes) a8w4_grouped_ws = nullptr;
  decltype(&arc_a8w4_grouped_gemm) a8w4_grouped = nullptr;
  decltype(&arc_group_rows_workspace_bytes) group_rows_ws = nullptr;
  decltype(&arc_group_rows) group_rows = nullptr;
};
Api g_api;

// A failed library call, turned into arc.ArcError where Python is entered again.
struct ArcFailure : std::runtime_error {
  ArcFailure(int s, const std::string& m) : std::runtime_error(m), status(s) {}
  int status;
};

void check(int status, const char* what) {
  if (status != ARC_OK) {
    throw ArcFailure(status, std::string(what) + ": " + g_api.status_string(status) + ": " + g_api.last_error());
  }
}

template <typename... Args>
[[noreturn]] void bad_value(const Args&... args) {
  throw py::value_error(c10::str(args...));
}
template <typename... Args>
[[noreturn]] void bad_type(const Args&... args) {
  throw py::type_error(c10::str(args...));
}

std::string shape_of(const Tensor& t) { return c10::str(t.sizes()); }

void expect_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda()) bad_value(name, " must be a CUDA tensor (there is no CPU path), got ", t.device().str());
}
void expect_device(const Tensor& t, const char* name, const at::Device& dev) {
  if (t.device() != dev) bad_value(name, " is on ", t.device().str(), ", expected ", dev.str());
}
void expect_dtype(const Tensor& t, const char* name, at::ScalarType dtype) {
  if (t.scalar_type() != dtype) bad_type(name, " must be ", dtype, ", got ", t.scalar_type());
}
void expect_dims(const Tensor& t, const char* name, int64_t dims) {
  if (t.dim() != dims) bad_value(name, " must be ", dims, "-D, got shape ", shape_of(t));
}
void expect_bf16(const Tensor& t, const char* name, int64_t dims) {
  expect_cuda(t, name);
  expect_dtype(t, name, at::kBFloat16);
  expect_dims(t, name, dims);
}
void expect_shape(const Tensor& t, const char* name, at::IntArrayRef shape) {
  if (t.sizes() != shape) bad_value(name, " must have shape ", c10::str(shape), ", got ", shape_of(t));
}
// One contiguous operand of the A8W4 product, or the offsets.
void expect(const Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef shape, const at::Device& dev) {
  expect_cuda(t, name);
  expect_device(t, name, dev);
  expect_dtype(t, name, dtype);
  expect_shape(t, name, shape);
  if (!t.is_contiguous()) bad_value(name, " must be contiguous");
}
int as_int(int64_t v, const char* name) {
  if (v > INT32_MAX) bad_value(name, " (", v, ") is too large");
  return static_cast<int>(v);
}

// ---------------------------------------------------------------------------------
// Layouts
// ---------------------------------------------------------------------------------
const uint16_t* u16(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
uint16_t* u16_mut(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }

// An empty bf16 tensor whose rows are 16-byte aligned (a view of padded storage).
Tensor padded(at::IntArrayRef shape, const at::TensorOptions& options) {
  std::vector<int64_t> wide(shape.begin(), shape.end());
  wide.back() = (wide.back() + 7) / 8 * 8;
  return at::empty(wide, options).narrow(-1, 0, shape.back());
}

// `t` [.., R, C] itself if TMA can read its rows, else a copy whose rows are 16-byte aligned.
Tensor product_rows(const Tensor& t) {
  const int64_t d = t.dim(), rows = t.size(d - 2), cols = t.size(d - 1), ld = t.stride(d - 2);
  bool fits = t.stride(d - 1) == 1 && ld >= cols && ld % 8 == 0 && aligned16(t);
  if (d == 3) fits = fits && t.stride(0) >= (rows - 1) * ld + cols && t.stride(0) % 8 == 0;
  if (fits) return t;
  Tensor out = padded(t.sizes(), t.options().requires_grad(false));
  return out.copy_(t.detach());
}

// Rows for the epilogue and the gradients: any leading dimension.
Tensor unit_rows(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}

// Their leading dimension (a single row may have any stride).
int64_t row_ld(const Tensor& t) { return t.size(0) == 1 ? std::max(t.stride(0), t.size(1)) : t.stride(0); }

void expect_out(const Tensor& out, int64_t rows, int64_t cols, const at::Device& dev) {
  expect_bf16(out, "out", 2);
  if (out.size(0) != rows || out.size(1) != cols || out.device() != dev || out.stride(1) != 1 ||
      (rows > 1 && out.stride(0) < cols)) {
    bad_value("out must be a row-major bf16 [", rows, ", ", cols, "] tensor on ", dev.str());
  }
}

// The bytes of a tensor, as runs of `width` bytes: `rows` of them `pitch` apart, `blocks` of those rows
// `step` apart (at most three dimensions, none of negative stride).
struct Runs {
  int64_t at = 0, width = 0, rows = 1, pitch = 0, blocks = 1, step = 0;
};

// The bytes from a tensor's first to behind its last one.
std::pair<int64_t, int64_t> span_of(const Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  const int64_t at = reinterpret_cast<intptr_t>(t.const_data_ptr());
  return {at, at + (last + 1) * static_cast<int64_t>(t.element_size())};
}

Runs runs_of(const Tensor& t) {
  const int64_t item = t.element_size();
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride in bytes, size; smallest stride first
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) > 1 && t.stride(d) > 0) dims.emplace_back(t.stride(d) * item, t.size(d));
  }
  std::sort(dims.begin(), dims.end());
  Runs r;
  r.at = reinterpret_cast<intptr_t>(t.const_data_ptr());
  r.width = item;
  size_t d = 0;
  for (; d < dims.size() && dims[d].first <= r.width; ++d) r.width += (dims[d].second - 1) * dims[d].first;
  if (dims.size() > d + 2) {  // no dimension without gaps: everything from the first byte to the last
    for (; d < dims.size(); ++d) r.width += (dims[d].second - 1) * dims[d].first;
  }
  if (d < dims.size()) r.pitch = dims[d].first, r.rows = dims[d].second, ++d;
  if (d < dims.size()) r.step = dims[d].first, r.blocks = dims[d].second;
  return r;
}

// Whether a run of [at, at + width) meets one of `rows` runs of `own` bytes from byte 0 on, `pitch`
// apart; the run itself may stand for `also` ones of the same pitch.
bool meets(int64_t at, int64_t width, int64_t also, int64_t own, int64_t rows, int64_t pitch) {
  // Rows i and j meet if at - own < (i - j) pitch < at + width.
  if (pitch == 0) return at < own && at + width > 0;
  const int64_t below = at - own;
  int64_t m = below >= 0 ? below / pitch + 1 : -((-below - 1) / pitch);  // the least multiple above `below`
  m = std::max(m, 1 - also);
  return m <= rows - 1 && m * pitch < at + width;
}

// Whether two tensors (`a` of two dimensions at most) share a byte. Decided by addresses and strides,
// exactly (but for operands of three dimensions that all have gaps): column slices of one buffer that
// lie side by side share none. One look for tensors of one pitch, else one per row of `b`.
bool share_bytes(const Tensor& ta, const Tensor& tb) {
  if (ta.numel() == 0 || tb.numel() == 0) return false;
  const auto sa = span_of(ta), sb = span_of(tb);
  if (sa.second <= sb.first || sb.second <= sa.first) return false;
  const Runs a = runs_of(ta), b = runs_of(tb);
  const bool together = a.rows == 1 || b.rows == 1 || a.pitch == b.pitch;
  const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
  for (int64_t k = 0; k < b.blocks; ++k) {
    for (int64_t j = 0; j < (together ? 1 : b.rows); ++j) {
      const int64_t at = b.at + k * b.step + j * b.pitch - a.at;
      if (meets(at, b.width, together ? b.rows : 1, a.width, a.rows, pitch)) return true;
    }
  }
  return false;
}

// The same elements in the same order.
bool same_view(const Tensor& a, const Tensor& b) {
  if (a.const_data_ptr() != b.const_data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d) {
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  }
  return true;
}

// An `out` that is about to be written: not a tensor whose gradient is recorded, not one of the
// operands that other blocks still read, and a new version for whoever has saved it.
void claim_out(const OptTensor& out, std::initializer_list<const Tensor*> operands) {
  if (!out) return;
  if (at::GradMode::is_enabled() && out->requires_grad()) bad_value("out must not require a gradient");
  for (const Tensor* t : operands) {
    if (share_bytes(*out, *t)) bad_value("out must not overlap an operand");
  }
  if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

// Forward-mode derivatives are not offered. A tangent must not be dropped unnoticed, whatever the grad
// mode: the result would pass for a constant.
bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... Ts>
void refuse_tangents(const Ts&... ts) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(ts) || ...)) {
    throw std::runtime_error("arc's operators have no forward-mode derivative, and an argument carries a tangent");
  }
}

// The gradients are not differentiable themselves: a second derivative raises, by dy or by the
// operands (grad mode is on in a backward pass only for create_graph).
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "the gradients of arc's operators cannot be differentiated again", static_cast<int64_t>(grads.size()));
  torch::autograd::variable_list tracked;
  for (auto& g : grads) tracked.push_back(g.defined() ? g.detach().requires_grad_() : g);
  return (*node)(std::move(tracked));
}

// ---------------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------------
void linear_call(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, const Tensor& out,
                 const Tensor& z, int act) {
  check(g_api.linear(u16(x), u16(w), bias ? u16(*bias) : nullptr, residual ? u16(*residual) : nullptr, u16_mut(out),
                     z.defined() ? u16_mut(z) : nullptr, x.size(0), w.size(0), x.size(1), x.stride(0), w.stride(0),
                     residual ? row_ld(*residual) : 0, row_ld(out), z.defined() ? z.stride(0) : 0, act,
                     stream_of(x)),
        "arc.linear");
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in,
                        const OptTensor& bias, const OptTensor& residual, int64_t act) {
    const c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = product_rows(x_in), w = product_rows(w_in);
    const int64_t m = x.size(0), n = w.size(0);
    Tensor out = at::empty({m, n}, x.options().requires_grad(false));
    Tensor z;
    if (m > 0) {
      if (act != ARC_ACT_NONE && (wants_grad(x_in) || wants_grad(w_in) || wants_grad(bias))) {
        z = padded({m, n}, x.options().requires_grad(false));
      }
      linear_call(x, w, bias ? OptTensor(bias->contiguous()) : bias, residual ? OptTensor(unit_rows(*residual)) : residual,
                  out, z, static_cast<int>(act));
    }
    // Only what a gradient will read: the rest may change or be freed.
    ctx->save_for_backward({wants_grad(w_in) ? x : Tensor(), wants_grad(x_in) ? w : Tensor(), z});
    ctx->saved_data["m"] = m;
    ctx->saved_data["n"] = n;
    ctx->saved_data["k"] = x.size(1);
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = wants_grad(bias);
    ctx->saved_data["residual"] = wants_grad(residual);
    ctx->saved_data["x"] = wants_grad(x_in);
    ctx->saved_data["w"] = wants_grad(w_in);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor x = saved[0], w = saved[1], z = saved[2];
    const Tensor& dy_in = grads[0];
    const bool need_x = ctx->saved_data["x"].toBool(), need_w = ctx->saved_data["w"].toBool(),
               need_bias = ctx->saved_data["bias"].toBool(), need_residual = ctx->saved_data["residual"].toBool();
    const int64_t m = ctx->saved_data["m"].toInt(), n = ctx->saved_data["n"].toInt(), k = ctx->saved_data["k"].toInt();
    torch::autograd::variable_list out(5);
    if (!dy_in.defined()) return out;
    if (!(need_x || need_w || need_bias)) {
      if (need_residual) out[3] = dy_in;
      return out;
    }
    const c10::cuda::CUDAGuard guard(dy_in.device());
    // Hooks on saved tensors may bring them back in a layout of their own.
    if (need_w) x = product_rows(x);
    if (need_x) w = product_rows(w);
    if (z.defined()) z = unit_rows(z);
    const Tensor dy = unit_rows(dy_in.detach());
    const auto options = dy.options();
    if (need_x) out[0] = at::empty({m, k}, options);
    if (need_w) out[1] = m > 0 ? at::empty({n, k}, options) : at::zeros({n, k}, options);
    if (need_bias) out[2] = m > 0 ? at::empty({n}, options) : at::zeros({n}, options);
    if (m > 0) {
      const bool need_dz = (need_x || need_w) && (z.defined() || row_ld(dy) % 8 != 0 || !aligned16(dy));
      size_t bytes = 0;
      check(g_api.linear_backward_ws(m, n, need_dz, need_bias, &bytes), "arc.linear backward");
      Tensor workspace;
      if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, options.dtype(at::kByte));
      check(g_api.linear_backward(u16(dy), need_w ? u16(x) : nullptr, need_x ? u16(w) : nullptr,
                                  z.defined() ? u16(z) : nullptr,
                                  need_x ? u16_mut(out[0]) : nullptr, need_w ? u16_mut(out[1]) : nullptr,
                                  need_bias ? u16_mut(out[2]) : nullptr, bytes > 0 ? workspace.data_ptr() : nullptr,
                                  bytes, m, n, k, row_ld(dy), need_w ? x.stride(0) : 0, need_x ? w.stride(0) : 0,
                                  z.defined() ? row_ld(z) : 0, k, k,
                                  static_cast<int>(ctx->saved_data["act"].toInt()), stream_of(dy)),
            "arc.linear backward");
    }
    out = once(std::move(out));
    if (need_residual) out[3] = dy_in;  // the identity, which can be differentiated again
    return out;
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t act,
              const OptTensor& out) {
  expect_bf16(x, "x", 2);
  expect_bf16(w, "w", 2);
  const int64_t m = x.size(0), n = w.size(0), k = x.size(1);
  if (k != w.size(1)) bad_value("Inner dimensions must match: ", k, " vs ", w.size(1));
  if (n == 0 || k == 0) bad_value("w must not be empty, got shape ", shape_of(w));
  as_int(m, "M"), as_int(n, "N"), as_int(k, "K");
  const at::Device dev = x.device();
  expect_device(w, "w", dev);
  if (bias) {
    if (bias->scalar_type() != at::kBFloat16 || bias->dim() != 1 || bias->size(0) != n) {
      bad_value("bias must be bfloat16 of shape [", n, "], got ", bias->scalar_type(), " ", shape_of(*bias));
    }
    expect_device(*bias, "bias", dev);
  }
  if (residual) {
    expect_bf16(*residual, "residual", 2);
    expect_shape(*residual, "residual", {m, n});
    expect_device(*residual, "residual", dev);
  }
  refuse_tangents(x, w, bias, residual, out);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(bias) || wants_grad(residual))) {
    if (out) bad_value("out cannot be given when an input requires a gradient");
    return LinearFunction::apply(x, w, bias, residual, act);
  }
  const c10::cuda::CUDAGuard guard(dev);
  if (out) expect_out(*out, m, n, dev);
  if (out && residual && !same_view(*out, *residual) && share_bytes(*out, *residual)) {
    bad_value("out must be residual itself or not overlap it");
  }
  claim_out(out, {&x, &w, bias ? &*bias : &w});
  const Tensor y = out ? *out : at::empty({m, n}, x.options().requires_grad(false));
  if (m > 0) {
    linear_call(product_rows(x), product_rows(w), bias ? OptTensor(bias->contiguous()) : bias,
                residual ? OptTensor(unit_rows(*residual)) : residual, y, Tensor(), static_cast<int>(act));
  }
  return y;
}

// ---------------------------------------------------------------------------------
// grouped_matmul
// ---------------------------------------------------------------------------------
constexpr int64_t kMaxGroups = 1024;

void expect_offsets(const Tensor& offsets, int64_t groups, const at::Device& dev) {
  if (groups < 1 || groups > kMaxGroups) {
    bad_value("between 1 and ", kMaxGroups, " groups are supported, got ", groups);
  }
  expect(offsets, "offsets", at::kInt, {groups + 1}, dev);
}

void grouped_call(const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& out, bool zero_others) {
  check(g_api.grouped(u16(x), u16(w), offsets.const_data_ptr<int32_t>(), u16_mut(out), x.size(0), w.size(0), w.size(1),
                      x.size(1), x.stride(0), w.stride(1), w.stride(0), row_ld(out),
                      zero_others ? ARC_GROUPED_ZERO_OTHERS : 0u, stream_of(x)),
        "arc.grouped_matmul");
}

struct GroupedFunction : torch::autograd::Function<GroupedFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in,
                        const Tensor& offsets) {
    const c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = product_rows(x_in), w = product_rows(w_in);
    Tensor out = at::empty({x.size(0), w.size(1)}, x.options().requires_grad(false));
    if (x.size(0) > 0) grouped_call(x, w, offsets, out, true);
    // Only what a gradient will read: the rest may change or be freed.
    ctx->save_for_backward({wants_grad(w_in) ? x : Tensor(), wants_grad(x_in) ? w : Tensor(), offsets});
    ctx->saved_data["x"] = wants_grad(x_in);
    ctx->saved_data["w"] = wants_grad(w_in);
    ctx->saved_data["t"] = x.size(0);
    ctx->saved_data["e"] = w.size(0);
    ctx->saved_data["n"] = w.size(1);
    ctx->saved_data["k"] = w.size(2);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor x = saved[0], w = saved[1];
    const Tensor offsets = saved[2].contiguous();
    const Tensor& dy_in = grads[0];
    const int64_t t = ctx->saved_data["t"].toInt(), e = ctx->saved_data["e"].toInt(), n = ctx->saved_data["n"].toInt(),
                  k = ctx->saved_data["k"].toInt();
    torch::autograd::variable_list out(3);
    if (!dy_in.defined()) return out;
    const c10::cuda::CUDAGuard guard(dy_in.device());
    const char* what = "arc.grouped_matmul backward";
    const auto options = dy_in.options().requires_grad(false);
    if (t == 0) {
      if (ctx->saved_data["x"].toBool()) out[0] = at::empty({0, k}, options);
      if (ctx->saved_data["w"].toBool()) out[1] = at::zeros({e, n, k}, options);
      return out;
    }
    // Hooks on saved tensors may bring them back in a layout of their own.
    if (ctx->saved_data["w"].toBool()) x = product_rows(x);
    if (ctx->saved_data["x"].toBool()) w = product_rows(w);
    const Tensor dy = product_rows(dy_in.detach());
    if (ctx->saved_data["x"].toBool()) {
      out[0] = at::empty({t, k}, options);
      check(g_api.grouped_dx(u16(dy), u16(w), offsets.const_data_ptr<int32_t>(), u16_mut(out[0]), t, e, n, k,
                             dy.stride(0), w.stride(1), w.stride(0), k, ARC_GROUPED_ZERO_OTHERS, stream_of(dy)),
            what);
    }
    if (ctx->saved_data["w"].toBool()) {
      out[1] = at::empty({e, n, k}, options);
      check(g_api.grouped_dw(u16(dy), u16(x), offsets.const_data_ptr<int32_t>(), u16_mut(out[1]), t, e, n, k,
                             dy.stride(0), x.stride(0), k, n * k, stream_of(dy)),
            what);
    }
    return once(std::move(out));
  }
};

Tensor grouped_matmul(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& out) {
  expect_bf16(x, "x", 2);
  expect_bf16(w, "w", 3);
  const at::Device dev = x.device();
  expect_device(w, "w", dev);
  const int64_t t = x.size(0), k = x.size(1), n = w.size(1);
  if (k != w.size(2)) bad_value("Inner dimensions must match: ", k, " vs ", w.size(2));
  if (n == 0 || k == 0) bad_value("w must not be empty, got shape ", shape_of(w));
  as_int(t, "T"), as_int(n, "N"), as_int(k, "K");
  expect_offsets(offsets, w.size(0), dev);
  refuse_tangents(x, w, out);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w))) {
    if (out) bad_value("out cannot be given when an input requires a gradient");
    return GroupedFunction::apply(x, w, offsets);
  }
  const c10::cuda::CUDAGuard guard(dev);
  if (out) expect_out(*out, t, n, dev);
  claim_out(out, {&x, &w, &offsets});
  const Tensor y = out ? *out : at::empty({t, n}, x.options().requires_grad(false));
  if (t > 0) grouped_call(product_rows(x), product_rows(w), offsets, y, !out);
  return y;
}

// ---------------------------------------------------------------------------------
// a8w4_grouped_matmul, group_rows
// ---------------------------------------------------------------------------------
constexpr int64_t kScaleGroup = 128;

Tensor a8w4_grouped_matmul(const Tensor& x, const Tensor& sa_in, const Tensor& wp, const Tensor& sb,
                           const Tensor& offsets, const OptTensor& out, bool prepacked) {
  expect_dims(x, "a[0]", 2);
  expect_dims(wp, "b[0]", 3);
  const int64_t t = x.size(0), k = x.size(1), e = wp.size(0), n = wp.size(1);
  if (k != 2 * wp.size(2)) bad_value("Inner dimensions must match: ", k, " vs 2*", wp.size(2));
  if (k == 0 || k % kScaleGroup != 0 || n == 0) {
    bad_value("K (", k, ") must be a positive multiple of ", kScaleGroup, " and N (", n, ") positive");
  }
  as_int(t, "T"), as_int(n, "N"), as_int(k, "K");
  const at::Device dev = x.device();
  const Tensor sa = sa_in.dim() == 2 && sa_in.size(1) == 1 ? sa_in.reshape({-1}) : sa_in;
  expect(x, "a[0]", at::kChar, {t, k}, dev);
  expect(sa, "a[1]", at::kFloat, {t}, dev);
  expect(wp, "b[0]", at::kByte, {e, n, k / 2}, dev);
  expect(sb, "b[1]", at::kBFloat16, {e, n, k / kScaleGroup}, dev);
  expect_offsets(offsets, e, dev);
  refuse_tangents(sa, sb, out);
  const c10::cuda::CUDAGuard guard(dev);
  if (out) expect(*out, "out", at::kBFloat16, {t, n}, dev);
  claim_out(out, {&x, &sa, &wp, &sb, &offsets});
  const Tensor y = out ? *out : at::empty({t, n}, x.options().dtype(at::kBFloat16));
  if (t == 0) return y;
  size_t bytes = 0;
  check(g_api.a8w4_grouped_ws(t, e, k, &bytes), "arc.a8w4_grouped_matmul");
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, x.options());
  const unsigned flags = (prepacked ? ARC_A8W4_PREPACKED : 0u) | (out ? 0u : ARC_GROUPED_ZERO_OTHERS);
  check(g_api.a8w4_grouped(x.const_data_ptr<int8_t>(), sa.const_data_ptr<float>(), wp.const_data_ptr<uint8_t>(),
                           u16(sb), offsets.const_data_ptr<int32_t>(), u16_mut(y),
                           bytes > 0 ? workspace.data_ptr() : nullptr, bytes, t, e, n, k,
                           static_cast<int>(kScaleGroup), flags, stream_of(x)),
        "arc.a8w4_grouped_matmul");
  return y;
}

std::tuple<Tensor, Tensor, Tensor> group_rows(const Tensor& ids_in, int64_t groups) {
  expect_cuda(ids_in, "ids");
  if (ids_in.scalar_type() != at::kInt && ids_in.scalar_type() != at::kLong) {
    bad_type("ids must be int32 or int64, got ", ids_in.scalar_type());
  }
  if (ids_in.dim() != 1 && ids_in.dim() != 2) bad_value("ids must be [T] or [T, top], got shape ", shape_of(ids_in));
  if (groups < 1 || groups > kMaxGroups) {
    bad_value("between 1 and ", kMaxGroups, " groups are supported, got ", groups);
  }
  const Tensor ids = ids_in.contiguous();
  const int slots = as_int(ids.numel(), "the number of ids");
  const c10::cuda::CUDAGuard guard(ids.device());
  const auto options = ids.options().dtype(at::kInt);
  Tensor offsets = slots > 0 ? at::empty({groups + 1}, options) : at::zeros({groups + 1}, options);
  Tensor rows = at::empty({slots}, options), positions = at::empty(ids.sizes(), options);
  if (slots > 0) {
    size_t bytes = 0;
    check(g_api.group_rows_ws(slots, groups, &bytes), "arc.group_rows");
    Tensor workspace;
    if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, ids.options().dtype(at::kByte));
    check(g_api.group_rows(ids.const_data_ptr(), static_cast<int>(ids.element_size()), offsets.data_ptr<int32_t>(),
                           rows.data_ptr<int32_t>(), positions.data_ptr<int32_t>(),
                           bytes > 0 ? workspace.data_ptr() : nullptr, bytes, slots,
                           ids.dim() == 2 ? static_cast<int>(ids.size(1)) : 1, groups, stream_of(ids)),
          "arc.group_rows");
  }
  return {offsets, rows, positions};
}

// ---------------------------------------------------------------------------------
// Module
// ---------------------------------------------------------------------------------
PyObject* g_arc_error = nullptr;  // arc.ArcError, one reference for the life of the process

void bind(const std::unordered_map<std::string, uintptr_t>& addresses, py::object arc_error) {
  const auto set = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(addresses.at(name));
  };
  set(g_api.last_error, "arc_last_error");
  set(g_api.status_string, "arc_status_string");
  set(g_api.linear, "arc_linear_bf16");
  set(g_api.linear_backward_ws, "arc_linear_backward_workspace_bytes");
  set(g_api.linear_backward, "arc_linear_backward");
  set(g_api.grouped, "arc_grouped_matmul");
  set(g_api.grouped_dx, "arc_grouped_matmul_dx");
  set(g_api.grouped_dw, "arc_grouped_matmul_dw");
  set(g_api.a8w4_grouped_ws, "arc_a8w4_grouped_workspace_bytes");
  set(g_api.a8w4_grouped, "arc_a8w4_grouped_gemm");
  set(g_api.group_rows_ws, "arc_group_rows_workspace_bytes");
  set(g_api.group_rows, "arc_group_rows");
  g_arc_error = arc_error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const ArcFailure& e) {
      const py::object error = py::handle(g_arc_error)(e.status, e.what());
      PyErr_SetObject(g_arc_error, error.ptr());
    }
  });
  m.def("bind", &bind);
  m.def("linear", &linear);
  m.def("grouped_matmul", &grouped_matmul);
  m.def("a8w4_grouped_matmul", &a8w4_grouped_matmul);
  m.def("group_rows", &group_rows);
}
