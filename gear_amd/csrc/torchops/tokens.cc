// The operators at both ends of a sequence model of tokens and between its blocks, as gear_amd.ops calls them.
#include <c10/core/DeviceGuard.h>

#include <cmath>

#include "host.hpp"

using namespace gear_hostops;

namespace {

[[noreturn]] void bad_value(const std::string &text) { throw py::value_error(text); }

std::string shape_text(at::IntArrayRef shape) {
  std::string text;
  for (const int64_t n : shape) text += (text.empty() ? "" : ", ") + std::to_string(n);
  return "[" + text + "]";
}

int element_type(const at::Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GEAR_HIP_F32;
    case at::kHalf: return GEAR_HIP_F16;
    case at::kBFloat16: return GEAR_HIP_BF16;
    default:
      throw py::type_error(std::string(name) + " must have dtype torch.float32, torch.float16 or torch.bfloat16, got " +
                           std::string(py::str(wrap(t).attr("dtype"))));
  }
}

const at::Tensor &on_gpu(const at::Tensor &t, const char *name) {
  if (!t.is_cuda()) bad_value(std::string(name) + " must live on the GPU");
  return t;
}
void same_device(const at::Tensor &t, const char *name, const at::Device &device) {
  on_gpu(t, name);
  if (t.device() != device) bad_value(std::string(name) + " must live on the device of the other arguments");
}

// [..., width]: rows of contiguous elements at one stride.
struct Matrix {
  at::Tensor t;
  int64_t rows = 1, width = 0, stride = 0;
  int dtype = 0;
  Matrix() = default;
  Matrix(py::handle h, const char *name) : t(any_tensor(h, name)) {
    dtype = element_type(t, name);
    on_gpu(t, name);
    init(name);
  }
  // of the type, the device and the shape of another
  Matrix(py::handle h, const char *name, const Matrix &like, const char *like_name, at::IntArrayRef shape) : t(any_tensor(h, name)) {
    dtype = element_type(t, name);
    if (dtype != like.dtype)
      throw py::type_error(std::string(name) + " must have the dtype of " + like_name + ", got " +
                           std::string(py::str(h.attr("dtype"))));
    same_device(t, name, like.t.device());
    if (t.sizes() != shape)
      bad_value(std::string(name) + " must have shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
    init(name);
  }
  at::IntArrayRef lead() const { return t.sizes().slice(0, t.dim() - 1); }
  void *ptr() const { return t.data_ptr(); }

 private:
  void init(const char *name) {
    if (t.dim() < 1) bad_value(std::string(name) + " must have at least one dimension");
    width = t.size(-1);
    if (width < 1) bad_value(std::string(name) + " must have at least one element a row");
    stride = width;
    bool fits = width == 1 || t.numel() == 0 || t.stride(-1) == 1, first = true;
    int64_t next = 0;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      rows *= t.size(i);
      if (t.size(i) == 1 || t.numel() == 0) continue;
      if (first)
        stride = t.stride(i);
      else
        fits = fits && t.stride(i) == next;
      next = t.stride(i) * t.size(i);
      first = false;
    }
    if (!fits)
      bad_value(std::string(name) + " must have contiguous elements in rows at one stride (call .contiguous())");
  }
};

struct Tokens {
  at::Tensor t;
  int wide = 0;
  Tokens() = default;
  Tokens(py::handle h, const char *name) : t(any_tensor(h, name)) { init(name); }
  Tokens(py::handle h, const char *name, const at::Device &device, at::IntArrayRef shape) : t(any_tensor(h, name)) {
    init(name);
    same_device(t, name, device);
    if (t.sizes() != shape)
      bad_value(std::string(name) + " must have shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
  }
  const void *ptr() const { return t.defined() ? t.data_ptr() : nullptr; }

 private:
  void init(const char *name) {
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
      throw py::type_error(std::string(name) + " must have dtype torch.int64 or torch.int32, got " +
                           std::string(py::str(wrap(t).attr("dtype"))));
    if (!t.is_contiguous()) bad_value(std::string(name) + " must be contiguous");
    on_gpu(t, name);
    wide = t.scalar_type() == at::kLong;
  }
};

// A float32 tensor of a given shape, or none.
at::Tensor floats(py::handle h, const char *name, const at::Device &device, at::IntArrayRef shape) {
  if (h.is_none()) return at::Tensor();
  const at::Tensor &t = need(h, at::kFloat, name);
  same_device(t, name, device);
  if (t.sizes() != shape)
    bad_value(std::string(name) + " must have shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
  return t;
}
float *float_ptr(const at::Tensor &t) { return t.defined() ? ptr<float>(t) : nullptr; }

at::Tensor make(at::IntArrayRef shape, at::ScalarType dtype, const at::Device &device) {
  py::gil_scoped_release nogil;
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(device));
}
std::vector<int64_t> with(at::IntArrayRef lead, int64_t last) {
  std::vector<int64_t> shape(lead.begin(), lead.end());
  shape.push_back(last);
  return shape;
}
py::object wrap_or_none(const at::Tensor &t) { return t.defined() ? wrap(t) : py::none(); }

float number(double x, const char *name) {
  if (!std::isfinite((float)x)) bad_value(std::string(name) + " must be a finite number of 32 bits");
  return (float)x;
}

// A call that is being captured gets scratch of its own, out of the graph's memory: graphs that were captured on one stream may
// be replayed on several.
Scratch scratch(py::handle ws, const char *tag, size_t bytes, const at::Device &device) {
  if (bytes == 0) return Scratch();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(static_cast<hipStream_t>(current_stream()), &status) != hipSuccess) {
    (void)hipGetLastError();  // (or the next launch would be taken for failed)
    status = hipStreamCaptureStatusNone;
  }
  if (status == hipStreamCaptureStatusNone) return Scratch(ws, tag, bytes, device);
  Scratch s;
  s.keep = empty((int64_t)std::max<size_t>(bytes, 256), at::kByte, device);
  s.ptr = s.keep.data_ptr(), s.bytes = (size_t)s.keep.numel();
  return s;
}

// ---- rows of a table by token --------------------------------------------------------------------
constexpr int64_t kMostTokens = ((int64_t)1 << 31) - 1;

py::object embed_tokens(py::handle tokens_, py::handle table_, double scale_) {
  const Tokens tokens(tokens_, "tokens");
  const at::Tensor &as_given = any_tensor(table_, "table");
  if (as_given.dim() != 2) bad_value("table must be [vocab, width]");
  const Matrix table(table_, "table");
  const at::Device device = table.t.device();
  same_device(tokens.t, "tokens", device);
  const float scale = number(scale_, "scale");
  const c10::DeviceGuard guard(device);
  const at::Tensor out = make(with(tokens.t.sizes(), table.width), table.t.scalar_type(), device);
  call("gear_hip_embed", Scratch(), gear_hip_embed, tokens.ptr(), tokens.wide, tokens.t.numel(), table.ptr(), table.stride,
       table.rows, table.width, table.dtype, scale, out.data_ptr(), current_stream());
  return wrap(out);
}

py::object embed_tokens_backward(py::handle dout_, py::handle tokens_, int64_t vocab, double scale_, py::handle ws) {
  const Matrix dout(dout_, "dout");
  const at::Device device = dout.t.device();
  const Tokens tokens(tokens_, "tokens", device, dout.lead());
  if (vocab < 0 || vocab >= kMostTokens) bad_value("vocab must be a number of tokens below 2^31 - 1");
  const float scale = number(scale_, "scale");
  const c10::DeviceGuard guard(device);
  const at::Tensor dtable = make({vocab, dout.width}, dout.t.scalar_type(), device);
  const Scratch s = scratch(ws, "embed_backward", gear_hip_embed_backward_workspace_bytes(dout.rows, dout.width), device);
  call("gear_hip_embed_backward", s, gear_hip_embed_backward, dout.ptr(), dout.stride, tokens.ptr(), tokens.wide, dout.rows, vocab,
       dout.width, dout.dtype, scale, dtable.data_ptr(), s.ptr, s.bytes, current_stream());
  return wrap(dtable);
}

// ---- layer norm ----------------------------------------------------------------------------------
struct LayerNorm {
  Matrix x;
  at::Tensor weight, bias;
  at::ScalarType weight_dtype = at::kFloat;
  gear_hip_layer_norm_desc d = {};

  LayerNorm(py::handle x_, const char *name, py::handle weight_, py::handle bias_, double eps) : x(x_, name) {
    if (x.width > 16384) bad_value(std::string(name) + " must have rows of at most 16384 elements, got " + std::to_string(x.width));
    one(weight_, "weight", weight);
    one(bias_, "bias", bias);
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
      throw py::type_error("weight and bias must have one dtype");
    if (!(eps >= 0) || !std::isfinite((float)eps)) bad_value("eps must be a number of at least 0");
    d.x = x.ptr(), d.x_stride = x.stride, d.rows = x.rows, d.width = x.width, d.dtype = x.dtype, d.eps = (float)eps;
    d.weight = weight.defined() ? weight.data_ptr() : nullptr;
    d.bias = bias.defined() ? bias.data_ptr() : nullptr;
    d.weight_f32 = weight_dtype == at::kFloat;
  }

 private:
  void one(py::handle h, const char *name, at::Tensor &keep) {
    if (h.is_none()) return;
    const at::Tensor &t = any_tensor(h, name);
    if (t.scalar_type() != at::kFloat && t.scalar_type() != x.t.scalar_type())
      throw py::type_error(std::string(name) + " must have dtype torch.float32 or that of the rows");
    need(h, t.scalar_type(), name);
    same_device(t, name, x.t.device());
    if (t.dim() != 1 || t.size(0) != x.width)
      bad_value(std::string(name) + " must have shape [" + std::to_string(x.width) + "], got " + shape_text(t.sizes()));
    keep = t;
    weight_dtype = t.scalar_type();
  }
};

py::object layer_norm(py::handle x, py::handle weight, py::handle bias, py::handle residual_, double eps) {
  LayerNorm n(x, "x", weight, bias, eps);
  const at::Device device = n.x.t.device();
  Matrix residual;
  if (!residual_.is_none()) {
    residual = Matrix(residual_, "residual", n.x, "x", n.x.t.sizes());
    n.d.residual = residual.ptr(), n.d.residual_stride = residual.stride;
  }
  const c10::DeviceGuard guard(device);
  const at::Tensor y = make(n.x.t.sizes(), n.x.t.scalar_type(), device);
  at::Tensor sum;
  if (residual.t.defined()) sum = make(n.x.t.sizes(), n.x.t.scalar_type(), device);
  call("gear_hip_layer_norm", Scratch(), gear_hip_layer_norm, &n.d, y.data_ptr(), sum.defined() ? sum.data_ptr() : nullptr,
       current_stream());
  if (!sum.defined()) return wrap(y);
  return py::make_tuple(wrap(y), wrap(sum));
}

py::object layer_norm_backward(py::handle dy_, py::handle x, py::handle weight, py::handle bias, py::handle dsum_, double eps,
                               py::handle ws) {
  LayerNorm n(x, "x", weight, bias, eps);
  const at::Device device = n.x.t.device();
  const Matrix dy(dy_, "dy", n.x, "x", n.x.t.sizes());
  Matrix dsum;
  if (!dsum_.is_none()) dsum = Matrix(dsum_, "dsum", n.x, "x", n.x.t.sizes());
  const c10::DeviceGuard guard(device);
  const at::Tensor dx = make(n.x.t.sizes(), n.x.t.scalar_type(), device);
  at::Tensor dweight, dbias;
  if (n.weight.defined()) dweight = make({n.x.width}, n.weight_dtype, device);
  if (n.bias.defined()) dbias = make({n.x.width}, n.weight_dtype, device);
  const Scratch s = n.weight.defined() || n.bias.defined()
                        ? scratch(ws, "layer_norm", gear_hip_layer_norm_backward_workspace_bytes(n.x.rows, n.x.width), device)
                        : Scratch();
  call("gear_hip_layer_norm_backward", s, gear_hip_layer_norm_backward, &n.d, dy.ptr(), dy.stride,
       dsum.t.defined() ? dsum.ptr() : nullptr, dsum.stride, dx.data_ptr(), dweight.defined() ? dweight.data_ptr() : nullptr,
       dbias.defined() ? dbias.data_ptr() : nullptr, s.ptr, s.bytes, current_stream());
  return py::make_tuple(wrap(dx), wrap_or_none(dweight), wrap_or_none(dbias));
}

// ---- logits --------------------------------------------------------------------------------------
struct Logits {
  Matrix x;
  gear_hip_logits_desc d = {};
  Logits(py::handle logits, double scale) : x(logits, "logits") {
    if (x.width > 1 << 20) bad_value("logits must have at most 2^20 tokens a row, got " + std::to_string(x.width));
    if (!((float)scale > 0) || !(scale < 1e30)) bad_value("scale must be a number above 0 (of 32 bits, below 1e30)");
    d.logits = x.ptr(), d.row_stride = x.stride, d.rows = x.rows, d.vocab = x.width, d.dtype = x.dtype, d.scale = (float)scale;
  }
  at::Device device() const { return x.t.device(); }
};

constexpr int64_t kMostTop = 64;

py::object token_log_probs(py::handle logits, py::handle tokens_, double scale, int64_t top, py::handle ws) {
  const Logits l(logits, scale);
  const at::Device device = l.device();
  const at::IntArrayRef lead = l.x.lead();
  Tokens tokens;
  if (!tokens_.is_none()) tokens = Tokens(tokens_, "tokens", device, lead);
  if (top < 0 || top > kMostTop || top > l.x.width) bad_value("top must be a number from 0 to 64, at most the tokens there are");
  const c10::DeviceGuard guard(device);
  at::Tensor log_probs, best, value;
  if (tokens.t.defined()) log_probs = make(lead, at::kFloat, device);
  const at::Tensor entropy = make(lead, at::kFloat, device), lse = make(lead, at::kFloat, device);
  if (top > 0) value = make(with(lead, top), at::kFloat, device), best = make(with(lead, top), at::kLong, device);
  const Scratch s = scratch(ws, "token_log_probs", gear_hip_token_log_probs_workspace_bytes(l.x.rows, l.x.width, top), device);
  call("gear_hip_token_log_probs", s, gear_hip_token_log_probs, &l.d, tokens.ptr(), tokens.wide, top, float_ptr(log_probs),
       ptr<float>(entropy), ptr<float>(lse), float_ptr(value), best.defined() ? ptr<int64_t>(best) : nullptr, s.ptr, s.bytes,
       current_stream());
  return py::make_tuple(wrap_or_none(log_probs), wrap(entropy), wrap(lse), wrap_or_none(value), wrap_or_none(best));
}

py::object token_log_probs_backward(py::handle dlog_probs_, py::handle dentropy_, py::handle logits, py::handle tokens_,
                                    py::handle lse_, py::handle entropy_, double scale) {
  const Logits l(logits, scale);
  const at::Device device = l.device();
  const at::IntArrayRef lead = l.x.lead();
  Tokens tokens;
  if (!tokens_.is_none()) tokens = Tokens(tokens_, "tokens", device, lead);
  const at::Tensor dlog_probs = floats(dlog_probs_, "dlog_probs", device, lead),
                   dentropy = floats(dentropy_, "dentropy", device, lead), lse = floats(lse_, "lse", device, lead),
                   entropy = floats(entropy_, "entropy", device, lead);
  if (!lse.defined()) bad_value("lse is needed");
  if (dlog_probs.defined() && !tokens.t.defined()) bad_value("dlog_probs needs the tokens that it belongs to");
  if (dentropy.defined() && !entropy.defined()) bad_value("dentropy needs the entropy");
  const c10::DeviceGuard guard(device);
  const at::Tensor dlogits = make(l.x.t.sizes(), l.x.t.scalar_type(), device);
  call("gear_hip_token_log_probs_backward", Scratch(), gear_hip_token_log_probs_backward, &l.d, float_ptr(dlog_probs),
       float_ptr(dentropy), tokens.ptr(), tokens.wide, ptr<float>(lse), float_ptr(entropy), dlogits.data_ptr(), current_stream());
  return wrap(dlogits);
}

struct Teacher {
  Tokens tokens;
  at::Tensor logits;
  int64_t count = 0;
  Teacher(const Logits &l, py::handle top_tokens, py::handle top_logits) {
    const at::Tensor &t = any_tensor(top_tokens, "top_tokens");
    count = t.dim() > 0 ? t.size(-1) : 0;
    if (count < 1 || count > kMostTop) bad_value("top_tokens must name 1 to 64 tokens a row");
    const std::vector<int64_t> shape = with(l.x.lead(), count);
    tokens = Tokens(top_tokens, "top_tokens", l.device(), shape);
    logits = floats(top_logits, "top_logits", l.device(), shape);
    if (!logits.defined()) bad_value("top_logits is needed");
  }
};

py::object distill(py::handle logits, py::handle top_tokens, py::handle top_logits, double scale, py::handle ws) {
  const Logits l(logits, scale);
  const Teacher q(l, top_tokens, top_logits);
  const at::Device device = l.device();
  const c10::DeviceGuard guard(device);
  const at::Tensor loss = make(l.x.lead(), at::kFloat, device), lse = make(l.x.lead(), at::kFloat, device);
  const Scratch s = scratch(ws, "distill", gear_hip_distill_workspace_bytes(l.x.rows, l.x.width), device);
  call("gear_hip_distill", s, gear_hip_distill, &l.d, q.tokens.ptr(), q.tokens.wide, ptr<float>(q.logits), q.count,
       ptr<float>(loss), ptr<float>(lse), s.ptr, s.bytes, current_stream());
  return py::make_tuple(wrap(loss), wrap(lse));
}

py::object distill_backward(py::handle dloss_, py::handle logits, py::handle top_tokens, py::handle top_logits, py::handle lse_,
                            double scale) {
  const Logits l(logits, scale);
  const Teacher q(l, top_tokens, top_logits);
  const at::Device device = l.device();
  const at::Tensor dloss = floats(dloss_, "dloss", device, l.x.lead()), lse = floats(lse_, "lse", device, l.x.lead());
  if (!dloss.defined() || !lse.defined()) bad_value("dloss and lse are needed");
  const c10::DeviceGuard guard(device);
  const at::Tensor dlogits = make(l.x.t.sizes(), l.x.t.scalar_type(), device);
  call("gear_hip_distill_backward", Scratch(), gear_hip_distill_backward, &l.d, ptr<float>(dloss), q.tokens.ptr(), q.tokens.wide,
       ptr<float>(q.logits), q.count, ptr<float>(lse), dlogits.data_ptr(), current_stream());
  return wrap(dlogits);
}

}  // namespace

void bind_tokens(py::module_ &m) {
  m.def("embed_tokens", &embed_tokens);
  m.def("embed_tokens_backward", &embed_tokens_backward);
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("token_log_probs", &token_log_probs);
  m.def("token_log_probs_backward", &token_log_probs_backward);
  m.def("distill", &distill);
  m.def("distill_backward", &distill_backward);
}
