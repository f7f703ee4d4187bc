// The operators between a batch of windows and a sequence model, as gear_amd.ops calls them.
#include <c10/core/DeviceGuard.h>

#include <cmath>

#include "host.hpp"

using namespace gear_hostops;

namespace {

[[noreturn]] void bad_value(const std::string &text) { throw py::value_error(text); }

int element_type(const at::Tensor &t, const char *name, bool with_f32) {
  switch (t.scalar_type()) {
    case at::kHalf: return GEAR_HIP_F16;
    case at::kBFloat16: return GEAR_HIP_BF16;
    case at::kFloat:
      if (with_f32) return GEAR_HIP_F32;
      [[fallthrough]];
    default:
      throw py::type_error(std::string(name) + " must have dtype " + (with_f32 ? "torch.float32, " : "") +
                           "torch.float16 or torch.bfloat16, got " + std::string(py::str(wrap(t).attr("dtype"))));
  }
}

// Rows of heads: [batch, tokens, heads, head_dim], the last contiguous, every row at a multiple of 16 bytes.
struct Rows {
  at::Tensor t;
  int64_t stride[3] = {0, 0, 0};
  Rows() = default;
  Rows(py::handle h, const char *name, at::ScalarType dtype, const at::Device &device) : t(any_tensor(h, name)) {
    if (t.scalar_type() != dtype)
      throw py::type_error(std::string(name) + " must have dtype " + std::string(c10::toString(dtype)) + " like q, got " +
                           std::string(c10::toString(t.scalar_type())));
    init(name);
    if (t.device() != device) bad_value(std::string(name) + " must live on the device of q");
  }
  Rows(py::handle h, const char *name) : t(any_tensor(h, name)) { init(name); }
  void shape(const char *name, int64_t batch, int64_t tokens, int64_t heads, int64_t dim) const {
    if (t.size(0) != batch || t.size(1) != tokens || t.size(2) != heads || t.size(3) != dim)
      bad_value(std::string(name) + " must have shape [" + std::to_string(batch) + ", " + std::to_string(tokens) + ", " +
                std::to_string(heads) + ", " + std::to_string(dim) + "], got " + std::string(py::str(wrap(t).attr("shape"))));
  }
  void *ptr() const { return t.data_ptr(); }

 private:
  void init(const char *name) {
    if (t.dim() != 4) bad_value(std::string(name) + " must be [batch, tokens, heads, head_dim]");
    if (!t.is_cuda()) bad_value(std::string(name) + " must live on the GPU");
    const int64_t size = (int64_t)t.element_size();
    bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(3) <= 1 || t.stride(3) == 1);
    for (int i = 0; i < 3; ++i) {
      stride[i] = t.size(i) <= 1 ? 0 : t.stride(i);
      fits = fits && stride[i] * size % 16 == 0;
    }
    if (!fits && t.numel() > 0)
      bad_value(std::string(name) + " must have contiguous head_dim elements and rows at multiples of 16 bytes "
                "(call .contiguous())");
  }
};

const at::Tensor &need_like(py::handle h, at::ScalarType dtype, const char *name, const at::Device &device,
                            at::IntArrayRef shape) {
  const at::Tensor &t = need(h, dtype, name);
  if (t.device() != device) bad_value(std::string(name) + " must live on the device of the other arguments");
  if (t.sizes() != shape) {
    std::string text;
    for (const int64_t n : shape) text += (text.empty() ? "" : ", ") + std::to_string(n);
    bad_value(std::string(name) + " must have shape [" + text + "], got " + std::string(py::str(wrap(t).attr("shape"))));
  }
  return t;
}

at::Tensor make(at::IntArrayRef shape, at::ScalarType dtype, const at::Device &device) {
  py::gil_scoped_release nogil;
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(device));
}

// ---- ranges of keys --------------------------------------------------------------------------------
const uint8_t *steps_flags(py::handle h, const char *name, at::Tensor &keep, at::IntArrayRef shape) {
  if (h.is_none()) return nullptr;
  const at::Tensor &t = any_tensor(h, name);
  if (t.scalar_type() != at::kByte && t.scalar_type() != at::kBool)
    throw py::type_error(std::string(name) + " must have dtype torch.uint8 or torch.bool");
  keep = need_like(h, t.scalar_type(), name, keep.defined() ? keep.device() : t.device(), shape);
  return static_cast<const uint8_t *>(keep.data_ptr());
}

py::object token_ranges(py::handle mask_, py::handle done_, int64_t tokens, const std::string &mode, int64_t prefix,
                        py::handle grid) {
  const py::handle some = mask_.is_none() ? done_ : mask_;
  if (some.is_none()) bad_value("mask or done is needed (for the shape of the batch)");
  const at::Tensor &shape_of = any_tensor(some, mask_.is_none() ? "done" : "mask");
  if (shape_of.dim() != 2) bad_value("mask and done must be [batch, steps]");
  int kind;
  if (mode == "causal")
    kind = GEAR_HIP_RANGE_CAUSAL;
  else if (mode == "step")
    kind = GEAR_HIP_RANGE_STEP;
  else if (mode == "document")
    kind = GEAR_HIP_RANGE_DOCUMENT;
  else
    bad_value("mode must be 'causal', 'step' or 'document', got '" + mode + "'");
  if (tokens < 1) bad_value("tokens_per_step must be at least 1");
  if (prefix < 0) bad_value("prefix must not be negative");
  int64_t rows = 0, cols = 0;
  if (!grid.is_none()) {
    const auto rc = grid.cast<std::pair<int64_t, int64_t>>();
    rows = rc.first, cols = rc.second;
    if (rows < 1 || cols < 1 || rows > tokens || rows * cols != tokens) bad_value("grid must be (rows, columns) of tokens_per_step tokens");
  }
  const at::Device device = shape_of.device();
  at::Tensor mask, done;
  const uint8_t *m = steps_flags(mask_, "mask", mask, shape_of.sizes());
  done = mask;
  const uint8_t *d = steps_flags(done_, "done", done, shape_of.sizes());
  const int64_t batch = shape_of.size(0), steps = shape_of.size(1);
  if (steps > 0 && tokens > ((int64_t)1 << 31) / steps) bad_value("steps * tokens_per_step must be below 2^31");
  const c10::DeviceGuard guard(device);
  const at::Tensor lo = make({batch, steps * tokens}, at::kInt, device), hi = make({batch, steps * tokens}, at::kInt, device),
                   pos = make({batch, steps * tokens, rows > 0 ? 3 : 1}, at::kInt, device);
  call("gear_hip_token_ranges", Scratch(), gear_hip_token_ranges, m, d, batch, steps, tokens, kind, prefix, rows, cols,
       ptr<int32_t>(lo), ptr<int32_t>(hi), ptr<int32_t>(pos), current_stream());
  return py::make_tuple(wrap(lo), wrap(hi), wrap(pos));
}

// ---- norm and rotation of heads --------------------------------------------------------------------
struct NormRotate {
  Rows q, k;
  at::Tensor keep[4];  // pos, freqs, weights
  at::ScalarType dtype, weight_dtype = at::kFloat;
  gear_hip_norm_rotate_desc d = {};

  NormRotate(py::handle q_, py::handle k_, py::handle pos, py::handle freqs, const std::vector<int64_t> &sections,
             py::handle q_weight, py::handle k_weight, double eps)
      : q(q_, "q") {
    dtype = q.t.scalar_type();
    d.dtype = element_type(q.t, "q", true);
    const at::Device device = q.t.device();
    k = Rows(k_, "k", dtype, device);
    const int64_t batch = q.t.size(0), tokens = q.t.size(1), dim = q.t.size(3);
    k.shape("k", batch, tokens, k.t.size(2), dim);
    if (dim < 16 || dim > 256 || dim % 16 != 0) bad_value("head_dim must be a multiple of 16, at most 256, got " + std::to_string(dim));
    if (sections.empty() || sections.size() > 4) bad_value("sections must name 1 to 4 axes");
    int64_t pairs = 0;
    for (size_t i = 0; i < sections.size(); ++i) {
      if (sections[i] < 0 || sections[i] > dim / 2) bad_value("sections must be numbers of pairs, 0 to head_dim / 2");
      pairs += sections[i];
      d.sections[i] = (int32_t)sections[i];
    }
    if (pairs > dim / 2) bad_value("sections hold more pairs than head_dim / 2");
    if (!(eps >= 0) || !std::isfinite(eps)) bad_value("eps must be a number of at least 0");
    d.axes = (int32_t)sections.size();
    keep[0] = need_like(pos, at::kInt, "pos", device, {batch, tokens, (int64_t)sections.size()});
    keep[1] = need_like(freqs, at::kDouble, "freqs", device, {pairs});
    weight(q_weight, "q_weight", 2, dim, device);
    weight(k_weight, "k_weight", 3, dim, device);
    if (keep[2].defined() && keep[3].defined() && keep[2].scalar_type() != keep[3].scalar_type())
      throw py::type_error("q_weight and k_weight must have one dtype");
    d.q = q.ptr(), d.k = k.ptr();
    std::copy(q.stride, q.stride + 3, d.q_stride);
    std::copy(k.stride, k.stride + 3, d.k_stride);
    d.batch = batch, d.tokens = tokens;
    d.q_heads = (int32_t)q.t.size(2), d.k_heads = (int32_t)k.t.size(2), d.head_dim = (int32_t)dim;
    d.pos = ptr<int32_t>(keep[0]), d.freqs = ptr<double>(keep[1]);
    d.q_weight = keep[2].defined() ? keep[2].data_ptr() : nullptr;
    d.k_weight = keep[3].defined() ? keep[3].data_ptr() : nullptr;
    d.weight_f32 = weight_dtype == at::kFloat;
    d.eps = (float)eps;
  }
  at::Device device() const { return q.t.device(); }

 private:
  void weight(py::handle h, const char *name, int at, int64_t dim, const at::Device &device) {
    if (h.is_none()) return;
    const at::Tensor &t = any_tensor(h, name);
    if (t.scalar_type() != at::kFloat && t.scalar_type() != dtype)
      throw py::type_error(std::string(name) + " must have dtype torch.float32 or that of q");
    weight_dtype = t.scalar_type();
    keep[at] = need_like(h, weight_dtype, name, device, {dim});
  }
};

py::object norm_rotate(py::handle q, py::handle k, py::handle pos, py::handle freqs, const std::vector<int64_t> &sections,
                       py::handle q_weight, py::handle k_weight, double eps) {
  NormRotate n(q, k, pos, freqs, sections, q_weight, k_weight, eps);
  const c10::DeviceGuard guard(n.device());
  const at::Tensor qo = make(n.q.t.sizes(), n.dtype, n.device()), ko = make(n.k.t.sizes(), n.dtype, n.device());
  call("gear_hip_norm_rotate", Scratch(), gear_hip_norm_rotate, &n.d, qo.data_ptr(), ko.data_ptr(), current_stream());
  return py::make_tuple(wrap(qo), wrap(ko));
}

py::object norm_rotate_append(py::handle q, py::handle k, py::handle v_, py::handle pos, py::handle freqs,
                              const std::vector<int64_t> &sections, py::handle q_weight, py::handle k_weight,
                              py::handle slots_, py::handle k_cache_, py::handle v_cache_, double eps) {
  NormRotate n(q, k, pos, freqs, sections, q_weight, k_weight, eps);
  const at::Device device = n.device();
  const Rows v(v_, "v", n.dtype, device), kc(k_cache_, "k_cache", n.dtype, device), vc(v_cache_, "v_cache", n.dtype, device);
  v.shape("v", n.d.batch, n.d.tokens, n.d.k_heads, n.d.head_dim);
  kc.shape("k_cache", n.d.batch, kc.t.size(1), n.d.k_heads, n.d.head_dim);
  vc.shape("v_cache", n.d.batch, kc.t.size(1), n.d.k_heads, n.d.head_dim);
  const at::Tensor &slots = need_like(slots_, at::kInt, "slots", device, {n.d.batch, n.d.tokens});
  const c10::DeviceGuard guard(device);
  const at::Tensor qo = make(n.q.t.sizes(), n.dtype, device);
  call("gear_hip_norm_rotate_append", Scratch(), gear_hip_norm_rotate_append, &n.d, v.ptr(), v.stride, qo.data_ptr(),
       ptr<int32_t>(slots), kc.t.size(1), kc.ptr(), kc.stride, vc.ptr(), vc.stride, current_stream());
  return wrap(qo);
}

py::object norm_rotate_backward(py::handle gq_, py::handle gk_, py::handle q, py::handle k, py::handle pos, py::handle freqs,
                                const std::vector<int64_t> &sections, py::handle q_weight, py::handle k_weight, double eps,
                                py::handle ws) {
  NormRotate n(q, k, pos, freqs, sections, q_weight, k_weight, eps);
  const at::Device device = n.device();
  const Rows gq(gq_, "dq_out", n.dtype, device), gk(gk_, "dk_out", n.dtype, device);
  gq.shape("dq_out", n.d.batch, n.d.tokens, n.d.q_heads, n.d.head_dim);
  gk.shape("dk_out", n.d.batch, n.d.tokens, n.d.k_heads, n.d.head_dim);
  const c10::DeviceGuard guard(device);
  const at::Tensor dq = make(n.q.t.sizes(), n.dtype, device), dk = make(n.k.t.sizes(), n.dtype, device);
  py::object dqw = py::none(), dkw = py::none();
  if (n.d.q_weight) dqw = wrap(make({n.d.head_dim}, n.weight_dtype, device));
  if (n.d.k_weight) dkw = wrap(make({n.d.head_dim}, n.weight_dtype, device));
  const Scratch s = n.d.q_weight || n.d.k_weight
                        ? Scratch(ws, "norm_rotate", gear_hip_norm_rotate_backward_workspace_bytes(n.d.head_dim), device)
                        : Scratch();
  call("gear_hip_norm_rotate_backward", s, gear_hip_norm_rotate_backward, &n.d, gq.ptr(), gq.stride, gk.ptr(), gk.stride,
       dq.data_ptr(), dk.data_ptr(), ptr_or_null<void>(dqw, "dq_weight"), ptr_or_null<void>(dkw, "dk_weight"), s.ptr, s.bytes,
       current_stream());
  return py::make_tuple(wrap(dq), wrap(dk), dqw, dkw);
}

// ---- attention -------------------------------------------------------------------------------------
struct Attention {
  Rows q, k, v;
  at::Tensor keep[3];  // lo, hi, slopes
  at::ScalarType dtype;
  gear_hip_attention_desc d = {};

  Attention(py::handle q_, py::handle k_, py::handle v_, py::handle lo, py::handle hi, py::handle scale, double cap,
            py::handle slopes, const char *k_name, const char *v_name)
      : q(q_, "q") {
    dtype = q.t.scalar_type();
    d.dtype = element_type(q.t, "q", false);
    const at::Device device = q.t.device();
    k = Rows(k_, k_name, dtype, device), v = Rows(v_, v_name, dtype, device);
    const int64_t batch = q.t.size(0), queries = q.t.size(1), heads = q.t.size(2), dim = q.t.size(3);
    if (dim < 16 || dim > 128 || dim % 16 != 0) bad_value("head_dim must be a multiple of 16, at most 128, got " + std::to_string(dim));
    k.shape(k_name, batch, k.t.size(1), k.t.size(2), dim);
    v.shape(v_name, batch, k.t.size(1), k.t.size(2), dim);
    if (heads < 1 || k.t.size(2) < 1 || heads % k.t.size(2) != 0)
      bad_value("the heads of q must be a multiple of those of " + std::string(k_name));
    keep[0] = need_like(lo, at::kInt, "lo", device, {batch, queries});
    keep[1] = need_like(hi, at::kInt, "hi", device, {batch, queries});
    if (!slopes.is_none()) keep[2] = need_like(slopes, at::kFloat, "slopes", device, {heads});
    const double s = scale.is_none() ? 1.0 / std::sqrt((double)dim) : scale.cast<double>();
    if (!((float)s > 0) || !(s < 1e30)) bad_value("scale must be a number above 0 (of 32 bits, below 1e30)");
    if (!(cap >= 0) || !(cap < 1e30) || (cap > 0 && !(s / cap < 1e30)))
      bad_value("cap must be a number of at least 0 (0: no cap), below 1e30 and above 1e-30 times the scale");
    d.q = q.ptr(), d.k = k.ptr(), d.v = v.ptr();
    std::copy(q.stride, q.stride + 3, d.q_stride);
    std::copy(k.stride, k.stride + 3, d.k_stride);
    std::copy(v.stride, v.stride + 3, d.v_stride);
    d.batch = batch, d.queries = queries, d.keys = k.t.size(1);
    d.heads = (int32_t)heads, d.kv_heads = (int32_t)k.t.size(2), d.head_dim = (int32_t)dim;
    d.lo = ptr<int32_t>(keep[0]), d.hi = ptr<int32_t>(keep[1]);
    d.slopes = keep[2].defined() ? ptr<float>(keep[2]) : nullptr;
    d.scale = (float)s, d.cap = (float)cap;
  }
  at::Device device() const { return q.t.device(); }
};

py::object range_attention(py::handle q, py::handle k, py::handle v, py::handle lo, py::handle hi, py::handle scale, double cap,
                           py::handle slopes) {
  Attention a(q, k, v, lo, hi, scale, cap, slopes, "k", "v");
  const c10::DeviceGuard guard(a.device());
  const at::Tensor out = make(a.q.t.sizes(), a.dtype, a.device()),
                   lse = make({a.d.batch, a.d.heads, a.d.queries}, at::kFloat, a.device());
  call("gear_hip_attention", Scratch(), gear_hip_attention, &a.d, out.data_ptr(), ptr<float>(lse), current_stream());
  return py::make_tuple(wrap(out), wrap(lse));
}

py::object range_attention_backward(py::handle dout_, py::handle q, py::handle k, py::handle v, py::handle out_,
                                    py::handle lse_, py::handle lo, py::handle hi, py::handle scale, double cap,
                                    py::handle slopes, py::handle ws) {
  Attention a(q, k, v, lo, hi, scale, cap, slopes, "k", "v");
  const at::Device device = a.device();
  const Rows dout(dout_, "dout", a.dtype, device);
  dout.shape("dout", a.d.batch, a.d.queries, a.d.heads, a.d.head_dim);
  const at::Tensor &out = need_like(out_, a.dtype, "out", device, a.q.t.sizes()),
                   &lse = need_like(lse_, at::kFloat, "lse", device, {a.d.batch, a.d.heads, a.d.queries});
  const c10::DeviceGuard guard(device);
  const at::Tensor dq = make(a.q.t.sizes(), a.dtype, device), dk = make(a.k.t.sizes(), a.dtype, device),
                   dv = make(a.k.t.sizes(), a.dtype, device);
  const Scratch s(ws, "attention_backward", gear_hip_attention_backward_workspace_bytes(a.d.batch, a.d.queries, a.d.heads), device);
  call("gear_hip_attention_backward", s, gear_hip_attention_backward, &a.d, dout.ptr(), dout.stride, out.data_ptr(),
       ptr<float>(lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), s.ptr, s.bytes, current_stream());
  return py::make_tuple(wrap(dq), wrap(dk), wrap(dv));
}

py::object range_attention_step(py::handle q, py::handle k, py::handle v, py::handle lo, py::handle hi, py::handle scale,
                                double cap, py::handle slopes, py::handle ws) {
  Attention a(q, k, v, lo, hi, scale, cap, slopes, "k_cache", "v_cache");
  const at::Device device = a.device();
  const c10::DeviceGuard guard(device);
  const at::Tensor out = make(a.q.t.sizes(), a.dtype, device);
  const Scratch s(ws, "attention_step",
                  gear_hip_attention_step_workspace_bytes(a.d.batch, a.d.queries, a.d.keys, a.d.heads, a.d.kv_heads, a.d.head_dim),
                  device);
  call("gear_hip_attention_step", s, gear_hip_attention_step, &a.d, out.data_ptr(), s.ptr, s.bytes, current_stream());
  return wrap(out);
}

}  // namespace

void bind_sequence(py::module_ &m) {
  m.def("token_ranges", &token_ranges);
  m.def("norm_rotate", &norm_rotate);
  m.def("norm_rotate_append", &norm_rotate_append);
  m.def("norm_rotate_backward", &norm_rotate_backward);
  m.def("range_attention", &range_attention);
  m.def("range_attention_backward", &range_attention_backward);
  m.def("range_attention_step", &range_attention_step);
}
