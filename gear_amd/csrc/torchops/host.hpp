// What the sources of `_hostops` share: arguments, scratch, calls into libgearhip.so.
#pragma once
#include <ATen/ATen.h>
#include <ATen/hip/HIPGeneratorImpl.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "gear_hip.h"

namespace gear_hostops {

namespace py = pybind11;

// ---- arguments -----------------------------------------------------------------------------------
inline const char *dtype_text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kLong: return "torch.int64";
    case at::kByte: return "torch.uint8";
    default: return c10::toString(t);
  }
}

inline const at::Tensor &any_tensor(py::handle h, const char *name) {
  if (!THPVariable_Check(h.ptr())) throw py::type_error(std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(h.ptr());
}

inline const at::Tensor &need(py::handle h, at::ScalarType dtype, const char *name) {
  const at::Tensor &t = any_tensor(h, name);
  if (t.scalar_type() != dtype)
    throw py::type_error(std::string(name) + " must have dtype " + dtype_text(dtype) + ", got " +
                         std::string(py::str(h.attr("dtype"))));
  if (!t.is_contiguous()) throw py::value_error(std::string(name) + " must be contiguous");
  if (!t.is_cuda()) throw py::value_error(std::string(name) + " must live on the GPU");
  return t;
}

template <typename T>
T *ptr(const at::Tensor &t) {
  return static_cast<T *>(t.data_ptr());
}
// an optional output: the tensor, or null
template <typename T>
T *ptr_or_null(py::handle h, const char *name) {
  return h.is_none() ? nullptr : static_cast<T *>(any_tensor(h, name).data_ptr());
}

// (where the GIL is held)
inline at::Tensor empty(int64_t n, at::ScalarType dtype, const at::Device &device) {
  py::gil_scoped_release nogil;
  return at::empty({n}, at::TensorOptions().dtype(dtype).device(device));
}

inline py::object wrap(const at::Tensor &t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

inline void *current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

// (with or without the GIL)
inline void check(const char *fn, int code) {
  if (code == 0) return;
  py::gil_scoped_acquire gil;
  py::module_::import("gear_amd._cabi").attr("check")(fn, code);  // raises
}

// ---- scratch -------------------------------------------------------------------------------------
// Scratch tensors per (purpose, device, stream), grown on demand and reused: no allocation in
// steady state, and calls enqueued on different streams never share a workspace.  Python sees
// get(); an instance whose get() was replaced is asked through it.
class Workspace {
 public:
  struct Entry {
    at::Tensor buf;
    std::mutex order;  // held while a call enqueues its launches on the buffer's stream
  };
  // (the GIL is held)
  std::shared_ptr<Entry> entry(const char *tag, const at::Device &device) {
    const c10::DeviceIndex index = device.has_index() ? device.index() : c10::hip::current_device();
    std::shared_ptr<Entry> &slot = entries_[Key{tag, index, c10::hip::getCurrentHIPStream(index).stream()}];
    if (!slot) slot = std::make_shared<Entry>();
    return slot;
  }
  static at::Tensor buffer(Entry &e, size_t bytes, const at::Device &device) {
    if (!e.buf.defined() || (size_t)e.buf.numel() < bytes) {
      at::Tensor grown = empty((int64_t)std::max<size_t>(bytes, 256), at::kByte, device);
      // (another thread may have been here meanwhile)
      if (!e.buf.defined() || e.buf.numel() < grown.numel()) e.buf = grown;
    }
    return e.buf;
  }

 private:
  struct Key {
    std::string tag;
    c10::DeviceIndex device;
    void *stream;
    bool operator==(const Key &o) const { return stream == o.stream && device == o.device && tag == o.tag; }
  };
  struct Hash {
    size_t operator()(const Key &k) const {
      return std::hash<std::string>()(k.tag) ^ (std::hash<void *>()(k.stream) * 31 + (size_t)k.device);
    }
  };
  std::unordered_map<Key, std::shared_ptr<Entry>, Hash> entries_;
};

struct Scratch {
  void *ptr = nullptr;
  size_t bytes = 0;
  at::Tensor keep;
  std::shared_ptr<Workspace::Entry> entry;
  Scratch() = default;  // none
  Scratch(py::handle ws, const char *tag, size_t want, const at::Device &device) {
    entry = ws.cast<Workspace &>().entry(tag, device);
    PyObject **dict = _PyObject_GetDictPtr(ws.ptr());
    if (dict != nullptr && *dict != nullptr && PyDict_GET_SIZE(*dict) != 0)
      keep = THPVariable_Unpack(
          ws.attr("get")(tag, want, py::reinterpret_steal<py::object>(THPDevice_New(device))).ptr());
    else
      keep = Workspace::buffer(*entry, want, device);
    ptr = keep.data_ptr();
    bytes = (size_t)keep.numel();
  }
};

// f(args) without the GIL.  Two threads that enqueue on one stream share its scratch: the launches of
// one call follow each other, so that no other call's lie between them.
template <typename F>
int launches(const Scratch &s, const F &f) {
  if (!s.entry) return f();
  std::lock_guard<std::mutex> order(s.entry->order);
  return f();
}
template <typename F, typename... A>
void call(const char *name, const Scratch &s, const F &f, A... args) {
  int code;
  {
    py::gil_scoped_release nogil;
    code = launches(s, [&] { return f(args...); });
  }
  check(name, code);
}

}  // namespace gear_hostops
