// Python side of the paged-cache operators (instantllm_b200/paged.py): checks the tensors of a call, allocates its results and
// hands it to the C ABI (include/vpass.h, vp_paged_*). Written against torch's C++ tensors because a call of a few
// microseconds on the GPU took 7 us to check and pack in Python.
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/vpass.h"

namespace {

struct Refused : std::runtime_error {  // becomes a ValueError
  using std::runtime_error::runtime_error;
};
void want(bool ok, const std::string& what) {
  if (!ok) throw Refused(what);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

// The operators have no backward: a result that silently has no gradient would be wrong.
void no_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts)
    want(!t->requires_grad(), "the paged operators have no gradients: call them under torch.no_grad() or on detached tensors");
}

// The stride of a dimension; torch leaves any number in those of one element, which mean nothing.
int64_t stride(const at::Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

// An int argument, held within 32 bits (a window past every length is no window).
int32_t small(PyObject* o) {
  const long x = PyLong_AsLong(o);
  return (int32_t)std::max(-1l, std::min(x, 0x7fffffffl));
}

struct Call {  // the layer's part of every call: its cache struct (ctypes memory) and device
  const vp_paged* c;
  int device;
  at::ScalarType type;
  Call(PyObject* cache, PyObject* dev)
      : c(static_cast<const vp_paged*>(PyLong_AsVoidPtr(cache))), device((int)PyLong_AsLong(dev)),
        type(c->type == VP_T_F16 ? at::kHalf : at::kBFloat16) {
    if (c10::cuda::current_device() != device)
      throw Refused("the cache lives on cuda:" + std::to_string(device) + ": make it the current device");
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == device; }

  // contiguous int32 of a shape; None gives null
  const int32_t* index(PyObject* o, const char* name, at::IntArrayRef shape, bool optional = false) const {
    if (optional && o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kInt || t.sizes() != shape || !here(t) || !t.is_contiguous()) {
      std::string s;
      for (int64_t x : shape) s += (s.empty() ? "" : ", ") + std::to_string(x);
      throw Refused(std::string(name) + " must be a contiguous int32 tensor of shape (" + s + ") on cuda:" + std::to_string(device));
    }
    return t.const_data_ptr<int32_t>();
  }
  at::Tensor out(PyObject* o, at::IntArrayRef shape) const {
    if (o == Py_None) return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)device));
    const at::Tensor& t = tensor(o, "out");
    want(t.sizes() == shape && t.scalar_type() == type && here(t) && t.stride(-1) == 1,
         "out must have q's shape and the cache's type, elements of a head adjacent");
    return t;
  }
};

// Runs f; what it throws becomes a Python exception.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// append(cache, device, q, k, v, seq, slot, pos, rope, interleaved, out) -> rotated queries, or an error code
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    want(n_args == 11, "append takes 11 arguments");
    const Call call(a[0], a[1]);
    const vp_paged& c = *call.c;
    const at::Tensor &q = tensor(a[2], "q"), &k = tensor(a[3], "k"), &v = tensor(a[4], "v");
    no_grad({&q, &k, &v});
    const at::ScalarType in = q.scalar_type();
    want(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == in && v.scalar_type() == in,
         "q, k and v must be [rows][heads][head_dim] of one type");
    const int64_t n = q.size(0);
    want(n <= 0x7fffffff, "too many rows");
    want(q.size(2) == c.head_dim && k.size(0) == n && k.size(1) == c.n_kv && k.size(2) == c.head_dim,
         "expected k and v of " + std::to_string(n) + " rows and " + std::to_string(c.n_kv) + " heads of " + std::to_string(c.head_dim));
    want(in == call.type || in == at::kFloat, "rows must have the cache's type or fp32");
    want(q.stride(2) == 1 && k.stride(2) == 1 && v.stride(2) == 1, "the elements of a head must be adjacent");
    want(call.here(q) && call.here(k) && call.here(v), "rows must be on cuda:" + std::to_string(call.device));
    vp_paged_rows r{};
    const at::IntArrayRef rows(&n, 1);
    r.seq = call.index(a[5], "seq", rows);
    r.slot = call.index(a[6], "slot", rows);
    if (a[8] != Py_None) {
      const at::Tensor& rope = tensor(a[8], "rope");
      want(rope.dim() == 3 && rope.size(2) == 2 && rope.scalar_type() == at::kFloat && rope.is_contiguous() && call.here(rope),
           "rope must be a contiguous fp32 [positions][rot_dim / 2][2] tensor on the cache's device");
      want(a[7] != Py_None, "a rotation needs pos");
      r.pos = call.index(a[7], "pos", rows);
      r.rope = rope.const_data_ptr<float>();
      r.rope_rows = (int32_t)rope.size(0);
      r.rot_dim = (int32_t)(2 * rope.size(1));
    }
    const at::Tensor out = call.out(a[10], q.sizes());
    r.q = q.const_data_ptr();
    r.k = k.const_data_ptr();
    r.v = v.const_data_ptr();
    r.q_out = out.data_ptr();
    r.q_row = stride(q, 0), r.q_head = stride(q, 1);
    r.k_row = stride(k, 0), r.k_head = stride(k, 1);
    r.v_row = stride(v, 0), r.v_head = stride(v, 1);
    r.out_row = stride(out, 0), r.out_head = stride(out, 1);
    r.type = in == at::kFloat ? VP_T_F32 : c.type;
    r.rows = (int32_t)n;
    r.n_q = (int32_t)q.size(1);
    r.interleaved = PyObject_IsTrue(a[9]);
    const int rc = vp_paged_append(&c, &r, call.stream());
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  });
}

// attend(prompts, cache, device, work, q, lens, mask, q_start, seqs, window, sinks, scale, out, return_lse)
// -> out, or (out, lse), or an error code. work: a list whose first tensor is the workspace of the cache's layers.
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    want(n_args == 14, "attend takes 14 arguments");
    const bool prompts = a[0] == Py_True;
    const Call call(a[1], a[2]);
    const vp_paged& c = *call.c;
    const at::Tensor &q = tensor(a[4], "q"), &lens = tensor(a[5], "lens");
    want(q.dim() == 3 || (q.dim() == 4 && !prompts), prompts ? "q must be [rows][query heads][head_dim]"
                                                             : "q must be [n][rows][query heads][head_dim] or [n][query heads][head_dim]");
    no_grad({&q});
    const bool one = q.dim() == 3 && !prompts;
    want(q.size(-1) == c.head_dim && q.scalar_type() == call.type && call.here(q) && q.stride(-1) == 1,
         "q must have the cache's type, device and head_dim, elements of a head adjacent");
    want(lens.dim() == 1, "lens must be one-dimensional");
    const int64_t n = prompts ? lens.size(0) : q.size(0), rows = prompts ? q.size(0) : one ? 1 : q.size(1);
    want(n < 0x7fffffff && rows <= 0x7fffffff, "too many rows");
    vp_paged_attn t{};
    t.lens = call.index(a[5], "lens", {n});
    t.mask = call.index(a[6], "mask", {n, rows}, true);
    if (prompts) t.q_start = call.index(a[7], "q_start", {n + 1});
    t.seqs = call.index(a[8], "seqs", {n}, true);
    want(t.seqs || n <= c.n_seqs, std::to_string(n) + " requests, and a table of " + std::to_string(c.n_seqs));
    t.n_q = (int32_t)q.size(-2);
    const at::Tensor out = call.out(a[12], q.sizes());
    at::Tensor lse;
    if (PyObject_IsTrue(a[13])) {
      lse = at::empty(q.sizes().slice(0, q.dim() - 1), at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, (c10::DeviceIndex)call.device));
      t.lse = lse.mutable_data_ptr<float>();
    }
    // The layer brought the workspace when it was built, large enough for every call: a captured graph holds its address, and
    // its counters were zeroed outside any capture, so a call never makes or replaces one.
    PyObject* held = PyList_Size(a[3]) > 0 ? PyList_GetItem(a[3], 0) : Py_None;  // borrowed
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor& work = tensor(held, "work");
    want(call.here(work) && (size_t)work.nbytes() >= vp_paged_work_bytes(c.head_dim, t.n_q, c.n_kv, (int32_t)rows),
         "the layer's workspace was replaced by another");
    t.work = work.data_ptr();
    t.work_bytes = (uint64_t)work.nbytes();
    t.q = q.const_data_ptr();
    t.out = out.data_ptr();
    const int heads = (int)q.dim() - 2;
    t.q_head = stride(q, heads), t.out_head = stride(out, heads);
    if (prompts) t.q_row = stride(q, 0), t.out_row = stride(out, 0);
    else t.q_seq = stride(q, 0), t.out_seq = stride(out, 0);
    if (!prompts && !one) t.q_row = stride(q, 1), t.out_row = stride(out, 1);
    t.scale = a[11] == Py_None ? 1.f / std::sqrt((float)c.head_dim) : (float)PyFloat_AsDouble(a[11]);
    t.n = (int32_t)n;
    t.rows = (int32_t)rows;
    t.window = small(a[9]);
    t.sinks = small(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const int rc = (prompts ? vp_paged_prefill : vp_paged_decode)(&c, &t, call.stream());
    if (rc) return PyLong_FromLong(rc);
    if (!lse.defined()) return THPVariable_Wrap(out);
    PyObject *x = THPVariable_Wrap(out), *y = THPVariable_Wrap(lse), *both = PyTuple_Pack(2, x, y);
    Py_DECREF(x);
    Py_DECREF(y);
    return both;
  });
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
