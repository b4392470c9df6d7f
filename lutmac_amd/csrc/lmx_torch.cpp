// lmx_torch.cpp -- the 8-bit serving operators on torch tensors: what
// lutmac_amd.kv8 and lutmac_amd.linear_i8 check of their arguments, the outputs
// and workspaces that they allocate, and their calls into the C ABI.
//
// A serving loop calls them eagerly many times a step, and in Python a call's
// checks took longer than the kernels of a small one (host time of an append of 64
// rows 12.4 us, here 5.0, on the GPU 6.7; of the attention of one row 11.1, 5.0
// and 6.0).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <memory>
#include <string>

#include "lutmac_hip.h"
#include "lutmac_kv8.h"

namespace {

struct PyError {};   // a Python exception is set

PyObject *g_lmx_error = nullptr;   // lutmac_amd.LmxError

[[noreturn]] void raise_lmx(int status, const std::string &message) {
  PyObject *e = PyObject_CallFunction(g_lmx_error, "is", status, message.c_str());
  if (e) {
    PyErr_SetObject(g_lmx_error, e);
    Py_DECREF(e);
  }
  throw PyError{};
}
void check(int status) {
  if (status != LMX_OK) raise_lmx(status, lmx_last_error());
}

std::string text(const at::Tensor &t) {
  std::string s = std::string(c10::toString(t.scalar_type())) + " [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  s += "] with strides (";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
  return s + ") on " + t.device().str();
}
[[noreturn]] void raise_value(const std::string &message) {
  PyErr_SetString(PyExc_ValueError, message.c_str());
  throw PyError{};
}
[[noreturn]] void bad(const char *name, const at::Tensor &t, const std::string &want) {
  raise_value(std::string(name) + ": " + text(t) + ", expected " + want);
}

const at::Tensor &tensor(const char *name, PyObject *o) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
    throw PyError{};
  }
  return THPVariable_Unpack(o);
}

int type_of(const char *name, const at::Tensor &t) {
  switch (t.scalar_type()) {
  case at::kFloat: return LMX_F32;
  case at::kHalf: return LMX_F16;
  case at::kBFloat16: return LMX_BF16;
  default: raise_lmx(LMX_ERR_UNSUPPORTED_FORMAT, std::string(name) + " is " + c10::toString(t.scalar_type()) + ": float32, float16 or bfloat16");
  }
}

bool has_sizes(const at::Tensor &t, at::IntArrayRef sizes) { return t.sizes().equals(sizes); }

// Every tensor of a call lies on one device, the current one, where it launches.
void check_device(const at::Tensor &t, int device) {
  if (!t.is_cuda() || t.get_device() != device)
    raise_value("expected tensors on the current device, got one on " + t.device().str());
}
int check_devices(std::initializer_list<const at::Tensor *> tensors) {   // (null: an argument left out)
  const at::Tensor &first = **tensors.begin();
  const int device = first.is_cuda() ? int(first.get_device()) : -1;
  for (const at::Tensor *t : tensors)
    if (t) check_device(*t, device);
  if (device != int(c10::hip::current_device()))
    raise_value("expected tensors on the current device, got " + first.device().str());
  return device;
}
// Work runs on torch's current stream, whose memory new outputs and workspaces are.
void *stream_on(int device) { return c10::hip::getCurrentHIPStream(c10::DeviceIndex(device)).stream(); }

// Runs f() -> new reference; C++ exceptions become Python's.
template <class F>
PyObject *guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const PyError &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool arguments(const char *name, Py_ssize_t got, Py_ssize_t want) {
  if (got != want) PyErr_Format(PyExc_TypeError, "%s: %zd arguments, expected %zd", name, got, want);
  return got == want;
}

// ---- cache ----

// The tensors of a cache: held, and looked at anew in every call, so that a call
// writes what they are then and nothing that they gave up.
struct Cache {
  at::Tensor k, v, scale[2];

  // Their sizes and pointers, checked.
  lmx_kv8_cache now() const {
    if (k.dim() != 4 || k.size(2) != LMX_KV8_PAGE || (k.size(3) != 64 && k.size(3) != 128) || k.scalar_type() != at::kChar ||
        !k.is_contiguous())
      bad("k", k, "contiguous int8 [pages, kv_heads, 64, 64 or 128]");
    const int64_t pages = k.size(0), heads = k.size(1), hd = k.size(3);
    if (v.scalar_type() != at::kChar || !has_sizes(v, {pages, heads, hd, LMX_KV8_PAGE}) || !v.is_contiguous())
      bad("v", v, "contiguous int8 [pages, kv_heads, head_dim, 64], as k has them");
    if (v.device() != k.device()) raise_value("the cache's tensors must be on one device");
    for (int i = 0; i < 2; ++i) {
      const at::Tensor &s = scale[i];
      if (s.scalar_type() != at::kFloat || !has_sizes(s, {pages, heads, LMX_KV8_PAGE / LMX_KV8_BLOCK}) || !s.is_contiguous())
        bad(i ? "v_scale" : "k_scale", s, "contiguous float32 [pages, kv_heads, 4], as k has them");
      if (s.device() != k.device()) raise_value("the cache's tensors must be on one device");
    }
    return {static_cast<int8_t *>(k.data_ptr()), static_cast<int8_t *>(v.data_ptr()), static_cast<float *>(scale[0].data_ptr()),
            static_cast<float *>(scale[1].data_ptr()), size_t(pages), size_t(heads), size_t(hd)};
  }
};
constexpr const char *kCache = "lutmac_amd.kv8_cache";
const Cache &cache_of(PyObject *o) {
  const Cache *c = static_cast<const Cache *>(PyCapsule_GetPointer(o, kCache));
  if (!c) throw PyError{};
  return *c;
}

// (k, v, k_scale, v_scale) -> what the calls take.
PyObject *kv8_cache(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_cache", n, 4)) throw PyError{};
    std::unique_ptr<Cache> c(new Cache{tensor("k", args[0]), tensor("v", args[1]), {tensor("k_scale", args[2]), tensor("v_scale", args[3])}});
    c->now();
    PyObject *o = PyCapsule_New(c.get(), kCache, [](PyObject *o) { delete static_cast<Cache *>(PyCapsule_GetPointer(o, kCache)); });
    if (!o) throw PyError{};
    c.release();
    return o;
  });
}

// A row tensor [rows, heads, head_dim], rows any stride apart: its row stride.
size_t row_stride(const char *name, const at::Tensor &t, at::ScalarType type, int64_t rows, int64_t heads, int64_t hd) {
  if (t.scalar_type() != type || !has_sizes(t, {rows, heads, hd}))
    bad(name, t, std::string(c10::toString(type)) + " [" + std::to_string(rows) + ", " + std::to_string(heads) + ", " +
                     std::to_string(hd) + "]");
  if (rows && (t.stride(2) != 1 || (heads > 1 && t.stride(1) != hd))) bad(name, t, "a row's heads side by side");
  return size_t(rows > 1 ? t.stride(0) : heads * hd);   // (a single row's stride says nothing)
}

// The call's batch, but for its tensors' device.
lmx_kv8_batch batch_of(PyObject *const *args, int64_t rows) {
  const at::Tensor &offsets = tensor("offsets", args[0]), &lengths = tensor("lengths", args[1]), &pages = tensor("pages", args[2]);
  if (pages.scalar_type() != at::kInt || pages.dim() != 2 || !pages.is_contiguous()) bad("pages", pages, "contiguous int32 of 2 dimensions");
  const int64_t n = pages.size(0);
  if (offsets.scalar_type() != at::kInt || !has_sizes(offsets, {n + 1}) || !offsets.is_contiguous())
    bad("offsets", offsets, "contiguous int32 [" + std::to_string(n + 1) + "] beside " + std::to_string(n) + " page table rows");
  if (lengths.scalar_type() != at::kInt || !has_sizes(lengths, {n}) || !lengths.is_contiguous())
    bad("lengths", lengths, "contiguous int32 [" + std::to_string(n) + "] beside " + std::to_string(n) + " page table rows");
  return {static_cast<const int32_t *>(offsets.data_ptr()), static_cast<const int32_t *>(lengths.data_ptr()),
          static_cast<const int32_t *>(pages.data_ptr()), size_t(n), size_t(pages.size(1)), size_t(rows)};
}

int check_call(const Cache &c, std::initializer_list<const at::Tensor *> tensors) {
  const int device = check_devices(tensors);
  if (c.k.device() != (*tensors.begin())->device()) raise_value("expected tensors on the cache's device");
  return device;
}

// (cache, k, v, offsets, lengths, pages, rope, q, q_out) -> q_out
PyObject *kv8_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_append", n, 9)) throw PyError{};
    const Cache &held = cache_of(args[0]);
    const lmx_kv8_cache c = held.now();
    const at::Tensor &k = tensor("k", args[1]), &v = tensor("v", args[2]);
    const int type = type_of("k", k);
    const at::ScalarType st = k.scalar_type();
    const int64_t kv = int64_t(c.n_kv_heads), hd = int64_t(c.head_dim), rows = k.dim() ? k.size(0) : 0;
    const size_t ks = row_stride("k", k, st, rows, kv, hd), vs = row_stride("v", v, st, rows, kv, hd);
    const lmx_kv8_batch b = batch_of(args + 3, rows);
    const at::Tensor *rope = args[6] != Py_None ? &tensor("rope", args[6]) : nullptr;
    const int64_t positions = rope && rope->dim() ? rope->size(0) : 0;
    if (rope && (rope->scalar_type() != at::kFloat || !has_sizes(*rope, {positions, hd / 2, 2}) || !rope->is_contiguous()))
      bad("rope", *rope, "contiguous float32 [positions, " + std::to_string(hd / 2) + ", 2]");
    const at::Tensor *q = args[7] != Py_None ? &tensor("q", args[7]) : nullptr;
    const at::Tensor *given = args[8] != Py_None ? &tensor("q_out", args[8]) : nullptr;
    if (given && !q) raise_value("q_out without q");
    const int64_t heads = q && q->dim() == 3 ? q->size(1) : 0;
    const size_t qs = q ? row_stride("q", *q, st, rows, heads, hd) : 0;
    const size_t os = given ? row_stride("q_out", *given, st, rows, heads, hd) : size_t(heads * hd);
    const int device = check_call(held, {&k, &v, &THPVariable_Unpack(args[3]), &THPVariable_Unpack(args[4]), &THPVariable_Unpack(args[5]), rope, q, given});
    at::Tensor out;
    if (q) out = given ? *given : at::empty({rows, heads, hd}, q->options());
    check(lmx_kv8_append(&c, &b, type, k.data_ptr(), ks, v.data_ptr(), vs, q ? q->data_ptr() : nullptr, qs,
                         q ? out.data_ptr() : nullptr, os, size_t(heads), rope ? static_cast<const float *>(rope->data_ptr()) : nullptr,
                         size_t(positions), stream_on(device)));
    if (!out.defined()) Py_RETURN_NONE;
    if (args[8] != Py_None) return Py_NewRef(args[8]);
    return THPVariable_Wrap(std::move(out));
  });
}

// Workspace of a call: the caller's, or one that torch allocates.
at::Tensor workspace_of(PyObject *given, size_t need, int device, void *&p, size_t &bytes) {
  at::Tensor t;
  p = nullptr;
  if (given != Py_None) {
    t = tensor("workspace", given);
    check_device(t, device);
    if (!t.is_contiguous()) bad("workspace", t, "a contiguous tensor");
    bytes = t.nbytes();
  } else {
    bytes = need;
    if (!need) return t;
    t = at::empty({int64_t(need)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, c10::DeviceIndex(device)));
  }
  p = t.data_ptr();
  return t;
}

// (cache, q, offsets, lengths, pages, scale, out, workspace) -> out
PyObject *kv8_attend(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_attend", n, 8)) throw PyError{};
    const Cache &held = cache_of(args[0]);
    const lmx_kv8_cache c = held.now();
    const at::Tensor &q = tensor("q", args[1]);
    const int type = type_of("q", q);
    const int64_t hd = int64_t(c.head_dim), rows = q.dim() == 3 ? q.size(0) : 0, heads = q.dim() == 3 ? q.size(1) : 0;
    const size_t qs = row_stride("q", q, q.scalar_type(), rows, heads, hd);
    const lmx_kv8_batch b = batch_of(args + 2, rows);
    double scale = 1.0 / std::sqrt(double(hd));
    if (args[5] != Py_None && (scale = PyFloat_AsDouble(args[5])) == -1.0 && PyErr_Occurred()) throw PyError{};
    const at::Tensor *given = args[6] != Py_None ? &tensor("out", args[6]) : nullptr;
    const size_t os = given ? row_stride("out", *given, q.scalar_type(), rows, heads, hd) : size_t(heads * hd);
    const int device = check_call(held, {&q, &THPVariable_Unpack(args[2]), &THPVariable_Unpack(args[3]), &THPVariable_Unpack(args[4]), given});
    at::Tensor out = given ? *given : at::empty({rows, heads, hd}, q.options());
    size_t need = 0, bytes = 0;
    check(lmx_kv8_attention_workspace(&c, &b, type, size_t(heads), &need));
    void *work;
    const at::Tensor w = workspace_of(args[7], need, device, work, bytes);
    check(lmx_kv8_attention(&c, &b, type, q.data_ptr(), qs, size_t(heads), float(scale), out.data_ptr(), os, work, bytes,
                            stream_on(device)));
    if (args[6] != Py_None) return Py_NewRef(args[6]);
    return THPVariable_Wrap(std::move(out));
  });
}

// (x, w, w_scale, bias, y, workspace) -> y
PyObject *linear_i8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("linear_i8", n, 6)) throw PyError{};
    const at::Tensor &x = tensor("x", args[0]), &w = tensor("w", args[1]), &scale = tensor("w_scale", args[2]);
    const int type = type_of("x", x);
    if (w.dim() != 2 || w.scalar_type() != at::kChar || w.stride(1) != 1) bad("w", w, "int8 [rows, cols] with neighbouring columns side by side");
    const int64_t rows = w.size(0), cols = w.size(1);
    if (x.dim() == 0 || x.size(-1) != cols || !x.is_contiguous()) bad("x", x, "contiguous, " + std::to_string(cols) + " values a row");
    if (scale.scalar_type() != at::kFloat || !has_sizes(scale, {rows}) || !scale.is_contiguous())
      bad("w_scale", scale, "contiguous float32 [" + std::to_string(rows) + "]");
    const at::Tensor *bias = args[3] != Py_None ? &tensor("bias", args[3]) : nullptr;
    if (bias && (bias->scalar_type() != x.scalar_type() || !has_sizes(*bias, {rows}) || !bias->is_contiguous()))
      bad("bias", *bias, std::string("contiguous ") + c10::toString(x.scalar_type()) + " [" + std::to_string(rows) + "]");
    const int64_t batch = cols ? x.numel() / cols : 0;
    const at::Tensor *given = args[4] != Py_None ? &tensor("y", args[4]) : nullptr;
    if (given && (given->scalar_type() != x.scalar_type() || given->numel() != batch * rows || !given->is_contiguous()))
      bad("y", *given, "contiguous, of x's type, " + std::to_string(batch) + " x " + std::to_string(rows));
    const int device = check_devices({&x, &w, &scale, bias, given});
    size_t need = 0, bytes = 0;
    check(lmx_linear_i8_workspace(size_t(rows), size_t(cols), size_t(batch), &need));
    at::Tensor y;
    if (given) {
      y = *given;
    } else {
      auto sizes = x.sizes().vec();
      sizes.back() = rows;
      y = at::empty(sizes, x.options());
    }
    void *work;
    const at::Tensor ws = workspace_of(args[5], need, device, work, bytes);
    // (the stride of a single row says nothing)
    check(lmx_linear_i8(static_cast<const int8_t *>(w.data_ptr()), size_t(rows > 1 ? w.stride(0) : (cols + 15) / 16 * 16),
                        static_cast<const float *>(scale.data_ptr()), bias ? bias->data_ptr() : nullptr, x.data_ptr(), y.data_ptr(), type, size_t(rows),
                        size_t(cols), size_t(batch), work, bytes, stream_on(device)));
    if (args[4] != Py_None) return Py_NewRef(args[4]);
    return THPVariable_Wrap(std::move(y));
  });
}

// (LmxError): set once by the package.
PyObject *set_error(PyObject *, PyObject *o) {
  Py_XDECREF(g_lmx_error);
  g_lmx_error = Py_NewRef(o);
  Py_RETURN_NONE;
}

#define LMX_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {LMX_FAST(kv8_cache), LMX_FAST(kv8_append), LMX_FAST(kv8_attend), LMX_FAST(linear_i8),
                           {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch", "The 8-bit serving operators on torch tensors.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch() { return PyModule_Create(&g_module); }
