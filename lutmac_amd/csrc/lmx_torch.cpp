// lmx_torch.cpp -- the serving operators on torch tensors: what lutmac_amd.kv8,
// linear_i8, linear_f8 and verify_drafts check of their arguments, the outputs and
// workspaces that they allocate, and their calls into the C ABI.
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
#include "lutmac_verify.h"

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

// A type as torch's users know it (the names inside torch are others).
const char *dtype_name(at::ScalarType t) {
  switch (t) {
  case at::kChar: return "int8";
  case at::kInt: return "int32";
  case at::kLong: return "int64";
  case at::kFloat: return "float32";
  case at::kFloat8_e4m3fn: return "float8_e4m3fn";
  default: return c10::toString(t);
  }
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

// What the two linear layers' arguments have in common: their sizes, the output.
struct Linear {
  const at::Tensor &x, &w, &scale;
  const at::Tensor *bias, *given;
  int type;
  int64_t rows, cols, batch;

  Linear(PyObject *const *args, at::ScalarType codes)
      : x(tensor("x", args[0])), w(tensor("w", args[1])), scale(tensor("w_scale", args[2])),
        bias(args[3] != Py_None ? &tensor("bias", args[3]) : nullptr), given(args[4] != Py_None ? &tensor("y", args[4]) : nullptr),
        type(type_of("x", x)) {
    if (w.dim() != 2 || w.scalar_type() != codes || w.stride(1) != 1)
      bad("w", w, std::string(dtype_name(codes)) + " [rows, cols] with neighbouring columns side by side");
    rows = w.size(0), cols = w.size(1);
    if (x.dim() == 0 || x.size(-1) != cols || !x.is_contiguous()) bad("x", x, "contiguous, " + std::to_string(cols) + " values a row");
  }
  void check_scale(at::IntArrayRef sizes) const {
    if (scale.scalar_type() != at::kFloat || !has_sizes(scale, sizes) || !scale.is_contiguous()) {
      std::string s;
      for (const int64_t n : sizes) s += (s.empty() ? "" : ", ") + std::to_string(n);
      bad("w_scale", scale, "contiguous float32 [" + s + "]");
    }
  }
  int check_rest() {   // -> the device
    if (bias && (bias->scalar_type() != x.scalar_type() || !has_sizes(*bias, {rows}) || !bias->is_contiguous()))
      bad("bias", *bias, std::string("contiguous ") + c10::toString(x.scalar_type()) + " [" + std::to_string(rows) + "]");
    batch = cols ? x.numel() / cols : 0;
    if (given && (given->scalar_type() != x.scalar_type() || given->numel() != batch * rows || !given->is_contiguous()))
      bad("y", *given, "contiguous, of x's type, " + std::to_string(batch) + " x " + std::to_string(rows));
    return check_devices({&x, &w, &scale, bias, given});
  }
  at::Tensor output() const {
    if (given) return *given;
    auto sizes = x.sizes().vec();
    sizes.back() = rows;
    return at::empty(sizes, x.options());
  }
  size_t stride() const { return size_t(rows > 1 ? w.stride(0) : (cols + 15) / 16 * 16); }   // (that of a single row says nothing)
  const float *scales() const { return static_cast<const float *>(scale.data_ptr()); }
  void *bias_pointer() const { return bias ? bias->data_ptr() : nullptr; }
};

// (x, w, w_scale, bias, y, workspace) -> y
PyObject *linear_i8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("linear_i8", n, 6)) throw PyError{};
    Linear l(args, at::kChar);
    l.check_scale({l.rows});
    const int device = l.check_rest();
    size_t need = 0, bytes = 0;
    check(lmx_linear_i8_workspace(size_t(l.rows), size_t(l.cols), size_t(l.batch), &need));
    at::Tensor y = l.output();
    void *work;
    const at::Tensor ws = workspace_of(args[5], need, device, work, bytes);
    check(lmx_linear_i8(static_cast<const int8_t *>(l.w.data_ptr()), l.stride(), l.scales(), l.bias_pointer(), l.x.data_ptr(), y.data_ptr(),
                        l.type, size_t(l.rows), size_t(l.cols), size_t(l.batch), work, bytes, stream_on(device)));
    if (l.given) return Py_NewRef(args[4]);
    return THPVariable_Wrap(std::move(y));
  });
}

// (x, w, w_scale, bias, y, workspace) -> y
PyObject *linear_f8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("linear_f8", n, 6)) throw PyError{};
    Linear l(args, at::kFloat8_e4m3fn);
    l.check_scale({(l.rows + 127) / 128, (l.cols + 127) / 128});
    const int device = l.check_rest();
    size_t need = 0, bytes = 0;
    check(lmx_linear_f8_workspace(size_t(l.rows), size_t(l.cols), size_t(l.batch), l.type, &need));
    at::Tensor y = l.output();
    void *work;
    const at::Tensor ws = workspace_of(args[5], need, device, work, bytes);
    check(lmx_linear_f8(static_cast<const uint8_t *>(l.w.data_ptr()), l.stride(), l.scales(), l.bias_pointer(), l.x.data_ptr(), y.data_ptr(),
                        l.type, size_t(l.rows), size_t(l.cols), size_t(l.batch), work, bytes, stream_on(device)));
    if (l.given) return Py_NewRef(args[4]);
    return THPVariable_Wrap(std::move(y));
  });
}

// ---- pages, rotation, verification ----

// A contiguous tensor of whole numbers.
const at::Tensor &whole(const char *name, PyObject *o, at::ScalarType type, at::IntArrayRef sizes) {
  const at::Tensor &t = tensor(name, o);
  if (t.scalar_type() != type || !has_sizes(t, sizes) || !t.is_contiguous()) {
    std::string s;
    for (const int64_t n : sizes) s += (s.empty() ? "" : ", ") + std::to_string(n);
    bad(name, t, std::string("contiguous ") + dtype_name(type) + " [" + s + "]");
  }
  return t;
}
template <class I>
I *pointer(const at::Tensor &t) { return static_cast<I *>(t.data_ptr()); }
at::Tensor int_tensor(int64_t n, int device) {
  return at::empty({n}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, c10::DeviceIndex(device)));
}

// (pages, lengths, free, n_free), checked but for their device.
lmx_kv8_pages pages_of(PyObject *const *args) {
  const at::Tensor &pages = tensor("pages", args[0]);
  if (pages.scalar_type() != at::kInt || pages.dim() != 2 || !pages.is_contiguous()) bad("pages", pages, "contiguous int32 of 2 dimensions");
  const at::Tensor &lengths = whole("lengths", args[1], at::kInt, {pages.size(0)});
  const at::Tensor &free = tensor("free", args[2]);
  if (free.scalar_type() != at::kInt || free.dim() != 1 || !free.is_contiguous()) bad("free", free, "contiguous int32 of 1 dimension");
  const at::Tensor &n_free = whole("n_free", args[3], at::kInt, {1});
  return {pointer<int32_t>(pages), pointer<int32_t>(lengths), pointer<int32_t>(free), pointer<int32_t>(n_free), size_t(pages.size(0)),
          size_t(pages.size(1)), size_t(free.size(0))};
}

// (pages, lengths, free, n_free): checked.
PyObject *kv8_pages(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_pages", n, 4)) throw PyError{};
    pages_of(args);
    for (int i = 1; i < 4; ++i)
      if (THPVariable_Unpack(args[i]).device() != THPVariable_Unpack(args[0]).device()) raise_value("the tensors of the pages must be on one device");
    Py_RETURN_NONE;
  });
}

// (pages, lengths, free, n_free, new, positions, slots, offsets, granted) -> (offsets, granted)
PyObject *kv8_extend(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_extend", n, 9)) throw PyError{};
    const lmx_kv8_pages p = pages_of(args);
    const int64_t seqs = int64_t(p.n_seqs);
    const at::Tensor &fresh = whole("new", args[4], at::kInt, {seqs});
    const at::Tensor &positions = tensor("positions", args[5]);
    if (positions.scalar_type() != at::kInt || positions.dim() != 1 || !positions.is_contiguous())
      bad("positions", positions, "contiguous int32 of 1 dimension");
    const at::Tensor *slots = args[6] != Py_None ? &whole("slots", args[6], at::kLong, {positions.size(0)}) : nullptr;
    const at::Tensor *off = args[7] != Py_None ? &whole("offsets", args[7], at::kInt, {seqs + 1}) : nullptr;
    const at::Tensor *yes = args[8] != Py_None ? &whole("granted", args[8], at::kInt, {seqs}) : nullptr;
    const int device = check_devices({&THPVariable_Unpack(args[0]), &THPVariable_Unpack(args[1]), &THPVariable_Unpack(args[2]),
                                      &THPVariable_Unpack(args[3]), &fresh, &positions, slots, off, yes});
    const at::Tensor offsets = off ? *off : int_tensor(seqs + 1, device), granted = yes ? *yes : int_tensor(seqs, device);
    check(lmx_kv8_extend(&p, pointer<int32_t>(fresh), size_t(positions.size(0)), pointer<int32_t>(offsets), pointer<int32_t>(granted),
                         pointer<int32_t>(positions), slots ? pointer<int64_t>(*slots) : nullptr, stream_on(device)));
    return Py_BuildValue("(NN)", off ? Py_NewRef(args[7]) : THPVariable_Wrap(offsets), yes ? Py_NewRef(args[8]) : THPVariable_Wrap(granted));
  });
}

// (pages, lengths, free, n_free, drop)
PyObject *kv8_trim(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("kv8_trim", n, 5)) throw PyError{};
    const lmx_kv8_pages p = pages_of(args);
    const at::Tensor &drop = whole("drop", args[4], at::kInt, {int64_t(p.n_seqs)});
    const int device = check_devices({&THPVariable_Unpack(args[0]), &THPVariable_Unpack(args[1]), &THPVariable_Unpack(args[2]),
                                      &THPVariable_Unpack(args[3]), &drop});
    check(lmx_kv8_trim(&p, pointer<int32_t>(drop), stream_on(device)));
    Py_RETURN_NONE;
  });
}

// (q, k, positions, rope, interleaved, inverse, q_out, k_out) -> (q_out, k_out)
PyObject *rotate(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("rotate", n, 8)) throw PyError{};
    const at::Tensor &q = tensor("q", args[0]);
    const int type = type_of("q", q);
    if (q.dim() != 3) bad("q", q, "[rows, heads, head_dim]");
    const at::ScalarType st = q.scalar_type();
    const int64_t rows = q.size(0), heads = q.size(1), hd = q.size(2);
    const at::Tensor *k = args[1] != Py_None ? &tensor("k", args[1]) : nullptr;
    const int64_t kv = k && k->dim() == 3 ? k->size(1) : 0;
    const size_t qs = row_stride("q", q, st, rows, heads, hd), ks = k ? row_stride("k", *k, st, rows, kv, hd) : 0;
    const at::Tensor &positions = whole("positions", args[2], at::kInt, {rows}), &rope = tensor("rope", args[3]);
    if (rope.scalar_type() != at::kFloat || rope.dim() != 3 || rope.size(2) != 2 || rope.size(1) < 1 || 2 * rope.size(1) > hd || !rope.is_contiguous())
      bad("rope", rope, "contiguous float32 [positions, 1.." + std::to_string(hd / 2) + ", 2]");
    const int interleaved = PyObject_IsTrue(args[4]), inverse = PyObject_IsTrue(args[5]);
    if (interleaved < 0 || inverse < 0) throw PyError{};
    const at::Tensor *qg = args[6] != Py_None ? &tensor("q_out", args[6]) : nullptr, *kg = args[7] != Py_None ? &tensor("k_out", args[7]) : nullptr;
    if (kg && !k) raise_value("k_out without k");
    const size_t qos = qg ? row_stride("q_out", *qg, st, rows, heads, hd) : size_t(heads * hd);
    const size_t kos = kg ? row_stride("k_out", *kg, st, rows, kv, hd) : size_t(kv * hd);
    const int device = check_devices({&q, k, &positions, &rope, qg, kg});
    const at::Tensor qo = qg ? *qg : at::empty({rows, heads, hd}, q.options());
    const at::Tensor ko = kg ? *kg : k ? at::empty({rows, kv, hd}, q.options()) : at::Tensor();
    check(lmx_rotary(type, q.data_ptr(), qs, qo.data_ptr(), qos, size_t(heads), k ? k->data_ptr() : nullptr, ks,
                     k ? ko.data_ptr() : nullptr, kos, size_t(kv), size_t(hd), size_t(2 * rope.size(1)), interleaved, inverse,
                     pointer<int32_t>(positions), size_t(rows), pointer<float>(rope), size_t(rope.size(0)), stream_on(device)));
    return Py_BuildValue("(NN)", qg ? Py_NewRef(args[6]) : THPVariable_Wrap(qo),
                         kg ? Py_NewRef(args[7]) : k ? THPVariable_Wrap(ko) : Py_NewRef(Py_None));
  });
}

// A matrix of `rows` rows of neighbouring elements: its row stride.
size_t matrix_stride(const char *name, const at::Tensor &t, int64_t rows, int64_t width) {
  if (!has_sizes(t, {rows, width})) bad(name, t, "[" + std::to_string(rows) + ", " + std::to_string(width) + "]");
  if (rows && width > 1 && t.stride(1) != 1) bad(name, t, "a row's elements side by side");
  return size_t(rows > 1 ? t.stride(0) : width);
}

// (logits, drafts, offsets, uniforms, probs, temperature, accepted, tokens, workspace) -> (accepted, tokens)
PyObject *verify_drafts(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (!arguments("verify_drafts", n, 9)) throw PyError{};
    const at::Tensor &logits = tensor("logits", args[0]);
    const int type = type_of("logits", logits);
    if (logits.dim() != 2) bad("logits", logits, "[rows, vocab]");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    const size_t stride = matrix_stride("logits", logits, rows, vocab);
    const at::Tensor &drafts = whole("drafts", args[1], at::kInt, {rows}), &offsets = tensor("offsets", args[2]);
    if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 || offsets.size(0) < 1 || !offsets.is_contiguous())
      bad("offsets", offsets, "contiguous int32 [sequences + 1]");
    const int64_t seqs = offsets.size(0) - 1;
    const at::Tensor &uniforms = whole("uniforms", args[3], at::kFloat, {rows, 2});
    const at::Tensor *probs = args[4] != Py_None ? &tensor("probs", args[4]) : nullptr;
    if (probs && probs->scalar_type() != at::kFloat) bad("probs", *probs, "float32");
    const size_t ps = probs ? matrix_stride("probs", *probs, rows, vocab) : 0;
    const at::Tensor *t = args[5] != Py_None ? &whole("temperature", args[5], at::kFloat, {seqs}) : nullptr;
    const at::Tensor *ag = args[6] != Py_None ? &whole("accepted", args[6], at::kInt, {seqs}) : nullptr;
    const at::Tensor *tg = args[7] != Py_None ? &whole("tokens", args[7], at::kInt, {rows}) : nullptr;
    const int device = check_devices({&logits, &drafts, &offsets, &uniforms, probs, t, ag, tg});
    const lmx_drafts d = {pointer<int32_t>(offsets), pointer<int32_t>(drafts), pointer<float>(uniforms), t ? pointer<float>(*t) : nullptr,
                          size_t(seqs), size_t(rows), size_t(vocab)};
    size_t need = 0, bytes = 0;
    check(lmx_verify_drafts_workspace(&d, type, &need));
    const at::Tensor accepted = ag ? *ag : int_tensor(seqs, device), tokens = tg ? *tg : int_tensor(rows, device);
    void *work;
    const at::Tensor ws = workspace_of(args[8], need, device, work, bytes);
    check(lmx_verify_drafts(&d, type, logits.data_ptr(), stride, probs ? pointer<float>(*probs) : nullptr, ps, pointer<int32_t>(accepted),
                            pointer<int32_t>(tokens), work, bytes, stream_on(device)));
    return Py_BuildValue("(NN)", ag ? Py_NewRef(args[6]) : THPVariable_Wrap(accepted), tg ? Py_NewRef(args[7]) : THPVariable_Wrap(tokens));
  });
}

// (LmxError): set once by the package.
PyObject *set_error(PyObject *, PyObject *o) {
  Py_XDECREF(g_lmx_error);
  g_lmx_error = Py_NewRef(o);
  Py_RETURN_NONE;
}

#define LMX_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {LMX_FAST(kv8_cache), LMX_FAST(kv8_append), LMX_FAST(kv8_attend), LMX_FAST(kv8_pages), LMX_FAST(kv8_extend),
                           LMX_FAST(kv8_trim), LMX_FAST(rotate), LMX_FAST(linear_i8), LMX_FAST(linear_f8), LMX_FAST(verify_drafts),
                           {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch", "The serving operators on torch tensors.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch() { return PyModule_Create(&g_module); }
