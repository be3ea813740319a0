// tensor_calls.cpp -- the C ABI's device calls on torch tensors.
//
// A call of the cache or of a 4-bit product costs the GPU a few microseconds, and
// Python's reading of the tensors (types, devices, strides, addresses), two
// allocations and a ctypes call cost as much again.  This module does that
// reading: each function checks its tensors, allocates what it returns and calls
// the C ABI (include/maxsim_hip.h) on the current stream.  It knows no kernels:
// the library's entry points are handed over when it is set up.
//
// Functions take a handle (a capsule) made by `cache` or `linear`, and return
// tensors.  ValueError, NotImplementedError and RuntimeError as elsewhere in the
// package.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstdlib>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/maxsim_hip.h"

namespace {

struct {
  const char* (*last_error)() = nullptr;
  decltype(&msim_kv4_append_async) append = nullptr;
  decltype(&msim_kv4_read_async) read = nullptr;
  decltype(&msim_kv4_attend_workspace) attend_workspace = nullptr;
  decltype(&msim_kv4_attend_async) attend = nullptr;
  decltype(&msim_linear4_async) linear = nullptr;
} abi;

struct Cache {
  msim_kv4_pool pool;
  at::Device device;
  at::Tensor tensors[4];  // key codes, key scales, value codes, value scales
};

struct Linear {
  at::Tensor codes, scales, bias;  // as the product reads them; bias may be undefined
  int64_t n, k, group;
};

template <typename T>
const char* handle_name();
template <>
const char* handle_name<Cache>() { return "maxsim_amd.cache"; }
template <>
const char* handle_name<Linear>() { return "maxsim_amd.linear"; }

template <typename T>
T* handle(PyObject* o) {
  T* h = static_cast<T*>(PyCapsule_GetPointer(o, handle_name<T>()));
  if (h == nullptr) throw python_error();
  return h;
}

template <typename T>
PyObject* make_handle(T* h) {
  return PyCapsule_New(h, handle_name<T>(), [](PyObject* o) {
    delete static_cast<T*>(PyCapsule_GetPointer(o, handle_name<T>()));
  });
}

void check(int status) {
  if (status == MSIM_OK) return;
  const char* message = abi.last_error();
  TORCH_CHECK_VALUE(status != MSIM_EINVAL, message);
  if (status == MSIM_ENOTSUP) TORCH_CHECK_NOT_IMPLEMENTED(false, message);
  TORCH_CHECK(false, message);
}

// A device made current, and its current stream.
struct Launch {
  c10::OptionalDeviceGuard guard;
  void* stream;
  explicit Launch(const at::Device& device) {
    if (c10::hip::current_device() != device.index()) guard.reset_device(device);
    stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  }
};

const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}

int type_of(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return MSIM_F32;
    case at::kHalf: return MSIM_F16;
    case at::kBFloat16: return MSIM_BF16;
    default: break;
  }
  TORCH_CHECK_VALUE(false, "dtype must be float32, float16 or bfloat16");
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

const at::Tensor& index_tensor(PyObject* o, const char* name, int64_t ndim, const at::Device& device) {
  const at::Tensor& t = tensor(o, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == ndim && t.device() == device, name,
                    " must be an int32 tensor of ", ndim, ndim > 1 ? " dimensions on " : " dimension on ", device);
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
  return t;
}

struct Batch {
  const int32_t *table, *lengths, *offsets;
  int64_t batch, max_pages, rows;
};

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

Batch read_batch(const Cache& c, PyObject* table, PyObject* lengths, PyObject* offsets, int64_t rows) {
  const at::Tensor& t = index_tensor(table, "page_table", 2, c.device);
  const at::Tensor& l = index_tensor(lengths, "lengths", 1, c.device);
  Batch b{ints(t), ints(l), nullptr, t.size(0), t.size(1), rows};
  TORCH_CHECK_VALUE(l.size(0) == b.batch, "lengths must have shape [batch]");
  if (offsets == Py_None) {
    TORCH_CHECK_VALUE(rows == b.batch, "without offsets there must be one row per sequence");
  } else {
    const at::Tensor& o = index_tensor(offsets, "offsets", 1, c.device);
    TORCH_CHECK_VALUE(o.size(0) == b.batch + 1, "offsets must have shape [batch + 1]");
    b.offsets = ints(o);
  }
  return b;
}

// Rows [rows, heads, head_dim] with any strides, dense in the last dimension;
// heads 0: any.
const at::Tensor& row_tensor(const Cache& c, PyObject* o, const char* name, int64_t heads) {
  const at::Tensor& t = tensor(o, name);
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == c.pool.dim && (heads == 0 || t.size(1) == heads), name,
                    " must be a tensor of shape [rows, ", heads == 0 ? std::string("heads") : std::to_string(heads), ", ",
                    c.pool.dim, "]");
  TORCH_CHECK_VALUE(t.device() == c.device, name, " must be on ", c.device);
  TORCH_CHECK_VALUE(t.stride(2) == 1 || t.numel() == 0, name, " must be dense in its last dimension");
  type_of(t.scalar_type());
  return t;
}

// First byte of a tensor's elements and the one behind its last (strides are not negative).
struct Span {
  uintptr_t first = 0, last = 0;
  explicit Span(const at::Tensor& t) {
    if (t.numel() == 0) return;
    int64_t most = 0;
    for (int64_t d = 0; d < t.dim(); ++d) most += (t.size(d) - 1) * t.stride(d);
    first = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    last = first + (most + 1) * t.element_size();
  }
  bool meets(const Span& o) const { return first < o.last && o.first < last; }
};

// Whether two tensors [rows, heads, dim] of one type share memory, other than an element
// with itself if `in_place`.  Views of one buffer may lie between each other: with equal
// strides the rows and heads that far apart are looked for, other strides count as shared.
bool share_memory(const at::Tensor& a, const at::Tensor& b, bool in_place) {
  if (!Span(a).meets(Span(b))) return false;
  int64_t step[2];
  for (int d = 0; d < 2; ++d) {
    step[d] = a.size(d) > 1 ? a.stride(d) : b.stride(d);
    if (b.size(d) > 1 && b.stride(d) != step[d]) return true;
  }
  const int64_t dim = a.size(2), size = a.element_size();
  const int64_t bytes = reinterpret_cast<intptr_t>(b.const_data_ptr()) - reinterpret_cast<intptr_t>(a.const_data_ptr());
  if (bytes % size != 0) return true;
  for (int64_t h = 1 - b.size(1); h < a.size(1); ++h) {
    const int64_t low = 1 - b.size(0), high = a.size(0) - 1;
    const int64_t away = bytes / size - h * step[1], near = step[0] > 0 ? away / step[0] : 0;
    const int64_t i0 = std::clamp(near, low, high);  // rows of that distance, or nearly
    for (int64_t i = std::max(low, i0 - 1); i <= std::min(high, i0 + 1); ++i)
      if (!(in_place && bytes == 0 && h == 0 && i == 0) && std::abs(i * step[0] - away) < dim) return true;
  }
  return false;
}

void check_output(const at::Tensor& t, const char* name) {
  // Heads within rows or rows within heads, which is what nearly all outputs are.
  auto nested = [&](int outer, int inner) {
    const int64_t piece = (t.size(inner) - 1) * t.stride(inner) + t.size(2);
    return (t.size(inner) <= 1 || t.stride(inner) >= t.size(2)) && (t.size(outer) <= 1 || t.stride(outer) >= piece);
  };
  TORCH_CHECK_VALUE(t.numel() == 0 || nested(0, 1) || nested(1, 0) || !share_memory(t, t, true), name,
                    " must not overlap itself");
}

void same_rows(const at::Tensor& k, const at::Tensor& v, const char* what) {
  TORCH_CHECK_VALUE(k.scalar_type() == v.scalar_type() && k.size(0) == v.size(0), what,
                    " must have the same shape and dtype");
}

void arguments(Py_ssize_t n, Py_ssize_t want) {
  TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n);
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* first = THPVariable_Wrap(a);
  PyObject* second = first ? THPVariable_Wrap(b) : nullptr;
  PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  if (both == nullptr) throw python_error();
  return both;
}

// setup(last_error, append, read, attend_workspace, attend, linear): addresses.
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  auto address = [&](int i) { return reinterpret_cast<void*>(integer(a[i])); };
  abi.last_error = reinterpret_cast<decltype(abi.last_error)>(address(0));
  abi.append = reinterpret_cast<decltype(abi.append)>(address(1));
  abi.read = reinterpret_cast<decltype(abi.read)>(address(2));
  abi.attend_workspace = reinterpret_cast<decltype(abi.attend_workspace)>(address(3));
  abi.attend = reinterpret_cast<decltype(abi.attend)>(address(4));
  abi.linear = reinterpret_cast<decltype(abi.linear)>(address(5));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// cache(k_codes, k_scales, v_codes, v_scales): a handle on the pool.
PyObject* make_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 4);
  const at::Tensor& codes = tensor(a[0], "k_codes");
  auto c = std::make_unique<Cache>(Cache{{}, codes.device(), {}});
  for (int i = 0; i < 4; ++i) {
    const at::Tensor& t = tensor(a[i], "the pool");
    TORCH_CHECK_VALUE(t.dim() == (i % 2 ? 3 : 4) && t.is_contiguous() && t.device() == c->device &&
                          t.scalar_type() == (i % 2 ? at::kFloat : at::kByte) && t.sizes().slice(0, 3) == codes.sizes().slice(0, 3),
                      "the pool's tensors must be dense and of one shape");
    c->tensors[i] = t;
  }
  c->pool = msim_kv4_pool{static_cast<uint8_t*>(c->tensors[0].data_ptr()), static_cast<float*>(c->tensors[1].data_ptr()),
                          static_cast<uint8_t*>(c->tensors[2].data_ptr()), static_cast<float*>(c->tensors[3].data_ptr()),
                          codes.size(0), (int32_t)codes.size(1), (int32_t)codes.size(2), (int32_t)(codes.size(3) * 2)};
  return make_handle(c.release());
  END_HANDLE_TH_ERRORS
}

// append(cache, k, v, page_table, lengths, offsets)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  const Cache& c = *handle<Cache>(a[0]);
  const at::Tensor& k = row_tensor(c, a[1], "k", c.pool.kv_heads);
  const at::Tensor& v = row_tensor(c, a[2], "v", c.pool.kv_heads);
  same_rows(k, v, "k and v");
  const Batch b = read_batch(c, a[3], a[4], a[5], k.size(0));
  const Launch launch(c.device);
  check(abi.append(&c.pool, b.table, b.lengths, b.offsets, b.batch, b.max_pages, b.rows, k.const_data_ptr(), k.stride(0),
                   k.stride(1), v.const_data_ptr(), v.stride(0), v.stride(1), type_of(k.scalar_type()), launch.stream));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// read(cache, page_table, lengths, offsets, rows, type, k, v): k and v None are
// allocated, [rows, kv_heads, head_dim] of C ABI type `type`.
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 8);
  const Cache& c = *handle<Cache>(a[0]);
  at::Tensor k, v;
  if (a[6] == Py_None) {
    const int64_t rows = integer(a[4]), type = integer(a[5]);
    TORCH_CHECK_VALUE(rows >= 0, "rows must not be negative");
    const auto options = at::TensorOptions().device(c.device).dtype(
        type == MSIM_F32 ? at::kFloat : (type == MSIM_F16 ? at::kHalf : at::kBFloat16));
    k = at::empty({rows, c.pool.kv_heads, c.pool.dim}, options);
    v = at::empty({rows, c.pool.kv_heads, c.pool.dim}, options);
  } else {
    k = row_tensor(c, a[6], "out[0]", c.pool.kv_heads);
    v = row_tensor(c, a[7], "out[1]", c.pool.kv_heads);
    same_rows(k, v, "both outputs");
    check_output(k, "out[0]");
    check_output(v, "out[1]");
    TORCH_CHECK_VALUE(!share_memory(k, v, false), "out[0] and out[1] must not overlap");
  }
  const Batch b = read_batch(c, a[1], a[2], a[3], k.size(0));
  const Launch launch(c.device);
  check(abi.read(&c.pool, b.table, b.lengths, b.offsets, b.batch, b.max_pages, b.rows, k.data_ptr(), k.stride(0),
                 k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), type_of(k.scalar_type()), launch.stream));
  return pair(k, v);
  END_HANDLE_TH_ERRORS
}

// attend(cache, q, page_table, lengths, offsets, scale, causal, window, mask, out, return_lse)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  const Cache& c = *handle<Cache>(a[0]);
  const at::Tensor& q = row_tensor(c, a[1], "q", 0);
  const int64_t rows = q.size(0), heads = q.size(1);
  TORCH_CHECK_VALUE(heads >= 1 && heads % c.pool.kv_heads == 0, "heads must be a multiple of kv_heads");
  const Batch b = read_batch(c, a[2], a[3], a[4], rows);
  const double scale = PyFloat_AsDouble(a[5]);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  const int causal = PyObject_IsTrue(a[6]);
  if (causal < 0) throw python_error();
  const uint8_t* mask = nullptr;
  int64_t mask_stride = 0, mask_width = 0;
  if (a[8] != Py_None) {
    const at::Tensor& m = tensor(a[8], "mask");
    TORCH_CHECK_VALUE(m.scalar_type() == at::kBool && m.dim() == 2 && m.size(0) == rows && m.device() == c.device,
                      "mask must be a bool tensor of shape [rows, width] on ", c.device);
    TORCH_CHECK_VALUE(m.size(1) <= 1 || m.stride(1) == 1, "mask must be dense in its last dimension");
    mask_stride = m.stride(0);
    mask_width = m.size(1);
    // An empty mask has no memory: it hides every key all the same.
    mask = mask_width > 0 ? static_cast<const uint8_t*>(m.const_data_ptr()) : c.pool.k_codes;
  }
  at::Tensor out, lse, work;
  if (a[9] == Py_None) {
    out = at::empty({rows, heads, c.pool.dim}, q.options().requires_grad(false));
  } else {
    out = row_tensor(c, a[9], "out", heads);
    TORCH_CHECK_VALUE(out.scalar_type() == q.scalar_type() && out.size(0) == rows, "out must have q's shape and dtype");
    check_output(out, "out");
    // In place of q is fine: a workgroup writes rows that it alone read, or the join does.
    TORCH_CHECK_VALUE(!share_memory(out, q, true), "out must not overlap q, unless it is q");
  }
  const bool want_lse = a[10] == Py_True;
  if (want_lse) lse = at::empty({rows, heads}, at::TensorOptions().device(c.device).dtype(at::kFloat));
  const Launch launch(c.device);
  uint64_t need = 0;
  check(abi.attend_workspace(&c.pool, b.batch, b.max_pages, rows, heads, &need));
  if (need > 0) work = at::empty({(int64_t)need}, at::TensorOptions().device(c.device).dtype(at::kByte));
  check(abi.attend(&c.pool, b.table, b.lengths, b.offsets, b.batch, b.max_pages, rows, q.const_data_ptr(), q.stride(0),
                   q.stride(1), heads, type_of(q.scalar_type()), scale, causal, integer(a[7]), mask, mask_stride,
                   mask_width, out.data_ptr(), out.stride(0), out.stride(1),
                   want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, need > 0 ? work.data_ptr() : nullptr, need,
                   launch.stream));
  return want_lse ? pair(out, lse) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// linear(codes, scales, bias, n, k, group): a handle on a laid-out matrix.
PyObject* make_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  auto h = std::make_unique<Linear>();
  h->codes = tensor(a[0], "codes");
  h->scales = tensor(a[1], "scales");
  if (a[2] != Py_None) h->bias = tensor(a[2], "bias");
  h->n = integer(a[3]);
  h->k = integer(a[4]);
  h->group = integer(a[5]);
  return make_handle(h.release());
  END_HANDLE_TH_ERRORS
}

// multiply(linear, x, out): x [..., k] to [..., n].
PyObject* multiply(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 3);
  const Linear& w = *handle<Linear>(a[0]);
  const at::Tensor& x = tensor(a[1], "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == w.k, "x must be a tensor of shape [..., ", w.k, "]");
  TORCH_CHECK_VALUE(x.device() == w.codes.device(), "x must be on ", w.codes.device());
  const int type = type_of(x.scalar_type());
  at::Tensor rows;  // x as a dense-rowed matrix, where it is none
  const at::Tensor* m = &x;
  if (x.dim() != 2 || x.stride(1) != 1) {
    rows = x.detach().reshape({-1, w.k});
    if (rows.stride(1) != 1) rows = rows.contiguous();
    m = &rows;
  }
  at::DimVector sizes(x.sizes());
  sizes.back() = w.n;
  at::Tensor out;
  if (a[2] == Py_None) {
    out = at::empty(sizes, x.options().requires_grad(false));
  } else {
    out = tensor(a[2], "out");
    TORCH_CHECK_VALUE(out.sizes() == at::IntArrayRef(sizes) && out.scalar_type() == x.scalar_type() &&
                          out.device() == x.device() && out.is_contiguous(),
                      "out must be a contiguous tensor of the result's shape, x's dtype and device");
    // Out is one piece of memory: it meets x where it meets one of x's rows.
    const Span to(out), from(*m);
    bool meets = to.meets(from);
    if (meets && m->size(0) > 1 && m->stride(0) > 0) {
      const int64_t step = m->stride(0) * x.element_size(), bytes = w.k * x.element_size();
      // The first row that ends behind out's start.
      const int64_t before = (int64_t)(to.first - from.first) - bytes;
      const int64_t row = to.first < from.first + bytes ? 0 : before / step + 1;
      meets = row < m->size(0) && from.first + row * step < to.last;
    }
    TORCH_CHECK_VALUE(!meets, "out must not overlap x");
  }
  const Launch launch(x.device());
  check(abi.linear(static_cast<const uint8_t*>(w.codes.const_data_ptr()),
                   static_cast<const uint16_t*>(w.scales.const_data_ptr()), w.n, w.k, w.group,
                   w.bias.defined() ? static_cast<const float*>(w.bias.const_data_ptr()) : nullptr, m->const_data_ptr(),
                   m->size(0), m->stride(0), type, out.data_ptr(), w.n, launch.stream));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define CALL(name, function) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    CALL("setup", setup),   CALL("cache", make_cache),   CALL("append", append),     CALL("read", read),
    CALL("attend", attend), CALL("linear", make_linear), CALL("multiply", multiply), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls() { return PyModule_Create(&module); }
