// Native forms of the hottest launchers of row_kernels.py, as a CPython
// module (_launch), and held_state, a check that a decode step makes.
//
// A launcher called from Python costs more than its kernel at small sizes:
// 7 to 16 us of attribute reads, checks, tensor allocations and a ctypes
// call, against 2 to 8 us of kernel. Here the operands are checked and the
// outputs allocated on at::Tensor, and the library is called directly.
//
// Each launcher takes a well-formed call only: it returns None, with nothing
// launched or changed, as soon as an operand is anything but what
// row_kernels.py would accept as it stands, and the Python launcher then
// handles the call (it raises, converts or allocates as it always did). A
// failed launch raises the RuntimeError of _hip.check. The GIL is released
// around allocation and launch, as torch and ctypes do.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <new>
#include <stdexcept>
#include <utility>
#include <vector>

#include "nhs.h"

namespace {

using at::Tensor;

struct Skip {};  // not a call for the native path

void need(bool ok) {
  if (!ok) throw Skip();
}

const Tensor& tensor(PyObject* o) {
  need(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  need(PyLong_CheckExact(o));
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Skip();
  }
  return v;
}

int32_t integer32(PyObject* o) {
  const int64_t v = integer(o);
  need(v >= INT32_MIN && v <= INT32_MAX);
  return (int32_t)v;
}

bool truth(PyObject* o) {
  need(o == Py_True || o == Py_False);
  return o == Py_True;
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return NHS_F32;
    case at::kHalf: return NHS_F16;
    case at::kBFloat16: return NHS_BF16;
    default: throw Skip();
  }
}

bool is_half(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// Plain strided GPU tensor with elements, sizes that fit the library's 32-bit arguments.
void on_gpu(const Tensor& t, int64_t dim) {
  need(t.is_cuda() && t.layout() == at::kStrided && t.dim() == dim && t.numel() > 0 && !t.is_neg());
  for (int64_t s : t.sizes()) need(s <= INT32_MAX);
}

void on_gpu(const Tensor& t, int64_t dim, const Tensor& other) {
  on_gpu(t, dim);
  need(t.device() == other.device());
}

bool same_sizes(const Tensor& t, at::IntArrayRef sizes) { return t.sizes() == sizes; }

// Whether dimensions from `first` on are laid out contiguously.
bool contiguous_from(const Tensor& t, int64_t first) {
  int64_t expected = 1;
  for (int64_t d = t.dim() - 1; d >= first; --d) {
    if (t.size(d) != 1 && t.stride(d) != expected) return false;
    expected *= t.size(d);
  }
  return true;
}

Tensor make(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Bytes between the blocks of a pool [blocks, 2, P, Hkv, D].
int64_t pool_block_stride(const Tensor& pool) {
  const int64_t P = pool.size(2), H = pool.size(3), D = pool.size(4);
  need(pool.size(1) == 2 && pool.stride(1) == P * H * D && pool.stride(2) == H * D && pool.stride(3) == D &&
       pool.stride(4) == 1 && pool.stride(0) >= 2 * P * H * D);
  return pool.stride(0) * pool.element_size();
}

// lengths as row_kernels._lengths_arg would pass them on unchanged
struct Lengths {
  const int64_t* per_item = nullptr;
  int64_t all = 0;
};
Lengths lengths_of(PyObject* o, int64_t batch, const Tensor& other) {
  Lengths l;
  if (PyLong_CheckExact(o)) {
    l.all = integer(o);
  } else {
    const Tensor& t = tensor(o);
    on_gpu(t, 1, other);
    need(t.scalar_type() == at::kLong && t.size(0) == batch && t.is_contiguous());
    l.per_item = static_cast<const int64_t*>(t.data_ptr());
  }
  return l;
}

PyObject* failed(const char* what, int status) {
  return PyErr_Format(PyExc_RuntimeError, "%s failed with status %d: %s", what, status, nhs_last_error());
}

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// Runs `body`; Skip and anything torch raises on an odd tensor leave the call to the Python launcher.
template <typename F>
PyObject* native(Py_ssize_t nargs, Py_ssize_t wanted, F body) {
  if (nargs != wanted) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return body();
  } catch (const Skip&) {
  } catch (const std::exception&) {
  }
  Py_RETURN_NONE;
}

PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* result = PyTuple_New((Py_ssize_t)tensors.size());
  if (!result) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* item;
    if (t.defined()) {
      item = THPVariable_Wrap(t);
    } else {
      item = Py_None;
      Py_INCREF(item);
    }
    if (!item) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i++, item);
  }
  return result;
}

// ---- decode linear layers -----------------------------------------------------------------

void check_linear(const Tensor& x, const Tensor& w) {
  on_gpu(x, 2);
  on_gpu(w, 2, x);
  need(is_half(x) && w.scalar_type() == x.scalar_type() && x.size(1) == w.size(1) && x.stride(1) == 1 &&
       w.stride(1) == 1);
}

const void* bias_of(PyObject* o, const Tensor& x, int64_t n) {
  if (o == Py_None) return nullptr;
  const Tensor& b = tensor(o);
  on_gpu(b, 1, x);
  need(b.size(0) == n && b.scalar_type() == x.scalar_type() && b.is_contiguous());
  return b.data_ptr();
}

PyObject* linear_small_m(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 4, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &w = tensor(a[1]);
    check_linear(x, w);
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    const void* bias = bias_of(a[2], x, n);
    Tensor out;
    if (a[3] != Py_None) {
      out = tensor(a[3]);
      on_gpu(out, 2, x);
      need(out.size(0) == m && out.size(1) == n && out.scalar_type() == x.scalar_type() && out.stride(1) == 1);
    }
    int st;
    {
      NoGil free;
      if (!out.defined()) out = make({m, n}, x, x.scalar_type());
      st = nhs_linear_small_m(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), bias, dtype_code(x), (int32_t)m,
                              (int32_t)n, (int32_t)k, out.data_ptr(), out.stride(0), stream_of(x));
    }
    return st ? failed("nhs_linear_small_m", st) : THPVariable_Wrap(out);
  });
}

PyObject* linear_silu_mul(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 2, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &w = tensor(a[1]);
    check_linear(x, w);
    need(w.size(0) % 2 == 0);
    const int64_t m = x.size(0), inter = w.size(0) / 2;
    Tensor out;
    int st;
    {
      NoGil free;
      out = make({m, inter}, x, x.scalar_type());
      st = nhs_linear_silu_mul(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), dtype_code(x), (int32_t)m,
                               (int32_t)inter, (int32_t)x.size(1), out.data_ptr(), out.stride(0), stream_of(x));
    }
    return st ? failed("nhs_linear_silu_mul", st) : THPVariable_Wrap(out);
  });
}

PyObject* linear_rope(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 7, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &w = tensor(a[1]), &cos = tensor(a[5]), &sin = tensor(a[6]);
    check_linear(x, w);
    const int64_t m = x.size(0), n = w.size(0);
    const void* bias = bias_of(a[2], x, n);
    const int32_t heads = integer32(a[3]), dim = integer32(a[4]);
    for (const Tensor* t : {&cos, &sin}) {
      on_gpu(*t, 2, x);
      need(t->size(0) == m && t->size(1) == dim / 2 && t->scalar_type() == x.scalar_type() && t->is_contiguous());
    }
    Tensor out;
    int st;
    {
      NoGil free;
      out = make({m, n}, x, x.scalar_type());
      st = nhs_linear_rope(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), bias, dtype_code(x), (int32_t)m,
                           (int32_t)n, (int32_t)x.size(1), dim, heads, cos.data_ptr(), sin.data_ptr(), out.data_ptr(),
                           out.stride(0), stream_of(x));
    }
    return st ? failed("nhs_linear_rope", st) : THPVariable_Wrap(out);
  });
}

PyObject* add_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 5, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &w = tensor(a[2]);
    on_gpu(x, 2);
    on_gpu(w, 1, x);
    need(x.is_contiguous() && w.size(0) == x.size(1) && w.scalar_type() == x.scalar_type() && w.is_contiguous());
    const void* delta = nullptr;
    if (a[1] != Py_None) {
      const Tensor& d = tensor(a[1]);
      on_gpu(d, 2, x);
      need(same_sizes(d, x.sizes()) && d.scalar_type() == x.scalar_type() && d.is_contiguous());
      delta = d.data_ptr();
    }
    need(PyFloat_CheckExact(a[3]));
    const float eps = (float)PyFloat_AS_DOUBLE(a[3]);
    const bool write_back = truth(a[4]);
    const int code = dtype_code(x);
    Tensor out;
    int st;
    {
      NoGil free;
      out = make(x.sizes(), x, x.scalar_type());
      st = nhs_add_rmsnorm((int32_t)x.size(0), (int32_t)x.size(1), code, x.data_ptr(), delta, write_back,
                           w.data_ptr(), eps, out.data_ptr(), stream_of(x));
    }
    return st ? failed("nhs_add_rmsnorm", st) : THPVariable_Wrap(out);
  });
}

// ---- attention ------------------------------------------------------------------------------

// workspace: a tensor, or the dict (device index, stream) -> tensor of row_kernels.attend_workspace
PyObject* attend_batched(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 6, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &pool = tensor(a[1]), &rows = tensor(a[2]);
    on_gpu(q, 3);
    on_gpu(pool, 5, q);
    need(rows.dim() == 2 || rows.dim() == 3);
    on_gpu(rows, rows.dim(), q);
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = pool.size(3), n = rows.size(-1);
    const int32_t P = integer32(a[3]);
    need(rows.scalar_type() == at::kLong && pool.size(4) == D && pool.size(2) == P && Hq % Hkv == 0 &&
         q.stride(2) == 1 && rows.size(0) == B && (rows.dim() == 2 || rows.size(1) == Hq) &&
         pool.size(0) * P < (int64_t(1) << 31));
    const int64_t stride = pool_block_stride(pool);
    const int q_code = dtype_code(q), kv_code = dtype_code(pool);
    void* const stream = stream_of(q);
    const int64_t bytes = nhs_attend_workspace_bytes((int32_t)B, (int32_t)Hq, (int32_t)D, (int32_t)n);
    PyObject* held = a[5];
    if (PyDict_CheckExact(held)) {
      PyObject* key = Py_BuildValue("(iK)", (int)q.device().index(), (unsigned long long)(uintptr_t)stream);
      if (!key) return nullptr;
      held = PyDict_GetItemWithError(a[5], key);  // borrowed; the tensor below shares ownership
      Py_DECREF(key);
      if (!held && PyErr_Occurred()) return nullptr;
      need(held != nullptr);
    }
    const Tensor ws = tensor(held);
    need(ws.device() == q.device() && (int64_t)ws.numel() * (int64_t)ws.element_size() >= bytes);
    Tensor out;
    if (a[4] != Py_None) {
      out = tensor(a[4]);
      on_gpu(out, 3, q);
      need(same_sizes(out, q.sizes()) && out.scalar_type() == q.scalar_type() && out.stride(2) == 1);
    }
    int st;
    {
      NoGil free;
      if (!out.defined()) out = make({B, Hq, D}, q, q.scalar_type());
      st = nhs_attend_rows(q.data_ptr(), q_code, q.stride(0), q.stride(1), pool.data_ptr(), kv_code, stride,
                           static_cast<const int64_t*>(rows.data_ptr()), rows.stride(0),
                           rows.dim() == 3 ? rows.stride(1) : 0, rows.stride(-1), (int32_t)B, (int32_t)n, (int32_t)Hq,
                           (int32_t)Hkv, (int32_t)D, P, out.data_ptr(), out.stride(0), out.stride(1), ws.data_ptr(),
                           (int64_t)ws.numel() * (int64_t)ws.element_size(), stream);
    }
    return st ? failed("nhs_attend_rows", st) : THPVariable_Wrap(out);
  });
}

PyObject* prefill_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 4, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    on_gpu(q, 3);
    on_gpu(k, 3, q);
    on_gpu(v, 3, q);
    need(is_half(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
         same_sizes(v, k.sizes()) && k.size(0) == q.size(0) && k.size(2) == q.size(2) && q.stride(2) == 1 &&
         k.stride(2) == 1 && v.stride(2) == 1);
    Tensor out;
    if (a[3] != Py_None) {
      out = tensor(a[3]);
      on_gpu(out, 3, q);
      need(same_sizes(out, q.sizes()) && out.scalar_type() == q.scalar_type() && out.stride(2) == 1);
    }
    int st;
    {
      NoGil free;
      if (!out.defined()) out = make(q.sizes(), q, q.scalar_type());
      st = nhs_prefill_attention(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                                 v.data_ptr(), v.stride(0), v.stride(1), dtype_code(q), (int32_t)q.size(0),
                                 (int32_t)q.size(1), (int32_t)k.size(1), (int32_t)q.size(2), out.data_ptr(),
                                 out.stride(0), out.stride(1), stream_of(q));
    }
    return st ? failed("nhs_prefill_attention", st) : THPVariable_Wrap(out);
  });
}

// ---- drafted tokens ---------------------------------------------------------------------------

// Makes t's device current for the launches that follow, as row_kernels._on does.
struct OnDevice {
  c10::DeviceGuard guard;
  explicit OnDevice(const Tensor& t) : guard(t.device()) {}
};

// A caller's output: a strided tensor whose heads are contiguous and whose elements are distinct (or Skip).
void check_out(const Tensor& out, const Tensor& like) {
  on_gpu(out, like.dim(), like);
  need(same_sizes(out, like.sizes()) && out.scalar_type() == like.scalar_type() && out.stride(-1) == 1);
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < out.dim(); ++d)
    if (out.size(d) > 1) dims.emplace_back(out.stride(d), out.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;  // elements that the dimensions of smaller strides reach over
  for (const auto& [stride, size] : dims) {
    need(stride >= span);
    span += stride * (size - 1);
  }
}

// Scratch memory of a call (nothing for 0 bytes): on the current stream's allocator, freed with the tensor.
Tensor scratch(int64_t bytes, const Tensor& like) { return bytes ? make({bytes}, like, at::kByte) : Tensor(); }
void* scratch_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject* tree_plan(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 2, [&]() -> PyObject* {
    const Tensor &parents = tensor(a[0]), &lengths = tensor(a[1]);
    on_gpu(parents, 2);
    on_gpu(lengths, 1, parents);
    const int64_t B = parents.size(0), T = parents.size(1);
    need(parents.scalar_type() == at::kInt && parents.stride(1) == 1 && lengths.scalar_type() == at::kLong &&
         lengths.size(0) == B && lengths.is_contiguous() && T <= NHS_MAX_TREE_NODES);
    Tensor mask, positions;
    int st;
    {
      NoGil free;
      const OnDevice on(parents);
      mask = make({B, T}, parents, at::kLong);
      positions = make({B, T}, parents, at::kLong);
      st = nhs_tree_plan((int32_t)B, (int32_t)T, static_cast<const int32_t*>(parents.data_ptr()), parents.stride(0),
                         static_cast<const int64_t*>(lengths.data_ptr()), static_cast<int64_t*>(mask.data_ptr()),
                         static_cast<int64_t*>(positions.data_ptr()), stream_of(parents));
    }
    return st ? failed("nhs_tree_plan", st) : tuple_of({mask, positions});
  });
}

PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 8, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &pool = tensor(a[1]), &rows = tensor(a[2]), &k = tensor(a[3]), &v = tensor(a[4]),
                 &mask = tensor(a[5]);
    on_gpu(q, 4);
    on_gpu(pool, 5, q);
    on_gpu(rows, 2, q);
    on_gpu(k, 4, q);
    on_gpu(v, 4, q);
    on_gpu(mask, 2, q);
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = pool.size(3), N = rows.size(1);
    const int32_t P = integer32(a[6]);
    const int code = dtype_code(q);
    need(same_sizes(v, k.sizes()) && k.size(0) == B && k.size(1) == T && k.size(2) == Hkv && k.size(3) == D &&
         pool.size(2) == P && pool.size(4) == D && Hq % Hkv == 0 && pool.scalar_type() == q.scalar_type() &&
         k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && rows.size(0) == B &&
         rows.scalar_type() == at::kLong && mask.size(0) == B && mask.size(1) == T && mask.stride(1) == 1 &&
         mask.scalar_type() == at::kLong && q.stride(3) == 1 && k.stride(3) == 1 && v.stride(3) == 1 &&
         T <= NHS_MAX_TREE_NODES && D <= NHS_MAX_TREE_HEAD_DIM && N <= (1 << 30) && pool.size(0) * P < (int64_t(1) << 31));
    const int64_t stride = pool_block_stride(pool);
    Tensor out;
    if (a[7] != Py_None) {
      out = tensor(a[7]);
      check_out(out, q);
    }
    int st;
    {
      NoGil free;
      const OnDevice on(q);
      if (!out.defined()) out = make(q.sizes(), q, q.scalar_type());
      const int64_t bytes = nhs_tree_attention_workspace_bytes((int32_t)B, (int32_t)T, (int32_t)N, (int32_t)Hq,
                                                               (int32_t)Hkv, (int32_t)D);
      const Tensor ws = scratch(bytes, q);
      st = nhs_tree_attention(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), k.stride(0),
                              k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
                              static_cast<const int64_t*>(mask.data_ptr()), mask.stride(0), code, pool.data_ptr(),
                              pool.size(0) * P, stride, static_cast<const int64_t*>(rows.data_ptr()), rows.stride(0),
                              rows.stride(1), (int32_t)B, (int32_t)T, (int32_t)N, (int32_t)Hq, (int32_t)Hkv,
                              (int32_t)D, P, out.data_ptr(), out.stride(0), out.stride(1), out.stride(2),
                              scratch_ptr(ws), bytes, stream_of(q));
    }
    return st ? failed("nhs_tree_attention", st) : THPVariable_Wrap(out);
  });
}

PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 9, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &k = tensor(a[1]), &qw = tensor(a[2]), &kw = tensor(a[3]), &cos = tensor(a[5]),
                 &sin = tensor(a[6]);
    on_gpu(q, 3);
    on_gpu(k, 3, q);
    const int64_t n = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(1);
    need(k.size(0) == n && k.size(2) == D && k.scalar_type() == q.scalar_type() && D % 2 == 0 && q.stride(2) == 1 &&
         k.stride(2) == 1);
    for (const Tensor* w : {&qw, &kw}) {
      on_gpu(*w, 1, q);
      need(w->size(0) == D && w->scalar_type() == q.scalar_type() && w->is_contiguous());
    }
    for (const Tensor* t : {&cos, &sin}) {
      on_gpu(*t, 2, q);
      need(t->size(1) == D / 2 && t->is_contiguous());
    }
    need(same_sizes(sin, cos.sizes()) && sin.scalar_type() == cos.scalar_type() &&
         (cos.scalar_type() == q.scalar_type() || cos.scalar_type() == at::kFloat));
    need(PyFloat_CheckExact(a[4]));
    const float eps = (float)PyFloat_AS_DOUBLE(a[4]);
    const int64_t* positions = nullptr;
    if (a[7] != Py_None) {
      const Tensor& p = tensor(a[7]);
      on_gpu(p, 1, q);
      need(p.size(0) == n && p.scalar_type() == at::kLong && p.is_contiguous());
      positions = static_cast<const int64_t*>(p.data_ptr());
    } else {
      need(cos.size(0) >= n);
    }
    const int code = dtype_code(q), table_code = dtype_code(cos);
    Tensor q_out, k_out;
    if (a[8] != Py_None) {
      need(PyTuple_CheckExact(a[8]) && PyTuple_GET_SIZE(a[8]) == 2);
      q_out = tensor(PyTuple_GET_ITEM(a[8], 0));
      k_out = tensor(PyTuple_GET_ITEM(a[8], 1));
      check_out(q_out, q);
      check_out(k_out, k);
      need(q_out.data_ptr() != k_out.data_ptr());
    }
    int st;
    {
      NoGil free;
      const OnDevice on(q);
      if (!q_out.defined()) {
        q_out = make(q.sizes(), q, q.scalar_type());
        k_out = make(k.sizes(), k, k.scalar_type());
      }
      st = nhs_qk_norm_rope((int32_t)n, (int32_t)Hq, (int32_t)Hkv, (int32_t)D, code, q.data_ptr(), q.stride(0),
                            q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), qw.data_ptr(), kw.data_ptr(), eps,
                            cos.data_ptr(), sin.data_ptr(), table_code, cos.size(0), positions, q_out.data_ptr(),
                            q_out.stride(0), q_out.stride(1), k_out.data_ptr(), k_out.stride(0), k_out.stride(1),
                            stream_of(q));
    }
    return st ? failed("nhs_qk_norm_rope", st) : tuple_of({q_out, k_out});
  });
}

PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 3, [&]() -> PyObject* {
    const Tensor &logits = tensor(a[0]), &tokens = tensor(a[1]);
    on_gpu(logits, 2);
    need(tokens.dim() == 1 || tokens.dim() == 2);
    on_gpu(tokens, tokens.dim(), logits);
    const int64_t R = logits.size(0), V = logits.size(1), per_row = tokens.dim() == 2 ? tokens.size(1) : 1;
    const int32_t top = integer32(a[2]);
    const int code = dtype_code(logits);
    need(logits.stride(1) == 1 && tokens.size(0) == R && tokens.scalar_type() == at::kLong && tokens.is_contiguous() &&
         top >= 0 && top <= NHS_MAX_TOP_LOGPROBS && top <= V && V <= (1 << 30));
    Tensor logprobs, entropy, ids, values;
    int st;
    {
      NoGil free;
      const OnDevice on(logits);
      logprobs = make(tokens.sizes(), logits, at::kFloat);
      entropy = make({R}, logits, at::kFloat);
      ids = make({R, top}, logits, at::kLong);
      values = make({R, top}, logits, at::kFloat);
      const int64_t bytes = nhs_token_logprobs_workspace_bytes((int32_t)R, (int32_t)V, code, top);
      const Tensor ws = scratch(bytes, logits);
      st = nhs_token_logprobs(logits.data_ptr(), logits.stride(0), code, (int32_t)R, (int32_t)V,
                              static_cast<const int64_t*>(tokens.data_ptr()), per_row, (int32_t)per_row, top,
                              static_cast<float*>(logprobs.data_ptr()), static_cast<float*>(entropy.data_ptr()),
                              static_cast<int64_t*>(ids.data_ptr()), static_cast<float*>(values.data_ptr()),
                              scratch_ptr(ws), bytes, stream_of(logits));
    }
    return st ? failed("nhs_token_logprobs", st) : tuple_of({logprobs, entropy, ids, values});
  });
}

// ---- selection --------------------------------------------------------------------------------

struct Selection {
  Tensor pages, positions;
  void allocate(int64_t B, int64_t top, int64_t P, const Tensor& like) {
    pages = make({B, top}, like, at::kInt);
    positions = make({B, top * P}, like, at::kInt);
  }
};

PyObject* quest_batched(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 8, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &lo = tensor(a[1]), &hi = tensor(a[2]);
    on_gpu(q, 3);
    on_gpu(lo, 4, q);
    on_gpu(hi, 4, q);
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), n_pages = lo.size(1), Hkv = lo.size(2);
    need(same_sizes(hi, lo.sizes()) && lo.size(0) == B && lo.size(3) == D && hi.scalar_type() == lo.scalar_type() &&
         hi.strides() == lo.strides() && contiguous_from(lo, 1) && q.stride(2) == 1);
    const Lengths len = lengths_of(a[3], B, q);
    const int32_t P = integer32(a[4]), top = integer32(a[5]);
    const bool keep_sink = truth(a[6]), select = truth(a[7]);
    need(P >= 1 && top >= 1 && (int64_t)top * P <= INT32_MAX);
    const int q_code = dtype_code(q), b_code = dtype_code(lo);
    Tensor scores;
    Selection s;
    int st;
    {
      NoGil free;
      scores = make({B, n_pages}, q, at::kFloat);
      if (select) s.allocate(B, top, P, q);
      st = nhs_quest_select((int32_t)B, q.data_ptr(), q_code, q.stride(0), q.stride(1), lo.data_ptr(), hi.data_ptr(),
                            b_code, lo.stride(0), (int32_t)Hq, (int32_t)Hkv, (int32_t)D, len.per_item, len.all, P,
                            (int32_t)n_pages, top, keep_sink, static_cast<float*>(scores.data_ptr()),
                            select ? static_cast<int32_t*>(s.pages.data_ptr()) : nullptr,
                            select ? static_cast<int32_t*>(s.positions.data_ptr()) : nullptr, stream_of(q));
    }
    return st ? failed("nhs_quest_select", st) : tuple_of({s.pages, s.positions, scores});
  });
}

void check_table(const Tensor& t, at::ScalarType type, int64_t B, const Tensor& other) {
  on_gpu(t, 2, other);
  need(t.scalar_type() == type && t.size(0) == B && t.stride(1) == 1);
}

PyObject* select_resolve_batched(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 12, [&]() -> PyObject* {
    const Tensor &scores = tensor(a[0]), &source = tensor(a[1]), &resident = tensor(a[2]), &hot = tensor(a[3]),
                 &tags = tensor(a[4]), &lru = tensor(a[5]);
    on_gpu(scores, 2);
    need(scores.scalar_type() == at::kFloat && scores.is_contiguous());
    const int64_t B = scores.size(0), max_pages = scores.size(1);
    check_table(source, at::kInt, B, scores);
    check_table(resident, at::kInt, B, scores);
    check_table(hot, at::kInt, B, scores);
    check_table(tags, at::kInt, B, scores);
    check_table(lru, at::kLong, B, scores);
    const Lengths len = lengths_of(a[6], B, scores);
    const int32_t P = integer32(a[7]), top = integer32(a[8]);
    const bool keep_sink = truth(a[9]);
    const int32_t mode = integer32(a[10]);
    need(P >= 1 && top >= 1 && (int64_t)top * P <= INT32_MAX);
    const int64_t H = tags.size(1), K = (int64_t)top * P;
    need(same_sizes(resident, source.sizes()) && resident.stride(0) == source.stride(0) && lru.size(1) == H &&
         hot.size(1) * P >= H);
    int64_t* total = nullptr;
    if (a[11] != Py_None) {
      const Tensor& t = tensor(a[11]);
      on_gpu(t, 1, scores);
      need(t.scalar_type() == at::kLong && t.size(0) == 3 && t.is_contiguous());
      total = static_cast<int64_t*>(t.data_ptr());
    }
    Selection s;
    Tensor physical, miss_host, miss_device, counts;
    int st;
    {
      NoGil free;
      s.allocate(B, top, P, scores);
      physical = make({B, K}, scores, at::kLong);
      miss_host = make({B, K}, scores, at::kLong);
      miss_device = make({B, K}, scores, at::kLong);
      counts = make({B, 3}, scores, at::kLong);
      st = nhs_select_resolve_rows(
          (int32_t)B, static_cast<const float*>(scores.data_ptr()), (int32_t)max_pages, mode, top, keep_sink,
          static_cast<const int32_t*>(source.data_ptr()), static_cast<const int32_t*>(resident.data_ptr()),
          source.stride(0), (int32_t)source.size(1), static_cast<const int32_t*>(hot.data_ptr()), hot.stride(0),
          static_cast<int32_t*>(tags.data_ptr()), tags.stride(0), static_cast<int64_t*>(lru.data_ptr()), lru.stride(0),
          (int32_t)H, len.per_item, len.all, P, static_cast<int32_t*>(s.pages.data_ptr()),
          static_cast<int32_t*>(s.positions.data_ptr()), static_cast<int64_t*>(physical.data_ptr()),
          static_cast<int64_t*>(miss_host.data_ptr()), static_cast<int64_t*>(miss_device.data_ptr()), K,
          static_cast<int64_t*>(counts.data_ptr()), total, stream_of(scores));
    }
    return st ? failed("nhs_select_resolve_rows", st)
              : tuple_of({s.pages, s.positions, physical, miss_host, miss_device, counts});
  });
}

// ---- rows in 8 bits ----------------------------------------------------------------------------

// A row_kernels.Rows8 that the library takes.
struct Form {
  int code;
  int32_t kv_heads, head_dim;
  int64_t row_bytes;
};
Form form_of(PyObject* o) {
  need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3 && THPDtype_Check(PyTuple_GET_ITEM(o, 0)));
  const at::ScalarType type = reinterpret_cast<THPDtype*>(PyTuple_GET_ITEM(o, 0))->scalar_type;
  need(type == at::kChar || type == at::kFloat8_e4m3fn);
  Form f;
  f.code = type == at::kChar ? NHS_CODE_I8 : NHS_CODE_E4M3;
  f.kv_heads = integer32(PyTuple_GET_ITEM(o, 1));
  f.head_dim = integer32(PyTuple_GET_ITEM(o, 2));
  need(f.kv_heads >= 1 && f.head_dim >= 1 && f.head_dim <= NHS_MAX_HEAD_DIM8);
  f.row_bytes = nhs_row8_bytes(f.kv_heads, f.head_dim);
  return f;
}

// Bytes between the blocks of a pool [blocks, 2, P, row_bytes].
int64_t pool8_block_stride(const Tensor& pool, const Form& f) {
  const int64_t P = pool.size(2), R = pool.size(3);
  need(pool.scalar_type() == at::kByte && pool.size(1) == 2 && R == f.row_bytes && pool.stride(1) == P * R &&
       pool.stride(2) == R && pool.stride(3) == 1 && pool.stride(0) >= 2 * P * R &&
       pool.size(0) * P < (int64_t(1) << 31));
  return pool.stride(0);
}

PyObject* attend_8bit(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 5, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &pool = tensor(a[1]), &rows = tensor(a[3]);
    const Form f = form_of(a[2]);
    on_gpu(q, 3);
    on_gpu(pool, 4, q);
    need(rows.dim() == 2 || rows.dim() == 3);
    on_gpu(rows, rows.dim(), q);
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), n = rows.size(-1);
    const int code = dtype_code(q);
    need(rows.scalar_type() == at::kLong && D == f.head_dim && Hq % f.kv_heads == 0 && q.stride(2) == 1 &&
         rows.size(0) == B && (rows.dim() == 2 || rows.size(1) == Hq) && n <= (1 << 30));
    const int64_t stride = pool8_block_stride(pool, f);
    Tensor out;
    if (a[4] != Py_None) {
      out = tensor(a[4]);
      check_out(out, q);
    }
    int st;
    {
      NoGil free;
      const OnDevice on(q);
      if (!out.defined()) out = make(q.sizes(), q, q.scalar_type());
      const int64_t bytes =
          nhs_attend_rows8_workspace_bytes((int32_t)B, (int32_t)n, (int32_t)Hq, f.kv_heads, f.head_dim);
      const Tensor ws = scratch(bytes, q);
      st = nhs_attend_rows8(q.data_ptr(), code, q.stride(0), q.stride(1), pool.data_ptr(), pool.size(0) * pool.size(2),
                            stride, f.code, static_cast<const int64_t*>(rows.data_ptr()), rows.stride(0),
                            rows.dim() == 3 ? rows.stride(1) : 0, rows.stride(-1), (int32_t)B, (int32_t)n, (int32_t)Hq,
                            f.kv_heads, f.head_dim, (int32_t)pool.size(2), out.data_ptr(), out.stride(0),
                            out.stride(1), scratch_ptr(ws), bytes, stream_of(q));
    }
    return st ? failed("nhs_attend_rows8", st) : THPVariable_Wrap(out);
  });
}

// read_rows_8bit into new tensors
PyObject* read_rows_8bit(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 4, [&]() -> PyObject* {
    const Tensor &pool = tensor(a[0]), &rows = tensor(a[2]);
    const Form f = form_of(a[1]);
    need(THPDtype_Check(a[3]));
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    need(type == at::kFloat || type == at::kHalf || type == at::kBFloat16);
    on_gpu(pool, 4);
    on_gpu(rows, 1, pool);
    need(rows.scalar_type() == at::kLong);
    const int64_t stride = pool8_block_stride(pool, f), n = rows.size(0), width = (int64_t)f.kv_heads * f.head_dim;
    Tensor k, v;
    int st;
    {
      NoGil free;
      const OnDevice on(pool);
      k = make({n, f.kv_heads, f.head_dim}, pool, type);
      v = make({n, f.kv_heads, f.head_dim}, pool, type);
      st = nhs_read_rows8(pool.data_ptr(), pool.size(0) * pool.size(2), stride, f.code, f.kv_heads, f.head_dim,
                          (int32_t)pool.size(2), static_cast<const int64_t*>(rows.data_ptr()), rows.stride(0), n,
                          dtype_code(k), k.data_ptr(), width, v.data_ptr(), width, stream_of(pool));
    }
    return st ? failed("nhs_read_rows8", st) : tuple_of({k, v});
  });
}

// A pinned host store [pages, 2, P, row_bytes] like the pool's blocks, given as a row_kernels.MappedHost or None.
struct Host8 {
  void* alias = nullptr;
  int64_t pages = 0;
};
Host8 host8_of(PyObject* o, const Tensor& pool) {
  Host8 h;
  if (o == Py_None) return h;
  PyObject *held = PyObject_GetAttrString(o, "tensor"), *pointer = PyObject_GetAttrString(o, "pointer");
  bool ok = held && pointer && THPVariable_Check(held) && PyLong_CheckExact(pointer);
  if (ok) {
    const Tensor& t = THPVariable_Unpack(held);
    ok = t.scalar_type() == at::kByte && t.dim() == 4 && t.is_contiguous() &&
         t.sizes().slice(1) == pool.sizes().slice(1);
    h.alias = PyLong_AsVoidPtr(pointer);
    h.pages = t.size(0);
  }
  Py_XDECREF(held);
  Py_XDECREF(pointer);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    ok = false;
  }
  need(ok && h.alias);
  return h;
}

// Checks k and v [tokens, Hkv, D] for appends; returns the elements between tokens.
int64_t check_append8(const Tensor& k, const Tensor& v, const Tensor& pool, const Form& f) {
  on_gpu(k, 3, pool);
  on_gpu(v, 3, pool);
  const int64_t width = (int64_t)f.kv_heads * f.head_dim, stride = k.size(0) > 1 ? k.stride(0) : width;
  need(k.size(1) == f.kv_heads && k.size(2) == f.head_dim && same_sizes(v, k.sizes()) &&
       v.scalar_type() == k.scalar_type() && contiguous_from(k, 1) && contiguous_from(v, 1) && stride >= width &&
       (k.size(0) == 1 || v.stride(0) == stride));
  return stride;
}

PyObject* append_items_8bit(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 7, [&]() -> PyObject* {
    const Tensor &k = tensor(a[0]), &v = tensor(a[1]), &pool = tensor(a[2]), &items = tensor(a[5]),
                 &lengths = tensor(a[6]);
    const Form f = form_of(a[3]);
    on_gpu(pool, 4);
    const int64_t token = check_append8(k, v, pool, f), stride = pool8_block_stride(pool, f), B = k.size(0);
    on_gpu(items, 2, pool);
    on_gpu(lengths, 1, pool);
    need(items.scalar_type() == at::kLong && items.size(0) == B && items.size(1) == 9 && items.is_contiguous() &&
         lengths.scalar_type() == at::kLong && lengths.size(0) == B && lengths.is_contiguous());
    const Host8 host = host8_of(a[4], pool);
    const int code = dtype_code(k);
    int st;
    {
      NoGil free;
      const OnDevice on(pool);
      st = nhs_append_items8((int32_t)B, k.data_ptr(), v.data_ptr(), token, code, f.code, f.kv_heads, f.head_dim,
                             (int32_t)pool.size(2), pool.data_ptr(), stride, host.alias,
                             static_cast<const nhs_layer_item*>(items.data_ptr()),
                             static_cast<const int64_t*>(lengths.data_ptr()), stream_of(pool));
    }
    if (st) return failed("nhs_append_items8", st);
    Py_RETURN_TRUE;
  });
}

// What row_kernels.PageAppender keeps of a write into rows in 8 bits, as bytes; page8 makes one page's call of it.
struct Write8 {
  const char *k, *v;
  char *pool, *host, *summary, *minimum, *maximum;
  void* stream;
  int64_t token, stride, tokens, blocks, host_pages, bounds, esize;
  int32_t dtype, code, kv_heads, head_dim, page_size, device;
};

PyObject* write8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 8, [&]() -> PyObject* {
    const Tensor &k = tensor(a[0]), &v = tensor(a[1]), &pool = tensor(a[2]);
    const Form f = form_of(a[3]);
    on_gpu(pool, 4);
    Write8 w;
    w.token = check_append8(k, v, pool, f);
    w.stride = pool8_block_stride(pool, f);
    const Host8 host = host8_of(a[4], pool);
    w.bounds = INT64_MAX;
    void* pointers[3];
    for (int i = 0; i < 3; ++i) {
      const Tensor& t = tensor(a[5 + i]);
      need(t.is_cuda() && t.device() == pool.device() && t.numel() > 0 && t.dim() >= 2 && t.is_contiguous() &&
           t.size(-2) == f.kv_heads && t.size(-1) == f.head_dim &&
           t.scalar_type() == (i == 0 ? at::kFloat : k.scalar_type()));
      pointers[i] = t.data_ptr();
      w.bounds = std::min(w.bounds, t.numel() / ((int64_t)f.kv_heads * f.head_dim));
    }
    w.k = static_cast<const char*>(k.data_ptr());
    w.v = static_cast<const char*>(v.data_ptr());
    w.pool = static_cast<char*>(pool.data_ptr());
    w.host = static_cast<char*>(host.alias);
    w.summary = static_cast<char*>(pointers[0]);
    w.minimum = static_cast<char*>(pointers[1]);
    w.maximum = static_cast<char*>(pointers[2]);
    w.stream = stream_of(pool);
    w.tokens = k.size(0);
    w.blocks = pool.size(0);
    w.host_pages = host.pages;
    w.esize = k.element_size();
    w.dtype = dtype_code(k);
    w.code = f.code;
    w.kv_heads = f.kv_heads;
    w.head_dim = f.head_dim;
    w.page_size = (int32_t)pool.size(2);
    w.device = pool.device().index();
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&w), sizeof w);
  });
}

// page8(write, first, count, block, within, host_page, bounds_index) -> the library's status, or None where an index
// is outside the write's tensors.
PyObject* page8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return native(nargs, 7, [&]() -> PyObject* {
    need(PyBytes_CheckExact(a[0]) && PyBytes_GET_SIZE(a[0]) == sizeof(Write8));
    Write8 w;
    memcpy(&w, PyBytes_AS_STRING(a[0]), sizeof w);
    const int64_t first = integer(a[1]), count = integer(a[2]), block = integer(a[3]), within = integer(a[4]),
                  host_page = integer(a[5]), at = integer(a[6]);
    need(first >= 0 && count >= 1 && count <= w.tokens && first <= w.tokens - count && block >= 0 && block < w.blocks &&
         within >= 0 && within <= w.page_size && count <= w.page_size && at >= 0 && at < w.bounds &&
         (!w.host || (host_page >= 0 && host_page < w.host_pages)));
    const int64_t width = (int64_t)w.kv_heads * w.head_dim, row = first * w.token * w.esize;
    int st;
    {
      NoGil free;
      const c10::OptionalDeviceGuard on(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)w.device));
      st = nhs_append_page8(w.k + row, w.v + row, w.token, w.dtype, w.code, w.kv_heads, w.head_dim, w.page_size, w.pool,
                            w.stride, block, (int32_t)within, (int32_t)count, w.host, w.host ? host_page : 0,
                            reinterpret_cast<float*>(w.summary) + at * width, w.minimum + at * width * w.esize,
                            w.maximum + at * width * w.esize, w.stream);
    }
    return PyLong_FromLong(st);
  });
}

// ---- append ------------------------------------------------------------------------------------

// nhs_append_page with the arguments row_kernels.PageAppender prepared (checked there), as whole numbers of any integer
// type; returns the status.
PyObject* append_page(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 17) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  int64_t v[17];
  for (int i = 0; i < 17; ++i) {  // negative numbers go to the library, which refuses them
    PyObject* whole = PyNumber_Index(a[i]);
    if (!whole) return nullptr;
    v[i] = (int64_t)PyLong_AsUnsignedLongLongMask(whole);
    Py_DECREF(whole);
    if (PyErr_Occurred()) return nullptr;
  }
  const auto at = [&](int i) { return reinterpret_cast<void*>((uintptr_t)v[i]); };
  int st;
  {
    NoGil free;
    st = nhs_append_page(at(0), at(1), v[2], (int32_t)v[3], (int32_t)v[4], (int32_t)v[5], at(6), v[7], v[8],
                         (int32_t)v[9], (int32_t)v[10], at(11), v[12], static_cast<float*>(at(13)), at(14), at(15),
                         at(16));
  }
  return PyLong_FromLong(st);
}

// ---- parameters --------------------------------------------------------------------------------

// Of a tensor its address, dtype, sizes and strides; of any other object, and of a tensor without them, its identity.
void add_state(std::vector<int64_t>& state, PyObject* value) {
  const size_t before = state.size();
  if (PyObject_TypeCheck(value, reinterpret_cast<PyTypeObject*>(THPVariableClass))) {
    try {
      const Tensor& t = THPVariable_Unpack(value);
      state.push_back((int64_t)(uintptr_t)t.const_data_ptr());
      state.push_back((int64_t)t.scalar_type() << 32 | t.dim());
      for (int64_t s : t.sizes()) state.push_back(s);
      for (int64_t s : t.strides()) state.push_back(s);
      return;
    } catch (const std::bad_alloc&) {
      throw;
    } catch (const std::exception&) {  // a sparse or wrapped tensor
      PyErr_Clear();
      state.resize(before);
    }
  }
  state.push_back((int64_t)(uintptr_t)value);
}

// The bytes that tell whether the dicts (of modules' parameters and child
// modules) hold what they held: each dict's size and its values' states. For
// checks made on every step.
PyObject* held_state(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 1 || !PyList_CheckExact(a[0])) {
    PyErr_SetString(PyExc_TypeError, "held_state takes a list of dicts");
    return nullptr;
  }
  try {
    std::vector<int64_t> state;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) {
      PyObject* dict = PyList_GET_ITEM(a[0], i);
      if (!PyDict_Check(dict)) {
        PyErr_SetString(PyExc_TypeError, "held_state takes a list of dicts");
        return nullptr;
      }
      state.push_back(PyDict_Size(dict));
      PyObject *key, *value;
      Py_ssize_t at = 0;
      while (PyDict_Next(dict, &at, &key, &value)) add_state(state, value);
    }
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(state.data()),
                                     (Py_ssize_t)(state.size() * sizeof(int64_t)));
  } catch (const std::bad_alloc&) {
    return PyErr_NoMemory();
  }
}

#define NHS_METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {NHS_METHOD(linear_small_m), NHS_METHOD(linear_silu_mul),   NHS_METHOD(linear_rope),
                         NHS_METHOD(add_rmsnorm),    NHS_METHOD(attend_batched),    NHS_METHOD(prefill_attention),
                         NHS_METHOD(quest_batched),  NHS_METHOD(select_resolve_batched),
                         NHS_METHOD(append_page),    NHS_METHOD(held_state),        NHS_METHOD(tree_plan),
                         NHS_METHOD(tree_attention), NHS_METHOD(qk_norm_rope),      NHS_METHOD(token_logprobs),
                         NHS_METHOD(attend_8bit),    NHS_METHOD(read_rows_8bit),    NHS_METHOD(append_items_8bit),
                         NHS_METHOD(write8),         NHS_METHOD(page8),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch() { return PyModule_Create(&module); }
