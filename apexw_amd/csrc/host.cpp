// Host-side scan of a step plan's tensors, once per optimizer step.
//
// A step plan keeps raw device pointers of every parameter and grad in its
// descriptor table.  Before each launch it must know whether the table is still
// right: a grad may be a new tensor (zero_grad(set_to_none=True) every step),
// and a parameter or grad may have had its storage swapped in place
// (`p.data = ...`, `module.to(dtype)`), which keeps the Python objects and
// changes address and dtype.  Checking that from Python costs about 100 ns per
// attribute read per tensor; this scan reads the tensors directly (about 10 ns
// each), which matters for groups of tens of thousands of tensors.
//
// Plain CPython module (no pybind11): the step's functions take Python lists of
// torch tensors and the addresses of caller-owned numpy buffers, the operators'
// ones (below) tensors.

#include <Python.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <vector>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// scan status (mirrored in apexw_amd/_plan.py)
constexpr long kSame = 0;        // every pointer and dtype as recorded
constexpr long kGradsMoved = 1;  // only grad pointers changed (written to the scratch buffer)
constexpr long kMissing = 2;     // a plan parameter lost its grad, or another parameter gained one
constexpr long kRebuilt = 3;     // a parameter's storage or dtype changed
constexpr long kSlowPath = 4;    // a grad is laid out unlike its parameter, or of another size
constexpr long kGradDtype = 5;   // a grad's dtype differs from the one the table was built for

bool unpack_list(PyObject* obj, const char* what) {
  if (!PyList_Check(obj)) {
    PyErr_Format(PyExc_TypeError, "%s must be a list of tensors", what);
    return false;
  }
  const Py_ssize_t n = PyList_GET_SIZE(obj);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_Check(PyList_GET_ITEM(obj, i))) {
      PyErr_Format(PyExc_TypeError, "%s[%zd] is not a tensor", what, i);
      return false;
    }
  }
  return true;
}

bool as_addr(PyObject* obj, uintptr_t* out) {
  *out = static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(obj));
  return !PyErr_Occurred();
}

// snapshot(params, p_ptrs_addr, dtypes_addr)
//   p_ptrs: uint64[n] <- data pointers; dtypes: int8[n] <- at::ScalarType codes
PyObject* snapshot(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "snapshot(params, p_ptrs_addr, dtypes_addr)");
    return nullptr;
  }
  uintptr_t pa, da;
  if (!unpack_list(args[0], "params") || !as_addr(args[1], &pa) || !as_addr(args[2], &da)) return nullptr;
  auto* p_ptrs = reinterpret_cast<uint64_t*>(pa);
  auto* dtypes = reinterpret_cast<int8_t*>(da);
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
    p_ptrs[i] = reinterpret_cast<uint64_t>(p.data_ptr());
    dtypes[i] = static_cast<int8_t>(p.scalar_type());
  }
  Py_RETURN_NONE;
}

// scan(params, inactive, p_ptrs_addr, dtypes_addr, g_ptrs_addr, g_scratch_addr, g_dtypes_addr) -> status
//   params: the plan's parameters, in table order; inactive: the group's other
//   trainable parameters.  g_ptrs holds the grad pointers the table was built
//   from; on kGradsMoved the current ones are in g_scratch.  g_dtypes: the grad
//   dtypes the table was built for (a grad may differ from its parameter's dtype:
//   torch's Tensor.grad_dtype).
PyObject* scan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7) {
    PyErr_SetString(PyExc_TypeError, "scan(params, inactive, p_ptrs, dtypes, g_ptrs, g_scratch, g_dtypes)");
    return nullptr;
  }
  uintptr_t pa, da, ga, sa, gda;
  if (!unpack_list(args[0], "params") || !unpack_list(args[1], "inactive") || !as_addr(args[2], &pa) ||
      !as_addr(args[3], &da) || !as_addr(args[4], &ga) || !as_addr(args[5], &sa) || !as_addr(args[6], &gda))
    return nullptr;
  const auto* p_ptrs = reinterpret_cast<const uint64_t*>(pa);
  const auto* dtypes = reinterpret_cast<const int8_t*>(da);
  const auto* g_ptrs = reinterpret_cast<const uint64_t*>(ga);
  auto* g_scratch = reinterpret_cast<uint64_t*>(sa);
  const auto* g_dtypes = reinterpret_cast<const int8_t*>(gda);

  const Py_ssize_t n_in = PyList_GET_SIZE(args[1]);
  for (Py_ssize_t i = 0; i < n_in; ++i) {
    const at::Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(args[1], i));
    if (p.grad().defined()) return PyLong_FromLong(kMissing);
  }
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  bool moved = false, slow = false, gdt = false;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
    if (reinterpret_cast<uint64_t>(p.data_ptr()) != p_ptrs[i] || static_cast<int8_t>(p.scalar_type()) != dtypes[i])
      return PyLong_FromLong(kRebuilt);
    const at::Tensor& g = p.grad();
    if (!g.defined()) return PyLong_FromLong(kMissing);
    if (static_cast<int8_t>(g.scalar_type()) != g_dtypes[i]) {
      gdt = true;
      continue;
    }
    // the step walks the grad in its parameter's memory layout
    if (g.strides() != p.strides() || g.numel() != p.numel()) {
      slow = true;
      continue;
    }
    const uint64_t gp = reinterpret_cast<uint64_t>(g.data_ptr());
    g_scratch[i] = gp;
    moved |= gp != g_ptrs[i];
  }
  if (gdt) return PyLong_FromLong(kGradDtype);
  if (slow) return PyLong_FromLong(kSlowPath);
  return PyLong_FromLong(moved ? kGradsMoved : kSame);
}

// ---------------------------------------------------------------------------
// The operators around the step (apexw_amd/ops.py, tokens.py, head.py): the usual call checked, its outputs allocated and the
// library called in one go, which takes a third of the time that the same takes from Python.  Each function
// returns None for what it does not take (another layout, device or type); the Python form then copies,
// converts or raises.  A nonzero apexw_status comes back as an int.
// ---------------------------------------------------------------------------
struct ClipTensor {   // apexw_clip_tensor of include/apexw_hip.h
  const void* g;
  void* out;
  int64_t n, first_unit;
  uint32_t g_dtype, out_dtype;
};
constexpr int kClipSmall = 48;        // APEXW_CLIP_SMALL
constexpr int kClipPartials = 2048;   // APEXW_CLIP_PARTIALS

struct Library {
  int (*norm_forward)(const void*, int64_t, int64_t, int64_t, int32_t, const void*, const void*, int32_t, float, void*,
                      float*, float*, void*);
  int (*norm_backward)(const void*, int64_t, const void*, int64_t, const float*, const float*, const void*, int64_t,
                       int64_t, int32_t, int32_t, void*, void*, void*, float*, void*);
  int64_t (*norm_workspace)(int64_t, int64_t);
  int (*expert_rows)(const void*, int64_t, const void*, int64_t, int64_t, int32_t, const int32_t*, int32_t, int64_t,
                     int64_t, int64_t, int32_t, void*, int64_t, void*, void*);
  int64_t (*expert_rows_workspace)(const void*, int64_t, const void*, int64_t, int64_t, int32_t, int32_t, int64_t,
                                   int64_t, int64_t);
  int (*expert_weight_grad)(const void*, int64_t, const void*, int64_t, const int32_t*, int32_t, int64_t, int64_t,
                            int64_t, int32_t, void*, int32_t, void*, void*);
  int64_t (*expert_weight_grad_workspace)(const void*, int64_t, const void*, int64_t, int32_t, int64_t, int64_t, int64_t);
  int64_t (*clip_layout)(ClipTensor*, int32_t);
  int (*clip_grads)(const ClipTensor*, int32_t, int64_t, int32_t, float, double*, float*, void*);
  int (*clip_grads_small)(const ClipTensor*, int32_t, int64_t, int32_t, float, double*, float*, void*);
  int64_t (*order_workspace)(int64_t, int32_t);
  int (*order)(const void*, int32_t, int64_t, int32_t, int32_t*, int32_t*, int32_t*, void*, void*);
  int (*dispatch)(const void*, int64_t, int64_t, int32_t, int64_t, int32_t, const int32_t*, const int32_t*, void*, void*);
  int (*combine)(const void*, int64_t, int64_t, int32_t, int64_t, int32_t, const int32_t*, const void*, int32_t, void*, void*);
  int (*combine_backward)(const void*, int64_t, const void*, int64_t, int64_t, int32_t, int64_t, int32_t, const int32_t*,
                          const int32_t*, const void*, int32_t, void*, void*, void*);
  int (*embedding)(const void*, int32_t, int64_t, const void*, int64_t, int64_t, int64_t, int32_t, float, void*, void*);
  int64_t (*embedding_grad_workspace)(int64_t, int64_t, int64_t);
  int (*embedding_grad)(const void*, int64_t, const void*, int32_t, int64_t, int64_t, int64_t, int32_t, float, void*,
                        int32_t, void*, void*);
  int64_t (*head_workspace)(const void*, int64_t, int64_t, int64_t, int64_t, int32_t);
  int (*head_forward)(const void*, int64_t, int64_t, int64_t, const void*, int64_t, int64_t, int32_t, const void*, int32_t,
                      int64_t, float*, float*, int32_t, float*, void*, void*);
  int (*head_backward)(const float*, int64_t, int32_t, const void*, int64_t, int64_t, int64_t, const void*, int64_t,
                       int64_t, int32_t, const void*, int32_t, int64_t, const float*, void*, void*, void*, void*);
} lib;
constexpr int kEntries = sizeof(Library) / sizeof(void*);

// bind(addresses): the entry points, in the order of Library
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != kEntries) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kEntries);
    return nullptr;
  }
  uintptr_t at[kEntries];
  for (int i = 0; i < kEntries; ++i)
    if (!as_addr(args[i], &at[i])) return nullptr;
  static_assert(sizeof(at) == sizeof(lib), "function pointers");
  std::memcpy(&lib, at, sizeof(lib));
  Py_RETURN_NONE;
}

bool dtype_code(const at::Tensor& t, uint32_t* code) {
  switch (t.scalar_type()) {
    case at::kFloat: *code = 0; return true;
    case at::kBFloat16: *code = 1; return true;
    case at::kHalf: *code = 2; return true;
    default: return false;
  }
}

// where a call runs: the current stream and device
struct Where {
  void* stream;
  long device;
  bool set(PyObject* s, PyObject* d) {
    uintptr_t p;
    if (!lib.norm_forward || !as_addr(s, &p)) return false;
    stream = reinterpret_cast<void*>(p);
    device = PyLong_AsLong(d);
    return !PyErr_Occurred();
  }
  bool has(const at::Tensor& t) const {
    return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device;
  }
};

PyObject* none_or_error() {
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyObject* pack(const at::Tensor* const* t, int n) {
  PyObject* out = PyTuple_New(n);
  if (!out) return nullptr;
  for (int i = 0; i < n; ++i) {
    PyObject* v;
    if (t[i]->defined()) {
      v = THPVariable_Wrap(*t[i]);
    } else {
      v = Py_None;
      Py_INCREF(v);
    }
    if (!v) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i, v);
  }
  return out;
}

bool optional_tensor(PyObject* o, at::Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}

// a weight or bias of `width` elements for rows of `code`; sets their common type
bool norm_param(const at::Tensor& t, const Where& w, int64_t width, uint32_t code, uint32_t* w_code) {
  if (!t.defined()) return true;
  uint32_t c;
  if (!w.has(t) || !dtype_code(t, &c) || t.dim() != 1 || t.size(0) != width || !t.is_contiguous()) return false;
  if ((c != code && c != 0) || (*w_code != ~0u && *w_code != c)) return false;
  *w_code = c;
  return true;
}

const void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// layer_norm_forward(x, weight, bias, eps, stream, device) -> (y, mean, rstd)
PyObject* layer_norm_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  at::Tensor w, b;
  if (nargs != 6 || !THPVariable_Check(args[0]) || !optional_tensor(args[1], &w) || !optional_tensor(args[2], &b) ||
      !where.set(args[4], args[5]))
    return none_or_error();
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  uint32_t code, w_code = ~0u;
  if (!where.has(x) || !dtype_code(x, &code) || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous() || !(eps >= 0)) return none_or_error();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  if (!norm_param(w, where, width, code, &w_code) || !norm_param(b, where, width, code, &w_code)) return none_or_error();
  if (w_code == ~0u) w_code = code;
  const at::Tensor y = at::empty(x.sizes(), x.options());
  const auto per_row = x.sizes().slice(0, x.dim() - 1);
  const at::Tensor mean = at::empty(per_row, x.options().dtype(at::kFloat)), rstd = at::empty(per_row, mean.options());
  const int status = lib.norm_forward(x.data_ptr(), rows, width, width, code, address(w), address(b), w_code,
                                      static_cast<float>(eps), y.data_ptr(), static_cast<float*>(mean.data_ptr()),
                                      static_cast<float*>(rstd.data_ptr()), where.stream);
  if (status) return PyLong_FromLong(status);
  const at::Tensor* out[] = {&y, &mean, &rstd};
  return pack(out, 3);
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dy, x, mean, rstd, weight, bias, need_x, need_w, need_b, stream, device) -> (dx, dw, db)
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  at::Tensor w, b;
  if (nargs != 11) return none_or_error();
  for (int i = 0; i < 4; ++i)
    if (!THPVariable_Check(args[i])) return none_or_error();
  if (!optional_tensor(args[4], &w) || !optional_tensor(args[5], &b) || !where.set(args[9], args[10]))
    return none_or_error();
  const at::Tensor &dy = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]),
                   &mean = THPVariable_Unpack(args[2]), &rstd = THPVariable_Unpack(args[3]);
  uint32_t code, w_code = ~0u;
  if (!where.has(x) || !dtype_code(x, &code) || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous()) return none_or_error();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  if (!where.has(dy) || dy.scalar_type() != x.scalar_type() || dy.sizes() != x.sizes() || !dy.is_contiguous())
    return none_or_error();
  for (const at::Tensor* t : {&mean, &rstd})
    if (!where.has(*t) || t->scalar_type() != at::kFloat || t->numel() != rows || !t->is_contiguous())
      return none_or_error();
  if (!norm_param(w, where, width, code, &w_code) || !norm_param(b, where, width, code, &w_code)) return none_or_error();
  if (w_code == ~0u) w_code = code;
  bool need[3];   // any truth values
  for (int i = 0; i < 3; ++i) {
    const int truth = PyObject_IsTrue(args[6 + i]);
    if (truth < 0) return nullptr;
    need[i] = truth != 0;
  }
  at::Tensor dx, dw, db, ws;
  if (need[0]) dx = at::empty(x.sizes(), x.options());
  if (need[1] && w.defined()) dw = at::empty({width}, w.options());
  if (need[2] && b.defined()) db = at::empty({width}, b.options());
  if (dw.defined() || db.defined()) {
    const int64_t floats = lib.norm_workspace(rows, width);
    if (floats < 0) return PyLong_FromLong(static_cast<long>(-floats));
    ws = at::empty({floats}, mean.options());
  }
  if (dx.defined() || ws.defined()) {
    const int status = lib.norm_backward(
        dy.data_ptr(), width, x.data_ptr(), width, static_cast<const float*>(mean.data_ptr()),
        static_cast<const float*>(rstd.data_ptr()), address(w), rows, width, code, w_code, const_cast<void*>(address(dx)),
        const_cast<void*>(address(dw)), const_cast<void*>(address(db)),
        static_cast<float*>(const_cast<void*>(address(ws))), where.stream);
    if (status) return PyLong_FromLong(status);
  }
  const at::Tensor* out[] = {&dx, &dw, &db};
  return pack(out, 3);
  END_HANDLE_TH_ERRORS
}

// rows of 16-bit elements, whole in their last dimension
bool expert_operand(const at::Tensor& t, const Where& w, uint32_t* code) {
  return w.has(t) && dtype_code(t, code) && *code != 0 && t.dim() == 2 && t.size(1) > 0 && t.stride(1) == 1;
}
bool expert_ends(const at::Tensor& t, const Where& w) {
  return w.has(t) && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) > 0 && t.is_contiguous();
}

// expert_rows(a, weight, ends, transposed, stream, device) -> weight[e] a[i], or weight[e]^T a[i]
PyObject* expert_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) ||
      !where.set(args[4], args[5]))
    return none_or_error();
  const at::Tensor &a = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]), &ends = THPVariable_Unpack(args[2]);
  const bool transposed = args[3] == Py_True;
  uint32_t code;
  if (!expert_operand(a, where, &code) || !expert_ends(ends, where) || !where.has(w) ||
      w.scalar_type() != a.scalar_type() || w.dim() != 3 || w.numel() == 0 || w.stride(2) != 1 ||
      w.size(0) != ends.size(0) || w.size(transposed ? 1 : 2) != a.size(1) || a.size(0) == 0)
    return none_or_error();
  const int64_t n = w.size(transposed ? 2 : 1);
  const auto experts = static_cast<int32_t>(ends.size(0));
  const int64_t bytes = lib.expert_rows_workspace(a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(1), w.stride(0),
                                                  transposed, experts, a.size(0), a.size(1), n);
  if (bytes < 0) return PyLong_FromLong(static_cast<long>(-bytes));
  const at::Tensor out = at::empty({a.size(0), n}, a.options());
  at::Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, a.options().dtype(at::kByte));
  const int status = lib.expert_rows(a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(1), w.stride(0), transposed,
                                     static_cast<const int32_t*>(ends.data_ptr()), experts, a.size(0), a.size(1), n, code,
                                     out.data_ptr(), n, const_cast<void*>(address(ws)), where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// expert_weight_grad(dy, x, ends, fp32, stream, device) -> dW
PyObject* expert_weight_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) ||
      !where.set(args[4], args[5]))
    return none_or_error();
  const at::Tensor &dy = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]), &ends = THPVariable_Unpack(args[2]);
  const bool fp32 = args[3] == Py_True;
  uint32_t code, x_code;
  if (!expert_operand(dy, where, &code) || !expert_operand(x, where, &x_code) || code != x_code ||
      !expert_ends(ends, where) || dy.size(0) != x.size(0) || dy.size(0) == 0)
    return none_or_error();
  const auto experts = static_cast<int32_t>(ends.size(0));
  const int64_t bytes = lib.expert_weight_grad_workspace(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), experts,
                                                         dy.size(0), dy.size(1), x.size(1));
  if (bytes < 0) return PyLong_FromLong(static_cast<long>(-bytes));
  at::Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  const at::Tensor dw = at::empty({ends.size(0), dy.size(1), x.size(1)}, fp32 ? dy.options().dtype(at::kFloat) : dy.options());
  const int status = lib.expert_weight_grad(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0),
                                            static_cast<const int32_t*>(ends.data_ptr()), experts, dy.size(0),
                                            dy.size(1), x.size(1), code, dw.data_ptr(), fp32 ? 0 : code,
                                            const_cast<void*>(address(ws)), where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(dw);
  END_HANDLE_TH_ERRORS
}

// Bytes [begin, end) of a clip's tensor
struct Span {
  uintptr_t begin, end;
};
Span span(const void* p, int64_t n, uint32_t code) {
  const auto at = reinterpret_cast<uintptr_t>(p);
  return {at, at + static_cast<uintptr_t>(n) * (code == 0 ? 4 : 2)};
}

// Every tensor that a clip writes has to lie apart from all others: the workgroups scale them at the same time.
// Gradients that are only read may share memory.  Lists in the order of their addresses are known to be apart
// in one pass; others are sorted (2000 tensors in another order 25 us).
// total: the norm that the scaling reads, or null.
bool apart(const ClipTensor* table, Py_ssize_t n, const char* name, const void* total) {
  const auto in_place = [](const ClipTensor& t) { return t.out == t.g && t.out_dtype == t.g_dtype; };
  Span written{UINTPTR_MAX, 0}, read{UINTPTR_MAX, 0};   // from the lowest to the highest byte
  bool ordered = true;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const ClipTensor& t = table[i];
    if (t.n == 0) continue;
    const Span o = span(t.out, t.n, t.out_dtype);
    if (o.begin < reinterpret_cast<uintptr_t>(total) + 4 && reinterpret_cast<uintptr_t>(total) < o.end) {
      PyErr_Format(PyExc_ValueError, "%s: tensor %zd, which it writes, holds total_norm", name, i);
      return false;
    }
    ordered = ordered && o.begin >= written.end;
    written = {std::min(written.begin, o.begin), std::max(written.end, o.end)};
    if (in_place(t)) continue;
    const Span g = span(t.g, t.n, t.g_dtype);
    read = {std::min(read.begin, g.begin), std::max(read.end, g.end)};
  }
  const bool mixed = read.begin < written.end && written.begin < read.end;
  if (ordered && !mixed) return true;

  struct Entry {
    Span at;
    Py_ssize_t tensor;
  };
  std::vector<Entry> outs, grads;
  outs.reserve(n);
  if (mixed) grads.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const ClipTensor& t = table[i];
    if (t.n == 0) continue;
    outs.push_back({span(t.out, t.n, t.out_dtype), i});
    if (mixed && !in_place(t)) grads.push_back({span(t.g, t.n, t.g_dtype), i});
  }
  for (auto* list : {&outs, &grads})
    std::sort(list->begin(), list->end(), [](const Entry& a, const Entry& b) { return a.at.begin < b.at.begin; });
  const auto shared = [name](const Entry& a, const Entry& b) {
    PyErr_Format(PyExc_ValueError, "%s: tensors %zd and %zd share memory that the clip writes", name,
                 std::min(a.tensor, b.tensor), std::max(a.tensor, b.tensor));
    return false;
  };
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].at.begin < outs[i - 1].at.end) return shared(outs[i - 1], outs[i]);
  size_t w = 0;
  for (const Entry& g : grads) {
    while (w < outs.size() && outs[w].at.end <= g.at.begin) ++w;
    if (w < outs.size() && outs[w].at.begin < g.at.end) return shared(outs[w], g);
  }
  return true;
}

// The entries of a clip's table (first_unit left 0).  Raises for tensors that the clip does not take:
// another device, type or layout, and, where it writes them, memory that two of them share.
bool fill_clip(PyObject* grads, PyObject* outs, ClipTensor* table, const char* name, bool writes,
               const void* total = nullptr) {
  const Py_ssize_t n = PyList_GET_SIZE(grads);
  if (PyList_GET_SIZE(outs) != n) {
    PyErr_SetString(PyExc_ValueError, "clip: lists of different lengths");
    return false;
  }
  const bool in_place = grads == outs;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& g = THPVariable_Unpack(PyList_GET_ITEM(grads, i));
    const at::Tensor& o = in_place ? g : THPVariable_Unpack(PyList_GET_ITEM(outs, i));
    ClipTensor& t = table[i];
    if (g.layout() != at::kStrided || o.layout() != at::kStrided) {
      PyErr_Format(PyExc_ValueError, "%s: tensor %zd is sparse", name, i);
      return false;
    }
    const at::Device device = THPVariable_Unpack(PyList_GET_ITEM(grads, 0)).device();
    if (g.device() != device || o.device() != device) {
      PyErr_Format(PyExc_ValueError, "%s: tensor %zd is on another device than the first one", name, i);
      return false;
    }
    if (!dtype_code(g, &t.g_dtype) || !dtype_code(o, &t.out_dtype)) {
      PyErr_Format(PyExc_TypeError, "%s: tensor %zd is not float32, bfloat16 or float16", name, i);
      return false;
    }
    const bool whole = g.is_contiguous();
    if (!whole && !g.is_non_overlapping_and_dense()) {
      PyErr_Format(PyExc_ValueError, "%s: tensor %zd is not dense", name, i);
      return false;
    }
    if (!in_place && (g.sizes() != o.sizes() || (whole ? !o.is_contiguous() : g.strides() != o.strides()))) {
      PyErr_Format(PyExc_ValueError, "%s: the copy of tensor %zd has another shape or layout", name, i);
      return false;
    }
    t.g = g.data_ptr();
    t.out = o.data_ptr();
    t.n = g.numel();
    t.first_unit = 0;
  }
  return !writes || apart(table, n, name, total);
}

// New versions for what a clip writes, as every in-place operation gives: autograd refuses to go back through
// what saved the old values.
void bump_versions(PyObject* outs) {
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(outs); ++i) {
    const at::Tensor& o = THPVariable_Unpack(PyList_GET_ITEM(outs, i));
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  }
}

// clip_table(grads, out, table_addr, name, writes, total_addr=0): fill_clip into the table at table_addr; a list
// that is about to be written gets new versions.  total_addr: of the norm to scale by, or 0
PyObject* clip_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 && nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "clip_table(grads, out, table_addr, name, writes, total_addr=0)");
    return nullptr;
  }
  uintptr_t ta, total = 0;
  if (!unpack_list(args[0], "grads") || !unpack_list(args[1], "out") || !as_addr(args[2], &ta) ||
      (nargs == 6 && !as_addr(args[5], &total)))
    return nullptr;
  const char* name = PyUnicode_AsUTF8(args[3]);
  const bool writes = args[4] == Py_True;
  if (!name || !fill_clip(args[0], args[1], reinterpret_cast<ClipTensor*>(ta), name, writes,
                          reinterpret_cast<const void*>(total)))
    return nullptr;
  if (writes) bump_versions(args[1]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// clip_grads(grads, out, max_norm, order, stream, device) -> the norm
PyObject* clip_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 6 || !where.set(args[4], args[5])) return none_or_error();
  if (!unpack_list(args[0], "grads") || !unpack_list(args[1], "out")) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  if (n == 0 || n > INT32_MAX) return none_or_error();
  const at::Tensor& first = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0));
  const double max_norm = PyFloat_AsDouble(args[2]);
  const long order = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!where.has(first)) return none_or_error();
  ClipTensor small[kClipSmall];
  at::Tensor host, table;
  ClipTensor* t = small;
  if (n > kClipSmall) {
    host = at::empty({static_cast<int64_t>(n * sizeof(ClipTensor))}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
    t = static_cast<ClipTensor*>(host.data_ptr());
  }
  if (!fill_clip(args[0], args[1], t, "clip_grads", true)) return nullptr;
  const int64_t units = lib.clip_layout(t, static_cast<int32_t>(n));
  if (units < 0) return PyLong_FromLong(static_cast<long>(-units));
  const auto options = at::TensorOptions().device(first.device());
  const at::Tensor ws = at::empty({kClipPartials}, options.dtype(at::kDouble)), norm = at::empty({}, options.dtype(at::kFloat));
  if (n > kClipSmall) table = host.to(first.device(), /*non_blocking=*/true);
  auto* call = n > kClipSmall ? lib.clip_grads : lib.clip_grads_small;
  const int status = call(n > kClipSmall ? static_cast<const ClipTensor*>(table.data_ptr()) : small, static_cast<int32_t>(n),
                          units, static_cast<int32_t>(order), static_cast<float>(max_norm),
                          static_cast<double*>(ws.data_ptr()), static_cast<float*>(norm.data_ptr()), where.stream);
  if (status) return PyLong_FromLong(status);
  bump_versions(args[1]);   // (while the GPU is at work)
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// rows of any of the three types, whole in their last dimension
bool matrix(const at::Tensor& t, const Where& w, uint32_t* code) {
  return w.has(t) && dtype_code(t, code) && t.dim() == 2 && t.size(1) > 0 && t.stride(1) == 1;
}
// contiguous ids of 4 or 8 bytes
bool ids_of(const at::Tensor& t, const Where& w, int32_t* bytes) {
  if (!w.has(t) || !t.is_contiguous()) return false;
  *bytes = t.scalar_type() == at::kLong ? 8 : t.scalar_type() == at::kInt ? 4 : 0;
  return *bytes != 0;
}
// an order's source and place: the number of tokens and of choices of each
bool order_of(const at::Tensor& source, const at::Tensor& place, const Where& w, int64_t* tokens, int32_t* k) {
  if (!expert_ends(source, w) || !w.has(place) || place.scalar_type() != at::kInt || !place.is_contiguous() ||
      (place.dim() != 1 && place.dim() != 2) || place.numel() != source.size(0))
    return false;
  *tokens = place.size(0);
  *k = place.dim() == 2 ? static_cast<int32_t>(place.size(1)) : 1;
  return true;
}
// a weight for each choice
bool order_weight(const at::Tensor& t, const at::Tensor& place, const Where& w, uint32_t code, uint32_t* w_code) {
  return w.has(t) && dtype_code(t, w_code) && (*w_code == code || *w_code == 0) && t.sizes() == place.sizes() && t.is_contiguous();
}
const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
void* space(int64_t bytes, const at::Tensor& like, at::Tensor* ws) {
  if (bytes > 0) *ws = at::empty({bytes}, like.options().dtype(at::kByte));
  return const_cast<void*>(address(*ws));
}
bool all_tensors(PyObject* const* args, int n) {
  for (int i = 0; i < n; ++i)
    if (!THPVariable_Check(args[i])) return false;
  return true;
}

// expert_order(expert, experts, stream, device) -> (source, place, ends)
PyObject* expert_order(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 4 || !THPVariable_Check(args[0]) || !PyLong_Check(args[1]) || !where.set(args[2], args[3])) return none_or_error();
  const at::Tensor& expert = THPVariable_Unpack(args[0]);
  const long experts = PyLong_AsLong(args[1]);
  int32_t bytes;
  if (PyErr_Occurred()) return nullptr;
  if (!ids_of(expert, where, &bytes) || expert.numel() == 0 || expert.dim() < 1 || expert.dim() > 2 || experts < 1 ||
      experts >= INT32_MAX)
    return none_or_error();
  const int64_t n = expert.numel(), need = lib.order_workspace(n, static_cast<int32_t>(experts));
  if (need < 0) return PyLong_FromLong(static_cast<long>(-need));
  const auto options = expert.options().dtype(at::kInt);
  const at::Tensor source = at::empty({n}, options), place = at::empty(expert.sizes(), options), ends = at::empty({experts}, options);
  at::Tensor ws;
  const int status = lib.order(expert.data_ptr(), bytes, n, static_cast<int32_t>(experts), static_cast<int32_t*>(source.data_ptr()),
                               static_cast<int32_t*>(place.data_ptr()), static_cast<int32_t*>(ends.data_ptr()),
                               space(need, expert, &ws), where.stream);
  if (status) return PyLong_FromLong(status);
  const at::Tensor* out[] = {&source, &place, &ends};
  return pack(out, 3);
  END_HANDLE_TH_ERRORS
}

// expert_dispatch(x, source, place, stream, device) -> rows
PyObject* expert_dispatch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 5 || !all_tensors(args, 3) || !where.set(args[3], args[4])) return none_or_error();
  const at::Tensor &x = THPVariable_Unpack(args[0]), &source = THPVariable_Unpack(args[1]), &place = THPVariable_Unpack(args[2]);
  uint32_t code;
  int64_t tokens;
  int32_t k;
  if (!matrix(x, where, &code) || !order_of(source, place, where, &tokens, &k) || x.size(0) != tokens) return none_or_error();
  const at::Tensor rows = at::empty({tokens * k, x.size(1)}, x.options());
  const int status = lib.dispatch(x.data_ptr(), x.stride(0), tokens, k, x.size(1), code, ints(source), ints(place), rows.data_ptr(),
                                  where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(rows);
  END_HANDLE_TH_ERRORS
}

// expert_combine(y, source, place, weight, stream, device) -> out
PyObject* expert_combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  at::Tensor w;
  if (nargs != 6 || !all_tensors(args, 3) || !optional_tensor(args[3], &w) || !where.set(args[4], args[5])) return none_or_error();
  const at::Tensor &y = THPVariable_Unpack(args[0]), &source = THPVariable_Unpack(args[1]), &place = THPVariable_Unpack(args[2]);
  uint32_t code, w_code;
  int64_t tokens;
  int32_t k;
  if (!matrix(y, where, &code) || !order_of(source, place, where, &tokens, &k) || y.size(0) != source.size(0)) return none_or_error();
  w_code = code;
  if (w.defined() && !order_weight(w, place, where, code, &w_code)) return none_or_error();
  const at::Tensor out = at::empty({tokens, y.size(1)}, y.options());
  const int status = lib.combine(y.data_ptr(), y.stride(0), tokens, k, y.size(1), code, ints(place), address(w), w_code, out.data_ptr(),
                                 where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// expert_combine_backward(dout, y, source, place, weight, need_y, need_w, stream, device) -> (dy, dweight)
PyObject* expert_combine_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  at::Tensor y;
  if (nargs != 9 || !THPVariable_Check(args[0]) || !optional_tensor(args[1], &y) || !all_tensors(args + 2, 3) ||
      !where.set(args[7], args[8]))
    return none_or_error();
  const at::Tensor &dout = THPVariable_Unpack(args[0]), &source = THPVariable_Unpack(args[2]), &place = THPVariable_Unpack(args[3]),
                   &w = THPVariable_Unpack(args[4]);
  const int need_y = PyObject_IsTrue(args[5]), need_w = PyObject_IsTrue(args[6]);
  if (need_y < 0 || need_w < 0) return nullptr;
  uint32_t code, y_code, w_code;
  int64_t tokens;
  int32_t k;
  if (!matrix(dout, where, &code) || !order_of(source, place, where, &tokens, &k) || dout.size(0) != tokens ||
      !order_weight(w, place, where, code, &w_code))
    return none_or_error();
  if (need_w && (!y.defined() || !matrix(y, where, &y_code) || y_code != code || y.size(0) != source.size(0) || y.size(1) != dout.size(1)))
    return none_or_error();
  at::Tensor dy, dw;
  if (need_y) dy = at::empty({tokens * k, dout.size(1)}, dout.options());
  if (need_w) dw = at::empty(w.sizes(), w.options());
  const int status = lib.combine_backward(dout.data_ptr(), dout.stride(0), need_w ? y.data_ptr() : nullptr, need_w ? y.stride(0) : 0,
                                          tokens, k, dout.size(1), code, ints(source), ints(place), w.data_ptr(), w_code,
                                          const_cast<void*>(address(dy)), const_cast<void*>(address(dw)), where.stream);
  if (status) return PyLong_FromLong(status);
  const at::Tensor* out[] = {&dy, &dw};
  return pack(out, 2);
  END_HANDLE_TH_ERRORS
}

// embedding_forward(ids, weight, scale, stream, device) -> out
PyObject* embedding_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 5 || !all_tensors(args, 2) || !where.set(args[3], args[4])) return none_or_error();
  const at::Tensor &ids = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  const double scale = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) return nullptr;
  uint32_t code;
  int32_t bytes;
  if (!ids_of(ids, where, &bytes) || !matrix(w, where, &code) || w.size(0) == 0 || !(std::fabs(scale) <= FLT_MAX)) return none_or_error();
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(w.size(1));
  const at::Tensor out = at::empty(shape, w.options());
  const int status = lib.embedding(ids.data_ptr(), bytes, ids.numel(), w.data_ptr(), w.stride(0), w.size(0), w.size(1), code,
                                   static_cast<float>(scale), out.data_ptr(), where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// embedding_weight_grad(dy, ids, vocab, scale, fp32, stream, device) -> dW
PyObject* embedding_weight_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 7 || !all_tensors(args, 2) || !PyLong_Check(args[2]) || !where.set(args[5], args[6])) return none_or_error();
  const at::Tensor &dy = THPVariable_Unpack(args[0]), &ids = THPVariable_Unpack(args[1]);
  const long vocab = PyLong_AsLong(args[2]);
  const double scale = PyFloat_AsDouble(args[3]);
  const bool fp32 = args[4] == Py_True;
  if (PyErr_Occurred()) return nullptr;
  uint32_t code;
  int32_t bytes;
  if (!ids_of(ids, where, &bytes) || !where.has(dy) || !dtype_code(dy, &code) || dy.dim() != ids.dim() + 1 || !dy.is_contiguous() ||
      dy.numel() == 0 || dy.sizes().slice(0, ids.dim()) != ids.sizes() || vocab < 1 || vocab >= INT32_MAX || !(std::fabs(scale) <= FLT_MAX))
    return none_or_error();
  const int64_t n = ids.numel(), width = dy.size(-1), need = lib.embedding_grad_workspace(n, vocab, width);
  if (need < 0) return PyLong_FromLong(static_cast<long>(-need));
  const at::Tensor dw = at::empty({vocab, width}, fp32 ? dy.options().dtype(at::kFloat) : dy.options());
  at::Tensor ws;
  const int status = lib.embedding_grad(dy.data_ptr(), width, ids.data_ptr(), bytes, n, vocab, width, code, static_cast<float>(scale),
                                        dw.data_ptr(), fp32 ? 0 : code, space(need, dy, &ws), where.stream);
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(dw);
  END_HANDLE_TH_ERRORS
}

// rows, weights and targets of a linear head
struct Head {
  int64_t n, width, vocab;
  uint32_t code;
  int32_t bytes;
  bool set(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target, const Where& where) {
    if (!where.has(x) || !dtype_code(x, &code) || code == 0 || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous() ||
        !where.has(w) || w.scalar_type() != x.scalar_type() || w.dim() != 2 || w.size(0) == 0 || w.stride(1) != 1 ||
        w.size(1) != x.size(-1) || !ids_of(target, where, &bytes) || target.sizes() != x.sizes().slice(0, x.dim() - 1))
      return false;
    width = x.size(-1), n = x.numel() / width, vocab = w.size(0);
    return true;
  }
};

// head_forward(x, weight, target, ignore_index, reduction, stream, device) -> (loss, lse, total)
PyObject* head_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 7 || !all_tensors(args, 3) || !where.set(args[5], args[6])) return none_or_error();
  const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]), &target = THPVariable_Unpack(args[2]);
  const long long ignore = PyLong_AsLongLong(args[3]);
  const long reduction = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  Head h;
  if (!h.set(x, w, target, where)) return none_or_error();
  const int64_t need = lib.head_workspace(w.data_ptr(), w.stride(0), h.n, h.width, h.vocab, 0);
  if (need < 0) return PyLong_FromLong(static_cast<long>(-need));
  const auto options = x.options().dtype(at::kFloat);
  const at::Tensor loss = at::empty(target.sizes(), options), lse = at::empty(target.sizes(), options);
  at::Tensor total, ws;
  if (reduction) total = at::empty({}, options);
  const int status = lib.head_forward(x.data_ptr(), h.width, h.n, h.width, w.data_ptr(), w.stride(0), h.vocab, h.code,
                                      target.data_ptr(), h.bytes, ignore, static_cast<float*>(loss.data_ptr()),
                                      static_cast<float*>(lse.data_ptr()), static_cast<int32_t>(reduction),
                                      static_cast<float*>(const_cast<void*>(address(total))), space(need, x, &ws), where.stream);
  if (status) return PyLong_FromLong(status);
  const at::Tensor* out[] = {&loss, &lse, &total};
  return pack(out, 3);
  END_HANDLE_TH_ERRORS
}

// head_backward(dloss, stride, mean, x, weight, target, lse, ignore_index, need_x, need_w, stream, device) -> (dx, dw)
PyObject* head_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Where where;
  if (nargs != 12 || !THPVariable_Check(args[0]) || !all_tensors(args + 3, 4) || !where.set(args[10], args[11]))
    return none_or_error();
  const at::Tensor &dloss = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[3]), &w = THPVariable_Unpack(args[4]),
                   &target = THPVariable_Unpack(args[5]), &lse = THPVariable_Unpack(args[6]);
  const long stride = PyLong_AsLong(args[1]), mean = PyLong_AsLong(args[2]);
  const long long ignore = PyLong_AsLongLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const int need_x = PyObject_IsTrue(args[8]), need_w = PyObject_IsTrue(args[9]);
  if (need_x < 0 || need_w < 0) return nullptr;
  Head h;
  if ((!need_x && !need_w) || !h.set(x, w, target, where) || !where.has(dloss) || dloss.scalar_type() != at::kFloat ||
      (stride ? dloss.numel() != h.n || !dloss.is_contiguous() : dloss.numel() < 1) || !where.has(lse) ||
      lse.scalar_type() != at::kFloat || lse.numel() != h.n || !lse.is_contiguous())
    return none_or_error();
  const int64_t need = lib.head_workspace(w.data_ptr(), w.stride(0), h.n, h.width, h.vocab, (need_x ? 1 : 0) | (need_w ? 2 : 0));
  if (need < 0) return PyLong_FromLong(static_cast<long>(-need));
  at::Tensor dx, dw, ws;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_w) dw = at::empty({h.vocab, h.width}, w.options());
  const int status = lib.head_backward(static_cast<const float*>(dloss.data_ptr()), stride, static_cast<int32_t>(mean), x.data_ptr(),
                                       h.width, h.n, h.width, w.data_ptr(), w.stride(0), h.vocab, h.code, target.data_ptr(),
                                       h.bytes, ignore, static_cast<const float*>(lse.data_ptr()), const_cast<void*>(address(dx)),
                                       const_cast<void*>(address(dw)), space(need, x, &ws), where.stream);
  if (status) return PyLong_FromLong(status);
  const at::Tensor* out[] = {&dx, &dw};
  return pack(out, 2);
  END_HANDLE_TH_ERRORS
}

template <class F> PyCFunction fast(F* f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef kMethods[] = {
    {"bind", fast(bind), METH_FASTCALL, "The addresses of the library's entry points."},
    {"layer_norm_forward", fast(layer_norm_forward), METH_FASTCALL, "The usual call, or None."},
    {"layer_norm_backward", fast(layer_norm_backward), METH_FASTCALL, "The usual call, or None."},
    {"expert_rows", fast(expert_rows), METH_FASTCALL, "The usual call, or None."},
    {"expert_weight_grad", fast(expert_weight_grad), METH_FASTCALL, "The usual call, or None."},
    {"clip_grads", fast(clip_grads), METH_FASTCALL, "The usual call, or None."},
    {"expert_order", fast(expert_order), METH_FASTCALL, "The usual call, or None."},
    {"expert_dispatch", fast(expert_dispatch), METH_FASTCALL, "The usual call, or None."},
    {"expert_combine", fast(expert_combine), METH_FASTCALL, "The usual call, or None."},
    {"expert_combine_backward", fast(expert_combine_backward), METH_FASTCALL, "The usual call, or None."},
    {"embedding_forward", fast(embedding_forward), METH_FASTCALL, "The usual call, or None."},
    {"embedding_weight_grad", fast(embedding_weight_grad), METH_FASTCALL, "The usual call, or None."},
    {"head_forward", fast(head_forward), METH_FASTCALL, "The usual call, or None."},
    {"head_backward", fast(head_backward), METH_FASTCALL, "The usual call, or None."},
    {"clip_table", fast(clip_table), METH_FASTCALL,
     "Fill the table of a clip by the global norm from lists of tensors."},
    {"snapshot", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(snapshot)), METH_FASTCALL,
     "Record data pointers and dtypes of a list of tensors."},
    {"scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scan)), METH_FASTCALL,
     "Check a step plan's tensors against the recorded pointers; returns a status code."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", "Per-step host scan of step-plan tensors.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
