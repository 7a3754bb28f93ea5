// Host side of the per-token operators in native code: the contract checks, the
// allocation of results and workspaces, and the marshalling of one library call,
// which in Python cost more than the kernels of a small decode step take (the
// same checks and ctypes calls took 40-60 us per append or attention call).
//
// Every function here is the fast path of one Python function and only ever
// answers "done" or "not mine" (None): whatever it does not serve, malformed
// arguments among it, goes through the Python path, which raises the errors.  C++
// exceptions (no memory, a tensor without storage, a device that cannot be set) leave as
// the Python exceptions that torch's own functions raise for them, and every tensor whose
// address goes to the library is held until the call returns.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../include/winnow_tq.h"

namespace {

PyObject *g_backend_error = nullptr;         // winnow_b200._lib.BackendError
struct Names {
  PyObject *k_pages, *k_norms, *v_pages, *v_norms, *page_table, *seq_lens, *k_quant, *v_quant, *head_dim, *Pi,
      *centroids, *boundaries, *bit_width;
} N;

// A new reference that is dropped at the end of the scope.
struct Ref {
  PyObject *o;
  explicit Ref(PyObject *p) : o(p) {
    if (!o) PyErr_Clear();
  }
  Ref(const Ref &) = delete;
  ~Ref() { Py_XDECREF(o); }
  explicit operator bool() const { return o != nullptr; }
};

// The interpreter lock is given up while the library launches (a full launch queue blocks).
struct Unlocked {
  PyThreadState *s;
  Unlocked() : s(PyEval_SaveThread()) {}
  Unlocked(const Unlocked &) = delete;
  ~Unlocked() { PyEval_RestoreThread(s); }
};

bool tensor(PyObject *o, at::Tensor &t) {
  if (o == nullptr || !THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return t.defined() && t.layout() == at::kStrided;
}
bool tensor_attr(PyObject *owner, PyObject *name, at::Tensor &t) {
  Ref a(PyObject_GetAttr(owner, name));
  return a && tensor(a.o, t);
}
bool int_attr(PyObject *owner, PyObject *name, int64_t &v) {
  Ref a(PyObject_GetAttr(owner, name));
  if (!a || !PyLong_Check(a.o)) return false;
  v = PyLong_AsLongLong(a.o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? WTQ_F32 : t == at::kHalf ? WTQ_F16 : t == at::kBFloat16 ? WTQ_BF16 : -1;
}
bool width_ok(int64_t bw, int64_t D) {
  return (bw == 2 || bw == 3 || bw == 4 || bw == 5 || bw == 6 || bw == 8) && D * bw % 8 == 0;
}

// Pages and norms of one side: (P, Hkv, S, NB) uint8 with contiguous (S, NB) rows, (P, Hkv, S) fp16.
bool side_pages(const at::Tensor &pages, const at::Tensor &norms, int64_t bw, int64_t D, wtq_side_t &s) {
  if (pages.dim() != 4 || norms.dim() != 3 || pages.scalar_type() != at::kByte || norms.scalar_type() != at::kHalf)
    return false;
  const int64_t nb = D * bw / 8;
  if (!width_ok(bw, D) || pages.size(3) != nb || pages.stride(3) != 1 || pages.stride(2) != nb || norms.stride(2) != 1)
    return false;
  for (int i = 0; i < 3; ++i)
    if (norms.size(i) != pages.size(i)) return false;
  s.pages = (uint8_t *)pages.data_ptr();
  s.norms = norms.data_ptr();
  s.page_stride = pages.stride(0);
  s.head_stride = pages.stride(1);
  s.norm_page_stride = norms.stride(0);
  s.norm_head_stride = norms.stride(1);
  s.bw = (int)bw;
  return true;
}

// The rotation and one table of a quantizer (`table`: centroids or boundaries).
struct Quant {
  int64_t bw = 0;
  at::Tensor pi, tab;
};
bool quant_table(PyObject *quant, PyObject *table, int64_t D, int64_t extra, const at::Device &dev, Quant &held,
                 const float *&Pi, const float *&values) {
  int64_t &bw = held.bw;
  at::Tensor &pi = held.pi, &tab = held.tab;
  if (!int_attr(quant, N.bit_width, bw) || bw < 1 || bw > 8 || !tensor_attr(quant, N.Pi, pi) ||
      !tensor_attr(quant, table, tab))
    return false;
  if (pi.scalar_type() != at::kFloat || pi.dim() != 2 || pi.size(0) != D || pi.size(1) != D || !pi.is_contiguous() ||
      pi.device() != dev)
    return false;
  if (tab.scalar_type() != at::kFloat || tab.numel() != ((int64_t)1 << bw) - extra || !tab.is_contiguous() ||
      tab.device() != dev)
    return false;
  Pi = pi.const_data_ptr<float>();
  values = tab.const_data_ptr<float>();
  return true;
}

bool table_and_lengths(const at::Tensor &table, const at::Tensor &lens, int64_t B, const at::Device &dev) {
  return table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt && table.stride(1) == 1 &&
         lens.dim() == 1 && lens.size(0) == B && lens.scalar_type() == at::kInt && lens.is_contiguous() &&
         table.device() == dev && lens.device() == dev;
}

// One layer's paged packed K/V (a PackedKV) for queries of head_dim D on `dev`.
struct Layer {
  wtq_side_t k, v;
  at::Tensor kp, kn, vp, vn, table, lens;
  Quant k_quant, v_quant;
  int64_t P, Hkv, S;
};
bool read_layer(PyObject *kv, int64_t B, int64_t D, const at::Device &dev, Layer &l) {
  int64_t head_dim = 0;
  at::Tensor &kp = l.kp, &kn = l.kn, &vp = l.vp, &vn = l.vn;
  if (!int_attr(kv, N.head_dim, head_dim) || head_dim != D || D < 1 || D > 256) return false;
  if (!tensor_attr(kv, N.k_pages, kp) || !tensor_attr(kv, N.k_norms, kn) || !tensor_attr(kv, N.v_pages, vp) ||
      !tensor_attr(kv, N.v_norms, vn) || !tensor_attr(kv, N.page_table, l.table) || !tensor_attr(kv, N.seq_lens, l.lens))
    return false;
  if (kp.device() != dev || kn.device() != dev || vp.device() != dev || vn.device() != dev ||
      !table_and_lengths(l.table, l.lens, B, dev))
    return false;
  Ref kq(PyObject_GetAttr(kv, N.k_quant)), vq(PyObject_GetAttr(kv, N.v_quant));
  l.k.bounds = l.v.bounds = nullptr;
  if (!kq || !vq || !quant_table(kq.o, N.centroids, D, 0, dev, l.k_quant, l.k.Pi, l.k.centroids) ||
      !quant_table(vq.o, N.centroids, D, 0, dev, l.v_quant, l.v.Pi, l.v.centroids))
    return false;
  if (!side_pages(kp, kn, l.k_quant.bw, D, l.k) || !side_pages(vp, vn, l.v_quant.bw, D, l.v)) return false;
  for (int i = 0; i < 3; ++i)
    if (kp.size(i) != vp.size(i)) return false;
  l.P = kp.size(0);
  l.Hkv = kp.size(1);
  l.S = kp.size(2);
  return l.P >= 1 && l.Hkv >= 1 && l.S >= 1 && l.table.size(1) >= 1;
}

bool optional_status(PyObject *o, const at::Device &dev, at::Tensor &t, int32_t *&p) {
  p = nullptr;
  if (o == Py_None) return true;
  if (!tensor(o, t) || t.scalar_type() != at::kInt || t.numel() < 1 || t.device() != dev) return false;
  p = t.mutable_data_ptr<int32_t>();
  return true;
}

PyObject *library_error(int rc) {
  PyErr_Format(g_backend_error ? g_backend_error : PyExc_RuntimeError, "libwinnow_tq error %d: %s", rc, wtq_last_error());
  return nullptr;
}

// One decode call: q (B, Hq, 1, D).  `out` / `ws` / `status_arg` may be None; without `out` the result is a new
// tensor, (B, Hq, 1, D) or, with `token_major`, (B, 1, Hq, D).
PyObject *run_decode(PyObject *q_arg, PyObject *kv, PyObject *scale_arg, long splits, PyObject *out_arg, PyObject *ws_arg,
                     PyObject *status_arg, bool token_major) {
  at::Tensor q, out, ws, status_tensor;
  if (!tensor(q_arg, q) || !q.is_cuda() || q.dim() != 4 || q.size(2) != 1 || q.stride(3) != 1) Py_RETURN_NONE;
  const int dtype = dtype_code(q.scalar_type());
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(3);
  const at::Device dev = q.device();
  Layer l;
  int32_t *status;
  if (dtype < 0 || B < 1 || Hq < 1 || !read_layer(kv, B, D, dev, l) || Hq % l.Hkv ||
      !optional_status(status_arg, dev, status_tensor, status))
    Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(scale_arg);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (out_arg != Py_None) {
    if (!tensor(out_arg, out) || out.dim() != 4 || out.size(0) != B || out.size(1) != Hq || out.size(2) != 1 ||
        out.size(3) != D || out.stride(3) != 1 || out.scalar_type() != q.scalar_type() || out.device() != dev)
      Py_RETURN_NONE;
  }
  if (ws_arg != Py_None && (!tensor(ws_arg, ws) || ws.device() != dev)) Py_RETURN_NONE;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  int64_t os[2] = {Hq * D, D};
  if (out.defined()) {
    os[0] = out.stride(0);
    os[1] = out.stride(1);
  } else {
    out = token_major ? at::empty({B, 1, Hq, D}, q.options()) : at::empty({B, Hq, 1, D}, q.options());
  }
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int64_t qs[2] = {q.stride(0), q.stride(1)};
  const int W = (int)l.table.size(1), S = (int)l.S, H = (int)l.Hkv;
  int rc = WTQ_ERR_UNSUPPORTED;
  if (splits <= 0 && !ws.defined()) {
    const Unlocked u;
    rc = wtq_decode_direct(q.const_data_ptr(), dtype, qs, out.mutable_data_ptr(), os, &l.k, &l.v,
                           l.table.const_data_ptr<int32_t>(), l.table.stride(0), l.lens.const_data_ptr<int32_t>(),
                           (float)scale, (int)B, (int)Hq, H, (int)D, S, (int)l.P, W, status, stream);
  }
  if (rc == WTQ_ERR_UNSUPPORTED) {
    if (!ws.defined()) {
      ws = at::empty({(int64_t)wtq_decode_workspace_bytes((int)B, (int)Hq, H, (int)D, W, S, (int)splits)},
                     q.options().dtype(at::kByte));
      ws.narrow(0, 0, (int64_t)wtq_decode_counter_bytes((int)B, H)).zero_();
    }
    const Unlocked u;
    rc = wtq_decode(q.const_data_ptr(), dtype, qs, out.mutable_data_ptr(), os, &l.k, &l.v,
                    l.table.const_data_ptr<int32_t>(), l.table.stride(0), l.lens.const_data_ptr<int32_t>(),
                    (float)scale, (int)B, (int)Hq, H, (int)D, S, (int)l.P, W, (int)splits, ws.mutable_data_ptr(),
                    (size_t)ws.numel(), status, stream);
  }
  if (rc) return library_error(rc);
  if (out_arg != Py_None) {
    Py_INCREF(out_arg);
    return out_arg;
  }
  return THPVariable_Wrap(std::move(out));
}

// decode(q, kv, scale, num_splits, out, workspace, status) -> out, or None
PyObject *decode(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !PyLong_Check(a[3])) Py_RETURN_NONE;
  const long splits = PyLong_AsLong(a[3]);
  if (splits == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  return run_decode(a[0], a[1], a[2], splits, a[4], a[5], a[6], false);
  END_HANDLE_TH_ERRORS
}

// attend(q, kv, scale, status) -> (B, 1, Hq, D), the layout attention interfaces hand back, or None
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  return run_decode(a[0], a[1], a[2], 0, Py_None, Py_None, a[3], true);
  END_HANDLE_TH_ERRORS
}

// append(k, v, k_pages, k_norms, v_pages, v_norms, page_table, seq_lens, k_tq, v_tq, order, status) -> True, or None
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor k, v, kp, kn, vp, vn, table, lens, status_tensor;
  Quant k_quant, v_quant;
  if (n != 12 || !tensor(a[0], k) || !tensor(a[1], v) || !tensor(a[2], kp) || !tensor(a[3], kn) || !tensor(a[4], vp) ||
      !tensor(a[5], vn) || !tensor(a[6], table) || !tensor(a[7], lens))
    Py_RETURN_NONE;
  const at::Device dev = k.device();
  if (!k.is_cuda() || k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() ||
      k.stride(3) != 1 || v.stride(3) != 1 || v.device() != dev)
    Py_RETURN_NONE;
  const int dtype = dtype_code(k.scalar_type());
  const int64_t B = k.size(0), Hkv = k.size(1), tokens = k.size(2), D = k.size(3);
  if (dtype < 0 || B < 1 || Hkv < 1 || tokens < 1 || D < 1 || D > 256) Py_RETURN_NONE;
  wtq_side_t sk, sv;
  int32_t *status;
  sk.centroids = sv.centroids = nullptr;
  if (kp.device() != dev || kn.device() != dev || vp.device() != dev || vn.device() != dev ||
      !table_and_lengths(table, lens, B, dev) || !quant_table(a[8], N.boundaries, D, 1, dev, k_quant, sk.Pi, sk.bounds) ||
      !quant_table(a[9], N.boundaries, D, 1, dev, v_quant, sv.Pi, sv.bounds) || !side_pages(kp, kn, k_quant.bw, D, sk) ||
      !side_pages(vp, vn, v_quant.bw, D, sv) || !optional_status(a[11], dev, status_tensor, status) || kp.size(1) != Hkv ||
      table.size(1) < 1)
    Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (kp.size(i) != vp.size(i)) Py_RETURN_NONE;
  const long order = PyLong_AsLong(a[10]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)}, vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    const Unlocked u;
    rc = wtq_append(k.const_data_ptr(), v.const_data_ptr(), dtype, ks, vs, &sk, &sv, table.const_data_ptr<int32_t>(),
                    table.stride(0), lens.const_data_ptr<int32_t>(), (int)B, (int)Hkv, (int)tokens, (int)D,
                    (int)kp.size(2), (int)kp.size(0), (int)table.size(1), (int)order, status, stream);
  }
  if (rc) return library_error(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// stage(dst, src, dst, src, dst, src) -> True, or None: copies of contiguous tensors of equal type and size
// (a pair of None: nothing to copy)
PyObject *stage(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor held[3][2];
  void *dst[3] = {};
  const void *src[3] = {};
  int64_t bytes[3] = {};
  at::Device dev(at::kCPU);
  if (n != 6) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i) {
    if (a[2 * i + 1] == Py_None) continue;
    at::Tensor &d = held[i][0], &s = held[i][1];
    if (!tensor(a[2 * i], d) || !tensor(a[2 * i + 1], s) || !d.is_cuda() || s.device() != d.device() ||
        d.scalar_type() != s.scalar_type() || d.sizes() != s.sizes() || !d.is_contiguous() || !s.is_contiguous() ||
        (dev.is_cuda() && dev != d.device()))
      Py_RETURN_NONE;
    dev = d.device();
    dst[i] = d.mutable_data_ptr();
    src[i] = s.const_data_ptr();
    bytes[i] = (int64_t)d.nbytes();
    if ((((uintptr_t)dst[i] | (uintptr_t)src[i]) & 15) != 0) Py_RETURN_NONE;
  }
  if (!dev.is_cuda()) Py_RETURN_TRUE;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    const Unlocked u;
    rc = wtq_stage(dst, src, bytes, stream);
  }
  if (rc) return library_error(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (a tangent of forward-mode differentiation is there whatever the mode of the backward one)
bool needs_grad(const at::Tensor &t) {
  return t.defined() && ((t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined());
}
bool optional(PyObject *o, at::Tensor &t) { return o == Py_None || tensor(o, t); }
bool words(const at::Tensor &t, const at::Device &dev, at::IntArrayRef shape) {
  return t.scalar_type() == at::kInt && t.device() == dev && t.sizes() == shape && t.is_contiguous();
}
PyObject *tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject *r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor &t : ts) {
    PyObject *o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// `shape` of one buffer's elements from `at` on, which moves past them (a tensor of its own, without the
// dispatcher: nine allocations or views of a plan cost as much as its kernel).
at::Tensor cut(const at::Tensor &buffer, int64_t &at, at::IntArrayRef shape) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  at += (t.numel() + 63) / 64 * 64;
  return t;
}

// rope(q, k, v, positions, table, q_weight, k_weight, eps, interleaved, out, status) -> (q, k[, v]), or None
PyObject *rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor x[3], y[3], w[2], positions, table, status_tensor;
  if (n != 11 || !tensor(a[0], x[0]) || !tensor(a[1], x[1]) || !optional(a[2], x[2]) || !tensor(a[3], positions) ||
      !tensor(a[4], table) || !optional(a[5], w[0]) || !optional(a[6], w[1]) || !PyFloat_Check(a[7]) || !PyBool_Check(a[8]))
    Py_RETURN_NONE;
  const int sides = x[2].defined() ? 3 : 2;
  const at::Tensor &q = x[0];
  const at::Device dev = q.device();
  if (!q.is_cuda() || q.dim() != 4) Py_RETURN_NONE;
  const int dtype = dtype_code(q.scalar_type());
  const int64_t B = q.size(0), tokens = q.size(2), D = q.size(3);
  int32_t *status;
  if (dtype < 0 || B < 1 || tokens < 1 || D < 2 || !optional_status(a[10], dev, status_tensor, status)) Py_RETURN_NONE;
  for (int i = 0; i < sides; ++i)
    if (x[i].dim() != 4 || x[i].device() != dev || x[i].scalar_type() != q.scalar_type() || x[i].size(0) != B ||
        x[i].size(1) < 1 || x[i].size(2) != tokens || x[i].size(3) != D || x[i].stride(3) != 1 || needs_grad(x[i]))
      Py_RETURN_NONE;
  if (sides == 3 && x[2].size(1) != x[1].size(1)) Py_RETURN_NONE;
  int weight_dtype = dtype;
  for (int i = 0; i < 2; ++i) {
    if (!w[i].defined()) continue;
    if (w[i].dim() != 1 || w[i].size(0) != D || !w[i].is_contiguous() || w[i].device() != dev || needs_grad(w[i]))
      Py_RETURN_NONE;
    weight_dtype = dtype_code(w[i].scalar_type());
    if (weight_dtype < 0 || (w[0].defined() && w[i].scalar_type() != w[0].scalar_type())) Py_RETURN_NONE;
  }
  if (positions.dim() != 2 || positions.size(0) != B || positions.size(1) != tokens || positions.stride(1) != 1 ||
      positions.scalar_type() != at::kInt || positions.device() != dev || needs_grad(table) || table.dim() != 2 || table.stride(1) != 1 ||
      table.scalar_type() != at::kFloat || table.device() != dev || table.size(1) > D || table.size(1) % 2)
    Py_RETURN_NONE;
  const bool given = a[9] != Py_None;
  if (given) {                            // buffers of their own, else the Python path looks closer
    if (!PyTuple_Check(a[9]) || PyTuple_GET_SIZE(a[9]) != sides) Py_RETURN_NONE;
    for (int i = 0; i < sides; ++i) {
      if (!tensor(PyTuple_GET_ITEM(a[9], i), y[i]) || y[i].sizes() != x[i].sizes() || y[i].stride(3) != 1 ||
          y[i].scalar_type() != q.scalar_type() || y[i].device() != dev || !y[i].is_non_overlapping_and_dense())
        Py_RETURN_NONE;
      for (int j = 0; j < sides; ++j)
        if (y[i].storage().data() == x[j].storage().data() || (j < i && y[i].storage().data() == y[j].storage().data()))
          Py_RETURN_NONE;
    }
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  for (int i = 0; i < sides && !given; ++i) y[i] = at::empty(x[i].sizes(), q.options());
  wtq_rope_side_t s[3] = {};
  for (int i = 0; i < sides; ++i) {
    s[i].x = x[i].const_data_ptr();
    s[i].out = y[i].mutable_data_ptr();
    for (int d = 0; d < 3; ++d) {
      s[i].strides[d] = x[i].stride(d);
      s[i].out_strides[d] = y[i].stride(d);
    }
    s[i].weight = i < 2 && w[i].defined() ? w[i].const_data_ptr() : nullptr;
    s[i].heads = (int)x[i].size(1);
  }
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const float eps = (float)PyFloat_AS_DOUBLE(a[7]);
  const int turned = a[8] == Py_True;
  int rc;
  {
    const Unlocked u;
    rc = wtq_qk_norm_rope(s, dtype, weight_dtype, eps, positions.const_data_ptr<int32_t>(), positions.stride(0),
                          table.const_data_ptr<float>(), table.stride(0), (int)table.size(0), (int)B, (int)tokens, (int)D,
                          (int)table.size(1), turned, status, stream);
  }
  if (rc) return library_error(rc);
  return sides == 3 ? tuple_of({y[0], y[1], y[2]}) : tuple_of({y[0], y[1]});
  END_HANDLE_TH_ERRORS
}

// plan(lengths, new_tokens, table, held, free_pages, free_count, page_size, tokens, parents, out, ticket, status)
// -> the nine tensors of a TokenPlan, or None
PyObject *plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor lengths, fresh, table, held, free_pages, free_count, parents, ticket, status_tensor, o[9];
  if (n != 12 || !tensor(a[0], lengths) || !optional(a[1], fresh) || !tensor(a[2], table) || !tensor(a[3], held) ||
      !tensor(a[4], free_pages) || !tensor(a[5], free_count) || !PyLong_Check(a[6]) || !PyLong_Check(a[7]) ||
      !optional(a[8], parents) || !optional(a[10], ticket))
    Py_RETURN_NONE;
  const int64_t S = PyLong_AsLongLong(a[6]), tokens = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const at::Device dev = lengths.device();
  int32_t *status;
  if (!lengths.is_cuda() || table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != dev ||
      table.stride(1) != 1 || table.size(1) < 1 || S < 1 || S > INT32_MAX || tokens < 0 || tokens > INT32_MAX ||
      !optional_status(a[11], dev, status_tensor, status))
    Py_RETURN_NONE;
  const int64_t B = table.size(0), W = table.size(1);
  const int64_t Q = parents.defined() ? (parents.dim() == 2 ? parents.size(1) : 0) : 0, words_of = (Q + 31) / 32;
  if (B < 1 || W > INT32_MAX || (B > 1 && table.stride(0) < W) || !words(lengths, dev, {B}) || !words(held, dev, {B}) ||
      !words(free_count, dev, {1}) || free_pages.dim() != 1 || !words(free_pages, dev, {free_pages.size(0)}) ||
      free_pages.size(0) > INT32_MAX || (ticket.defined() && !words(ticket, dev, {1})))
    Py_RETURN_NONE;
  if (parents.defined()) {
    if (Q < 1 || parents.size(0) != B || parents.scalar_type() != at::kInt || parents.device() != dev ||
        parents.stride(1) != 1 || B * Q != tokens || fresh.defined())
      Py_RETURN_NONE;
  } else if (!fresh.defined() || !words(fresh, dev, {B})) {
    Py_RETURN_NONE;
  }
  const bool given = a[9] != Py_None;
  if (given) {
    if (!PyTuple_Check(a[9]) || PyTuple_GET_SIZE(a[9]) != 9 || !ticket.defined()) Py_RETURN_NONE;
    for (int i = 0; i < 9; ++i)
      if (!optional(PyTuple_GET_ITEM(a[9], i), o[i]) || (i < 8 && !o[i].defined())) Py_RETURN_NONE;
    if (!words(o[0], dev, {B}) || !words(o[1], dev, {B}) || !words(o[2], dev, {1}) || !words(o[3], dev, {B + 1}) ||
        !words(o[4], dev, {tokens}) || !words(o[5], dev, {tokens}) || !words(o[6], dev, {tokens, 1}) ||
        !words(o[7], dev, {tokens}) || (parents.defined() && (!o[8].defined() || !words(o[8], dev, {B, Q, words_of}))))
      Py_RETURN_NONE;
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (!given) {
    const at::Tensor buffer = at::empty({9 * 64 + 3 * B + 2 + 4 * tokens + B * Q * words_of}, lengths.options());
    int64_t at = 0;
    o[0] = cut(buffer, at, {B});
    o[1] = cut(buffer, at, {B});
    o[2] = cut(buffer, at, {1});
    o[3] = cut(buffer, at, {B + 1});
    o[4] = cut(buffer, at, {tokens});
    o[5] = cut(buffer, at, {tokens});
    o[6] = cut(buffer, at, {tokens, 1});
    o[7] = cut(buffer, at, {tokens});
    if (parents.defined()) o[8] = cut(buffer, at, {B, Q, words_of});
  }
  int32_t *p[9];
  for (int i = 0; i < 9; ++i) p[i] = o[i].defined() ? o[i].mutable_data_ptr<int32_t>() : nullptr;
  const wtq_plan_t out = {p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8]};
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    const Unlocked u;
    rc = wtq_plan_tokens(lengths.const_data_ptr<int32_t>(), fresh.defined() ? fresh.const_data_ptr<int32_t>() : nullptr,
                         parents.defined() ? parents.const_data_ptr<int32_t>() : nullptr,
                         parents.defined() ? parents.stride(0) : 0, table.mutable_data_ptr<int32_t>(), table.stride(0),
                         held.const_data_ptr<int32_t>(), free_pages.const_data_ptr<int32_t>(),
                         free_count.const_data_ptr<int32_t>(), (int)B, (int)W, (int)S, (int)tokens, (int)Q,
                         (int)free_pages.size(0), &out, ticket.defined() ? ticket.mutable_data_ptr<int32_t>() : nullptr,
                         status, stream);
  }
  if (rc) return library_error(rc);
  return tuple_of({o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7], o[8]});
  END_HANDLE_TH_ERRORS
}

// tree(q, kv, mask, scale, out, workspace, status) -> out, or None
PyObject *tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor q, mask, out, ws, status_tensor;
  if (n != 7 || !tensor(a[0], q) || !tensor(a[2], mask) || !q.is_cuda() || q.dim() != 4 || q.stride(3) != 1 ||
      q._fw_grad(0).defined())
    Py_RETURN_NONE;
  const int dtype = dtype_code(q.scalar_type());
  const int64_t B = q.size(0), Hq = q.size(1), Q = q.size(2), D = q.size(3);
  const at::Device dev = q.device();
  Layer l;
  int32_t *status;
  if (dtype < 0 || B < 1 || Hq < 1 || Q < 1 || !read_layer(a[1], B, D, dev, l) || Hq % l.Hkv ||
      !optional_status(a[6], dev, status_tensor, status))
    Py_RETURN_NONE;
  if (mask.dim() != 3 || mask.size(0) != B || mask.size(1) != Q || mask.size(2) != (Q + 31) / 32 ||
      mask.stride(2) != 1 || mask.scalar_type() != at::kInt || mask.device() != dev)
    Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (a[4] != Py_None && (!tensor(a[4], out) || out.dim() != 4 || out.size(0) != B || out.size(1) != Hq ||
                          out.size(2) != Q || out.size(3) != D || out.stride(3) != 1 ||
                          out.scalar_type() != q.scalar_type() || out.device() != dev))
    Py_RETURN_NONE;
  if (a[5] != Py_None && (!tensor(a[5], ws) || ws.device() != dev || ws.scalar_type() != at::kByte || !ws.is_contiguous()))
    Py_RETURN_NONE;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const bool fresh = !out.defined();
  if (fresh) out = at::empty({B, Q, Hq, D}, q.options()).transpose(1, 2);
  if (!ws.defined())
    ws = at::empty({(int64_t)wtq_tree_workspace_bytes((int)B, (int)Hq, (int)l.Hkv, (int)Q, (int)D)},
                   q.options().dtype(at::kByte));
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)}, os[3] = {out.stride(0), out.stride(1), out.stride(2)};
  const int64_t ms[2] = {mask.stride(0), mask.stride(1)};
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    const Unlocked u;
    rc = wtq_tree(q.const_data_ptr(), dtype, qs, out.mutable_data_ptr(), os, &l.k, &l.v,
                  l.table.const_data_ptr<int32_t>(), l.table.stride(0), l.lens.const_data_ptr<int32_t>(),
                  mask.const_data_ptr<int32_t>(), ms, (float)scale, (int)B, (int)Hq, (int)l.Hkv, (int)Q, (int)D, (int)l.S,
                  (int)l.P, (int)l.table.size(1), ws.mutable_data_ptr(), (size_t)ws.numel(), status, stream);
  }
  if (rc) return library_error(rc);
  if (!fresh) return Py_NewRef(a[4]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// keep(k_pages, k_norms, v_pages, v_norms, page_table, seq_lens, keep, counts, drafted, granted, out, status) -> lengths,
// or None
PyObject *keep(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor pages[2], norms[2], table, lens, path, counts, granted, out, status_tensor;
  if (n != 12 || !tensor(a[0], pages[0]) || !tensor(a[1], norms[0]) || !tensor(a[2], pages[1]) || !tensor(a[3], norms[1]) ||
      !tensor(a[4], table) || !tensor(a[5], lens) || !tensor(a[6], path) || !tensor(a[7], counts) || !PyLong_Check(a[8]) ||
      !optional(a[9], granted) || !optional(a[10], out))
    Py_RETURN_NONE;
  const int64_t drafted = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const at::Device dev = pages[0].device();
  int32_t *status;
  if (!pages[0].is_cuda() || drafted < 0 || drafted > INT32_MAX || table.dim() != 2 || table.scalar_type() != at::kInt ||
      table.stride(1) != 1 || table.device() != dev || table.size(0) < 1 || table.size(1) < 1 ||
      (granted.defined() && !words(granted, dev, {1})) || !optional_status(a[11], dev, status_tensor, status))
    Py_RETURN_NONE;
  const int64_t B = table.size(0);
  wtq_pool_side_t s[2];
  for (int i = 0; i < 2; ++i) {
    const at::Tensor &p = pages[i], &m = norms[i];
    if (p.dim() != 5 || m.dim() != 4 || p.device() != dev || m.device() != dev || p.scalar_type() != at::kByte ||
        m.scalar_type() != at::kHalf || p.stride(4) != 1 || p.stride(3) != p.size(4) || m.stride(3) != 1 || p.numel() == 0)
      Py_RETURN_NONE;
    for (int d = 0; d < 4; ++d)
      if (m.size(d) != p.size(d) || p.size(d) != pages[0].size(d)) Py_RETURN_NONE;
    s[i] = {(uint8_t *)p.data_ptr(), m.data_ptr(), p.stride(0), p.stride(1), p.stride(2),
            m.stride(0), m.stride(1), m.stride(2), (int)p.size(4)};
  }
  if (!words(lens, dev, {B}) || !words(counts, dev, {B}) || path.dim() != 2 || path.size(0) != B || path.size(1) < 1 ||
      path.stride(1) != 1 || path.scalar_type() != at::kInt || path.device() != dev ||
      (out.defined() && !words(out, dev, {B})))
    Py_RETURN_NONE;
  if (out.defined())                      // memory of its own, else the Python path looks closer
    for (const at::Tensor *t : {&table, &lens, &path, &counts, &granted})
      if (t->defined() && out.storage().data() == t->storage().data()) Py_RETURN_NONE;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (!out.defined()) out = at::empty({B}, lens.options());
  void *stream = (void *)at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  {
    const Unlocked u;
    rc = wtq_keep_tokens(&s[0], &s[1], table.const_data_ptr<int32_t>(), table.stride(0), lens.const_data_ptr<int32_t>(),
                         path.const_data_ptr<int32_t>(), path.stride(0), counts.const_data_ptr<int32_t>(),
                         (int)pages[0].size(0), (int)B, (int)pages[0].size(2), (int)pages[0].size(3),
                         (int)pages[0].size(1), (int)table.size(1), (int)path.size(1), (int)drafted,
                         granted.defined() ? granted.const_data_ptr<int32_t>() : nullptr, out.mutable_data_ptr<int32_t>(),
                         status, stream);
  }
  if (rc) return library_error(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject *set_error(PyObject *, PyObject *type) {
  Py_INCREF(type);
  Py_XSETREF(g_backend_error, type);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"decode", (PyCFunction)(void (*)(void))decode, METH_FASTCALL, "decode(q, kv, scale, num_splits, out, workspace, status)"},
    {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, "attend(q, kv, scale, status)"},
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL,
     "append(k, v, k_pages, k_norms, v_pages, v_norms, page_table, seq_lens, k_tq, v_tq, order, status)"},
    {"stage", (PyCFunction)(void (*)(void))stage, METH_FASTCALL, "stage(dst, src, dst, src, dst, src)"},
    {"rope", (PyCFunction)(void (*)(void))rope, METH_FASTCALL,
     "rope(q, k, v, positions, table, q_weight, k_weight, eps, interleaved, out, status)"},
    {"plan", (PyCFunction)(void (*)(void))plan, METH_FASTCALL,
     "plan(lengths, new_tokens, table, held, free_pages, free_count, page_size, tokens, parents, out, ticket, status)"},
    {"tree", (PyCFunction)(void (*)(void))tree, METH_FASTCALL, "tree(q, kv, mask, scale, out, workspace, status)"},
    {"keep", (PyCFunction)(void (*)(void))keep, METH_FASTCALL,
     "keep(k_pages, k_norms, v_pages, v_norms, page_table, seq_lens, keep, counts, drafted, granted, out, status)"},
    {"set_error", set_error, METH_O, "the exception type library errors are raised as"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "native host side of winnow_b200", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  N.k_pages = PyUnicode_InternFromString("k_pages");
  N.k_norms = PyUnicode_InternFromString("k_norms");
  N.v_pages = PyUnicode_InternFromString("v_pages");
  N.v_norms = PyUnicode_InternFromString("v_norms");
  N.page_table = PyUnicode_InternFromString("page_table");
  N.seq_lens = PyUnicode_InternFromString("seq_lens");
  N.k_quant = PyUnicode_InternFromString("k_quant");
  N.v_quant = PyUnicode_InternFromString("v_quant");
  N.head_dim = PyUnicode_InternFromString("head_dim");
  N.Pi = PyUnicode_InternFromString("Pi");
  N.centroids = PyUnicode_InternFromString("centroids");
  N.boundaries = PyUnicode_InternFromString("boundaries");
  N.bit_width = PyUnicode_InternFromString("bit_width");
  return PyModule_Create(&module);
}
