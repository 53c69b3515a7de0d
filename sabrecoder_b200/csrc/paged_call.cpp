// The paged cache's torch-facing calls into libsabre_b200.so, compiled: the
// argument checks, allocations and strides of kernels.py's paged_store,
// paged_decode, paged_prefill and copy_pages. On the device a small store takes
// 3 us and a small decode 6, so the host's part counts: the same steps in
// Python over ctypes took 15 us a store, 20 a decode, 16 a prefill and 8.6 a
// copy; here 5.1, 8.5, 5.0 and 4.5, of which a launch is 2.
//
// Every function returns None when an argument is not what the kernels take
// (kernels.py then raises with what is wrong), a negative int, the status, when
// the C entry refused or failed (kernels.py raises with its message), else the
// number of kernels launched, attend behind its result.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <vector>

#include "../../include/sabre_b200.h"

namespace {

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool small(int64_t n) { return n >= 0 && n <= INT_MAX; }

// The arguments all paged calls share.
struct Pages {
  const at::Tensor *k, *v, *table, *lens, *starts;  // starts may be null
  int heads, dim, pages, page_size, batch, cols, dtype;
  int64_t ks[3], vs[3];
  c10::DeviceIndex dev;

  bool on(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == dev; }
  bool ints(const at::Tensor* t, int64_t n) const {
    return t && on(*t) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
  }
  // A [N, H, D] tensor of rows.
  bool rows(const at::Tensor* t) const {
    return t && on(*t) && t->scalar_type() == k->scalar_type() && t->dim() == 3 && t->size(2) == dim &&
           t->stride(2) == 1 && small(t->size(0)) && small(t->size(1));
  }

  // False: not what the kernels take.
  bool read(PyObject* kp, PyObject* vp, PyObject* tab, PyObject* sl, PyObject* qs) {
    k = tensor(kp), v = tensor(vp), table = tensor(tab), lens = tensor(sl);
    starts = qs == Py_None ? nullptr : tensor(qs);
    if (!k || !v || !table || !lens || (qs != Py_None && !starts)) return false;
    if (!k->is_cuda() || k->dim() != 4 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type()) return false;
    dev = k->get_device();
    if (k->scalar_type() == at::kBFloat16)
      dtype = SABRE_BF16;
    else if (k->scalar_type() == at::kHalf)
      dtype = SABRE_F16;
    else
      return false;
    for (int i = 0; i < 4; ++i)
      if (!small(k->size(i))) return false;
    pages = k->size(0), heads = k->size(1), page_size = k->size(2), dim = k->size(3);
    for (int i = 0; i < 3; ++i) ks[i] = k->stride(i), vs[i] = v->stride(i);
    if (k->stride(3) != 1 || v->stride(3) != 1 || !on(*v)) return false;
    if (!on(*table) || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(1) < 1 ||
        !small(table->size(0)) || !small(table->size(1)) || (table->size(1) > 1 && table->stride(1) != 1))
      return false;
    batch = table->size(0), cols = table->size(1);
    return ints(lens, batch) && (!starts || ints(starts, int64_t{batch} + 1));
  }
  const int32_t* i32(const at::Tensor* t) const { return t ? static_cast<const int32_t*>(t->const_data_ptr()) : nullptr; }
};

int integer(PyObject* o) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return static_cast<int>(x);
}

float number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(x);
}

PyObject* launched(int status, int64_t kernels) { return PyLong_FromLongLong(status == SABRE_OK ? kernels : status); }

PyObject* result(const at::Tensor& out, int kernels) { return Py_BuildValue("Ni", THPVariable_Wrap(out), kernels); }

// store(k, v, k_pages, v_pages, page_table, seq_lens, q_start) -> kernels
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  if (n != 7 || !p.read(a[2], a[3], a[4], a[5], a[6])) Py_RETURN_NONE;
  const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]);
  if (!p.rows(k) || !p.rows(v) || k->sizes() != v->sizes() || k->size(1) != p.heads) Py_RETURN_NONE;
  const int rows = k->size(0);
  if (!p.starts && rows != p.batch) Py_RETURN_NONE;
  if (rows == 0 || p.batch == 0) return PyLong_FromLong(0);
  const int64_t kr[2] = {k->stride(0), k->stride(1)}, vr[2] = {v->stride(0), v->stride(1)};
  const c10::cuda::CUDAGuard guard(p.dev);
  return launched(sabre_paged_store(k->const_data_ptr(), v->const_data_ptr(), p.k->data_ptr(), p.v->data_ptr(),
                                    p.i32(p.table), p.i32(p.lens), p.i32(p.starts), rows, p.batch, p.heads, p.dim,
                                    p.pages, p.page_size, p.cols, kr, vr, p.ks, p.vs, p.table->stride(0), p.dtype,
                                    c10::cuda::getCurrentCUDAStream(p.dev).stream()),
                  1);
  END_HANDLE_TH_ERRORS
}

// attend(q, k_pages, v_pages, page_table, seq_lens, q_start, window, prefix, scale, out, workspace) ->
// (out, kernels); decode without q_start.
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  if (n != 11 || !p.read(a[1], a[2], a[3], a[4], a[5])) Py_RETURN_NONE;
  const at::Tensor* q = tensor(a[0]);
  if (!p.rows(q) || (!p.starts && q->size(0) != p.batch)) Py_RETURN_NONE;
  const int window = integer(a[6]), prefix = integer(a[7]);
  const float scale = number(a[8]);
  at::Tensor out, ws;
  if (a[9] != Py_None) {
    const at::Tensor* o = tensor(a[9]);
    if (!p.rows(o) || o->sizes() != q->sizes() || at::has_internal_overlap(*o) == at::MemOverlap::Yes) Py_RETURN_NONE;
    out = *o;
  }
  const c10::cuda::CUDAGuard guard(p.dev);
  if (!out.defined()) out = at::empty(q->sizes(), q->options());
  if (q->numel() == 0 || p.batch == 0) return result(out, 0);
  const int rows = q->size(0), heads_q = q->size(1);
  const size_t need = p.starts ? sabre_paged_prefill_workspace_size(rows, p.batch, heads_q, p.heads, p.dim,
                                                                    p.page_size, p.cols, window, prefix)
                               : sabre_paged_decode_workspace_size(p.batch, heads_q, p.heads, p.dim);
  if (a[10] != Py_None) {
    const at::Tensor* w = tensor(a[10]);
    if (!w || !p.on(*w) || !w->is_contiguous() || w->nbytes() < need) Py_RETURN_NONE;
    ws = *w;
  } else if (need > 0) {
    ws = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
  }
  void* const wp = ws.defined() ? ws.data_ptr() : nullptr;
  const size_t wb = ws.defined() ? ws.nbytes() : 0;
  const int64_t qr[2] = {q->stride(0), q->stride(1)}, orr[2] = {out.stride(0), out.stride(1)};
  void* const stream = c10::cuda::getCurrentCUDAStream(p.dev).stream();
  const int st =
      p.starts ? sabre_paged_prefill(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(), out.data_ptr(),
                                     p.i32(p.table), p.i32(p.lens), p.i32(p.starts), rows, p.batch, heads_q, p.heads,
                                     p.dim, p.pages, p.page_size, p.cols, window, prefix, qr, p.ks, p.vs, orr,
                                     p.table->stride(0), scale, p.dtype, wp, wb, stream)
               : sabre_paged_decode(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(), out.data_ptr(),
                                    p.i32(p.table), p.i32(p.lens), p.batch, heads_q, p.heads, p.dim, p.pages,
                                    p.page_size, p.cols, window, prefix, qr, p.ks, p.vs, orr, p.table->stride(0),
                                    scale, p.dtype, wp, wb, stream);
  if (st != SABRE_OK) return PyLong_FromLong(st);
  // Parts are joined by a second kernel: in prompts that run in shares, which is
  // when they ask for a workspace; in decodes over more than one key tile.
  const bool joined = p.starts ? need > 0 : p.batch > 1 || p.heads > 1 || int64_t{p.cols} * p.page_size > 64;
  return result(out, joined ? 2 : 1);
  END_HANDLE_TH_ERRORS
}

// copy(pages, src, dst) -> kernels; src and dst lists of ints.
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* t = n == 3 ? tensor(a[0]) : nullptr;
  if (!t || !t->is_cuda() || t->dim() < 4 || !PyList_Check(a[1]) || !PyList_Check(a[2]) ||
      PyList_GET_SIZE(a[1]) != PyList_GET_SIZE(a[2]))
    Py_RETURN_NONE;
  const int64_t d = t->dim(), moves = PyList_GET_SIZE(a[1]);
  // Each page contiguous, the pools at one stride.
  int64_t unit = 1, buffers = 1, step = 0;
  for (int64_t i = d - 1; i > d - 4; --i) {
    if (t->size(i) > 1 && t->stride(i) != unit) Py_RETURN_NONE;
    unit *= t->size(i);
  }
  for (int64_t i = d - 5; i >= 0; --i) {
    if (t->size(i) > 1 && buffers > 1 && t->stride(i) != buffers * step) Py_RETURN_NONE;
    if (t->size(i) > 1 && buffers == 1) step = t->stride(i);
    buffers *= t->size(i);
  }
  const int64_t pages = t->size(d - 4), es = t->element_size();
  if (!small(pages) || !small(buffers) || !small(moves)) Py_RETURN_NONE;
  std::vector<int32_t> ids(2 * moves);
  for (int64_t i = 0; i < 2 * moves; ++i) {
    const int64_t id = PyLong_AsLongLong(PyList_GET_ITEM(a[1 + i / moves], i % moves));
    if (id == -1 && PyErr_Occurred()) throw python_error();
    if (id < 0 || id >= pages) Py_RETURN_NONE;
    ids[i] = static_cast<int32_t>(id);
  }
  if (t->numel() == 0 || moves == 0) return PyLong_FromLong(0);
  const c10::cuda::CUDAGuard guard(t->get_device());
  return launched(sabre_copy_pages(t->data_ptr(), static_cast<int>(buffers), step * es, static_cast<int>(pages),
                                   t->stride(d - 4) * es, unit * es, ids.data(), ids.data() + moves,
                                   static_cast<int>(moves), c10::cuda::getCurrentCUDAStream(t->get_device()).stream()),
                  (moves + 479) / 480);  // 480 moves travel with a launch
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(store)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"copy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(copy)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_call() { return PyModule_Create(&module); }
