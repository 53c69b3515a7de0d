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

#include <ATen/Context.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
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

const at::Tensor* optional(PyObject* o, bool& ok) {  // null for None
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  ok = ok && t;
  return t;
}

int code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? SABRE_BF16 : t.scalar_type() == at::kHalf ? SABRE_F16 : -1;
}

// Tables and lengths of a call without K and V pools.
struct Tables {
  const at::Tensor *table, *lens, *starts;
  int batch, cols;
  c10::DeviceIndex dev;

  bool on(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == dev; }
  bool ints(const at::Tensor* t, int64_t n) const {
    return t && on(*t) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
  }
  bool read(PyObject* tab, PyObject* sl, PyObject* qs) {
    bool ok = true;
    table = tensor(tab), lens = tensor(sl), starts = optional(qs, ok);
    if (!ok || !table || !lens || !table->is_cuda()) return false;
    dev = table->get_device();
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(1) < 1 || !small(table->size(0)) ||
        !small(table->size(1)) || (table->size(1) > 1 && table->stride(1) != 1))
      return false;
    batch = table->size(0), cols = table->size(1);
    return ints(lens, batch) && (!starts || ints(starts, int64_t{batch} + 1));
  }
  // Mean keys [pages, heads, D].
  bool means(const at::Tensor* m) const {
    return m && on(*m) && m->scalar_type() == at::kFloat && m->dim() == 3 && m->stride(2) == 1 && small(m->size(0)) &&
           small(m->size(1)) && small(m->size(2));
  }
};

// A tensor on the device: past the dispatcher (half a microsecond less), unless the
// dispatcher does more than allocate: fills it in deterministic mode, or shows it to a mode.
at::Tensor fresh_tensor(at::IntArrayRef size, at::ScalarType type, c10::DeviceIndex dev) {
  const c10::Device on(c10::kCUDA, dev);
  if (at::globalContext().deterministicAlgorithms() || c10::impl::TorchDispatchModeTLS::any_modes_set())
    return at::empty(size, at::TensorOptions(type).device(on));
  return at::Tensor(at::detail::empty_cuda(size, type, on, std::nullopt));
}

int32_t* i32(const at::Tensor* t) { return t ? static_cast<int32_t*>(t->data_ptr()) : nullptr; }

int integer(PyObject* o) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return static_cast<int>(x);
}

// A size of at least `low`, held to int32; false below that.
bool sized(PyObject* o, long long low, int& out) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  out = x > INT_MAX ? INT_MAX : static_cast<int>(x);
  return x >= low;
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

// store_slots(k, v, k_pages, v_pages, slots) -> kernels
PyObject* store_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]), *kp = tensor(a[2]), *vp = tensor(a[3]), *slots = tensor(a[4]);
  if (!k || !v || !kp || !vp || !slots || !kp->is_cuda() || kp->dim() != 4 || vp->sizes() != kp->sizes() ||
      code(*kp) < 0 || kp->stride(3) != 1 || vp->stride(3) != 1)
    Py_RETURN_NONE;
  for (const at::Tensor* t : {k, v, vp, slots})
    if (!t->is_cuda() || t->get_device() != kp->get_device()) Py_RETURN_NONE;
  for (const at::Tensor* t : {k, v, vp})
    if (t->scalar_type() != kp->scalar_type()) Py_RETURN_NONE;
  if (k->dim() != 3 || v->sizes() != k->sizes() || k->size(1) != kp->size(1) || k->size(2) != kp->size(3) ||
      k->stride(2) != 1 || v->stride(2) != 1 || slots->scalar_type() != at::kLong || slots->dim() != 1 ||
      slots->size(0) != k->size(0) || !slots->is_contiguous() || !small(k->size(0)))
    Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (!small(kp->size(i))) Py_RETURN_NONE;
  if (k->size(0) == 0) return PyLong_FromLong(0);
  const int64_t kr[2] = {k->stride(0), k->stride(1)}, vr[2] = {v->stride(0), v->stride(1)};
  const int64_t ks[3] = {kp->stride(0), kp->stride(1), kp->stride(2)};
  const int64_t vs[3] = {vp->stride(0), vp->stride(1), vp->stride(2)};
  const c10::cuda::CUDAGuard guard(kp->get_device());
  return launched(sabre_paged_store_slots(k->const_data_ptr(), v->const_data_ptr(), kp->data_ptr(), vp->data_ptr(),
                                          static_cast<const int64_t*>(slots->const_data_ptr()), k->size(0),
                                          kp->size(1), kp->size(3), kp->size(0), kp->size(2), kr, vr, ks, vs,
                                          code(*kp), c10::cuda::getCurrentCUDAStream(kp->get_device()).stream()),
                  1);
  END_HANDLE_TH_ERRORS
}

// extend(new_rows, page_table, seq_lens, free_pages, free_count, page_size, num_pages, rows, seq_lens_out or None,
// free_count_out or None, max_seq_len or None) -> (q_start, slots, positions, kernels)
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tables p;
  if (n != 11 || !p.read(a[1], a[2], Py_None) || p.batch == 0) Py_RETURN_NONE;
  const at::Tensor *fresh = tensor(a[0]), *free_pages = tensor(a[3]), *count = tensor(a[4]);
  bool ok = true;
  const at::Tensor *lens_out = optional(a[8], ok), *count_out = optional(a[9], ok);
  if (!ok || !p.ints(fresh, p.batch) || !free_pages || free_pages->dim() != 1 || !small(free_pages->size(0)) ||
      !p.ints(free_pages, free_pages->size(0)) || !p.ints(count, 1) || (lens_out && !p.ints(lens_out, p.batch)) ||
      (count_out && !p.ints(count_out, 1)))
    Py_RETURN_NONE;
  if (!lens_out) lens_out = p.lens;
  if (!count_out) count_out = count;
  int page_size, num_pages, rows, max_len = INT_MAX;
  if (!sized(a[5], 1, page_size) || !sized(a[6], 1, num_pages) || !sized(a[7], 0, rows) ||
      (a[10] != Py_None && !sized(a[10], 1, max_len)))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(p.dev);
  at::Tensor starts = fresh_tensor({int64_t{p.batch} + 1}, at::kInt, p.dev);
  at::Tensor slots = fresh_tensor({rows}, at::kLong, p.dev), positions = fresh_tensor({rows}, at::kLong, p.dev);
  const int st = sabre_paged_extend_within(
      i32(fresh), i32(p.table), i32(p.lens), i32(lens_out), i32(free_pages), i32(count), i32(count_out), i32(&starts),
      static_cast<int64_t*>(slots.data_ptr()), static_cast<int64_t*>(positions.data_ptr()), rows, p.batch,
      num_pages, page_size, p.cols, free_pages->size(0), max_len, p.table->stride(0),
      c10::cuda::getCurrentCUDAStream(p.dev).stream());
  if (st != SABRE_OK) return PyLong_FromLong(st);
  // More than 2048 rows are placed by a kernel of their own.
  return Py_BuildValue("NNNi", THPVariable_Wrap(starts), THPVariable_Wrap(slots), THPVariable_Wrap(positions),
                       rows > 2048 ? 2 : 1);
  END_HANDLE_TH_ERRORS
}

// key_means(k_pages, key_means, page_table, seq_lens, q_start, rows) -> kernels
PyObject* key_means(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tables p;
  if (n != 6 || !p.read(a[2], a[3], a[4])) Py_RETURN_NONE;
  const at::Tensor *k = tensor(a[0]), *m = tensor(a[1]);
  if (!k || !p.on(*k) || k->dim() != 4 || code(*k) < 0 || k->stride(3) != 1 || !p.means(m) ||
      m->size(0) != k->size(0) || m->size(1) != k->size(1) || m->size(2) != k->size(3) || !small(k->size(2)))
    Py_RETURN_NONE;
  int rows;
  if (!sized(a[5], 0, rows) || (!p.starts && rows != p.batch)) Py_RETURN_NONE;
  if (rows == 0 || p.batch == 0) return PyLong_FromLong(0);
  const int64_t ks[3] = {k->stride(0), k->stride(1), k->stride(2)}, ms[2] = {m->stride(0), m->stride(1)};
  const c10::cuda::CUDAGuard guard(p.dev);
  return launched(sabre_paged_key_means(k->const_data_ptr(), static_cast<float*>(m->data_ptr()), i32(p.table),
                                        i32(p.lens), i32(p.starts), rows, p.batch, k->size(1), k->size(3), k->size(0),
                                        k->size(2), p.cols, ks, ms, p.table->stride(0), code(*k),
                                        c10::cuda::getCurrentCUDAStream(p.dev).stream()),
                  1);
  END_HANDLE_TH_ERRORS
}

// select(q, key_means, page_table, seq_lens, q_start, page_size, topk, query_block, window, prefix) -> (lists, counts)
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tables p;
  if (n != 10 || !p.read(a[2], a[3], a[4])) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *m = tensor(a[1]);
  if (!p.means(m) || !q || !p.on(*q) || q->dim() != 3 || code(*q) < 0 || q->stride(2) != 1 ||
      q->size(2) != m->size(2) || !small(q->size(0)) || !small(q->size(1)) || m->size(1) == 0 ||
      (!p.starts && q->size(0) != p.batch))
    Py_RETURN_NONE;
  const int rows = q->size(0), heads = m->size(1);
  int page_size, topk, block, window, prefix;
  if (!sized(a[5], 1, page_size) || !sized(a[6], 0, topk) || !sized(a[7], 1, block) || !sized(a[8], 0, window) ||
      !sized(a[9], 0, prefix) || (!p.starts && block != 1))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(p.dev);
  const int blocks = sabre_paged_query_blocks(rows, p.batch, block);
  const int width = sabre_paged_select_width(page_size, p.cols, topk, block, window, prefix);
  at::Tensor lists = fresh_tensor({blocks, heads, width}, at::kInt, p.dev);
  at::Tensor counts = fresh_tensor({blocks, heads}, at::kInt, p.dev);
  if (rows > 0 && p.batch > 0) {
    const int64_t qr[2] = {q->stride(0), q->stride(1)}, ms[2] = {m->stride(0), m->stride(1)};
    const int st = sabre_paged_select(q->const_data_ptr(), static_cast<const float*>(m->const_data_ptr()), i32(p.table),
                                      i32(p.lens), i32(p.starts), i32(&lists), i32(&counts), rows, p.batch,
                                      q->size(1), heads, q->size(2), m->size(0), page_size, p.cols, topk, block,
                                      window, prefix, qr, ms, p.table->stride(0), code(*q),
                                      c10::cuda::getCurrentCUDAStream(p.dev).stream());
    if (st != SABRE_OK) return PyLong_FromLong(st);
  }
  return Py_BuildValue("NNi", THPVariable_Wrap(lists), THPVariable_Wrap(counts), rows > 0 && p.batch > 0 ? 1 : 0);
  END_HANDLE_TH_ERRORS
}

// attend_listed(q, k_pages, v_pages, page_table, seq_lens, q_start, lists, counts, query_block, scale, out, workspace)
// -> (out, kernels); decode without q_start.
PyObject* attend_listed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  if (n != 12 || !p.read(a[1], a[2], a[3], a[4], a[5])) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *lists = tensor(a[6]), *counts = tensor(a[7]);
  if (!p.rows(q) || (!p.starts && q->size(0) != p.batch)) Py_RETURN_NONE;
  int block;
  if (!sized(a[8], 1, block)) Py_RETURN_NONE;
  const float scale = number(a[9]);
  const int rows = q->size(0), heads_q = q->size(1);
  const int blocks = p.starts ? sabre_paged_query_blocks(rows, p.batch, block) : p.batch;
  for (const at::Tensor* t : {lists, counts})
    if (!t || !p.on(*t) || t->scalar_type() != at::kInt || t->dim() < 2 || t->size(0) < blocks ||
        t->size(1) != p.heads)
      Py_RETURN_NONE;
  if (lists->dim() != 3 || counts->dim() != 2 || lists->size(2) < 1 || !small(lists->size(2)) ||
      (lists->size(2) > 1 && lists->stride(2) != 1))
    Py_RETURN_NONE;
  at::Tensor out, ws;
  if (a[10] != Py_None) {
    const at::Tensor* o = tensor(a[10]);
    if (!p.rows(o) || o->sizes() != q->sizes() || at::has_internal_overlap(*o) == at::MemOverlap::Yes) Py_RETURN_NONE;
    out = *o;
  }
  const c10::cuda::CUDAGuard guard(p.dev);
  if (!out.defined()) out = fresh_tensor(q->sizes(), q->scalar_type(), p.dev);
  if (q->numel() == 0 || p.batch == 0) return result(out, 0);
  const int entries = lists->size(2);
  const size_t need = p.starts ? sabre_paged_prefill_listed_workspace_size(rows, p.batch, heads_q, p.heads, p.dim,
                                                                           p.page_size, block, entries)
                               : sabre_paged_decode_workspace_size(p.batch, heads_q, p.heads, p.dim);
  if (a[11] != Py_None) {
    const at::Tensor* w = tensor(a[11]);
    if (!w || !p.on(*w) || !w->is_contiguous() || w->nbytes() < need) Py_RETURN_NONE;
    ws = *w;
  } else if (need > 0) {
    ws = fresh_tensor({static_cast<int64_t>(need)}, at::kByte, p.dev);
  }
  void* const wp = ws.defined() ? ws.data_ptr() : nullptr;
  const size_t wb = ws.defined() ? ws.nbytes() : 0;
  const int64_t qr[2] = {q->stride(0), q->stride(1)}, orr[2] = {out.stride(0), out.stride(1)};
  const int64_t ls[2] = {lists->stride(0), lists->stride(1)}, cs[2] = {counts->stride(0), counts->stride(1)};
  void* const stream = c10::cuda::getCurrentCUDAStream(p.dev).stream();
  const int st =
      p.starts
          ? sabre_paged_prefill_listed(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(),
                                       out.data_ptr(), p.i32(p.table), p.i32(p.lens), p.i32(p.starts), i32(lists),
                                       i32(counts), entries, rows, p.batch, heads_q, p.heads, p.dim, p.pages,
                                       p.page_size, p.cols, block, qr, p.ks, p.vs, orr, ls, cs, p.table->stride(0),
                                       scale, p.dtype, wp, wb, stream)
          : sabre_paged_decode_listed(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(),
                                      out.data_ptr(), p.i32(p.table), p.i32(p.lens), i32(lists), i32(counts), entries,
                                      p.batch, heads_q, p.heads, p.dim, p.pages, p.page_size, p.cols, qr, p.ks, p.vs,
                                      orr, ls, cs, p.table->stride(0), scale, p.dtype, wp, wb, stream);
  if (st != SABRE_OK) return PyLong_FromLong(st);
  // As in attend: prompts whose pairs are cut into parts ask for a workspace; decodes of
  // more than one key tile are joined by a second kernel, unless they run in clusters:
  // up to 28 pairs of up to 32 tiles.
  const int64_t tiles = (int64_t{entries} * p.page_size + 63) / 64, pairs = int64_t{p.batch} * p.heads;
  const bool joined = p.starts ? need > 0 : tiles * pairs > 1 && !(pairs <= 28 && tiles > 1 && tiles <= 32);
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
    {"store_slots", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(store_slots)), METH_FASTCALL, nullptr},
    {"extend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(extend)), METH_FASTCALL, nullptr},
    {"key_means", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(key_means)), METH_FASTCALL, nullptr},
    {"select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(select)), METH_FASTCALL, nullptr},
    {"attend_listed", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend_listed)), METH_FASTCALL, nullptr},
    {"copy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(copy)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_call() { return PyModule_Create(&module); }
