// Calls of the decoding operators straight from Python, for arguments that need nothing
// done to them: a call is then its checks, its outputs and its launches (6 to 8 us less
// than by way of ctypes, half of a small step).  Whatever is not plain (another device,
// type, layout, a size that the library refuses) returns None, and the caller's own Python
// raises the error, or makes the copy, and calls by ctypes.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/quipsharp_b200.h"

namespace {

using at::Tensor;

// Unpacks tensors of one CUDA device, the current one.
struct Args {
  c10::DeviceIndex device = -1;
  bool ok = true;

  const Tensor *tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return ok = false, nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided) return ok = false, nullptr;
    if (device < 0) {
      device = t.get_device();
      if (device != c10::cuda::current_device()) ok = false;
    } else if (t.get_device() != device) {
      ok = false;
    }
    if (t.requires_grad() && c10::GradMode::is_enabled()) ok = false;
    if (t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined()) ok = false;  // a tangent
    return &t;
  }
  const Tensor *ints(PyObject *o, int64_t dims) {
    const Tensor *t = tensor(o);
    if (t && (t->scalar_type() != at::kInt || t->dim() != dims || !t->is_contiguous())) ok = false;
    return t;
  }
  cudaStream_t cuda_stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
  qs_stream_t stream() const { return cuda_stream(); }
};

int dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kHalf: return QS_F16;
    case at::kBFloat16: return QS_BF16;
    case at::kFloat: return QS_F32;
    default: return -1;
  }
}

bool in_pieces(const Tensor &t) {  // 16-byte pieces of two-byte values
  if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) & 7) return false;
  return true;
}

bool pool_of(const Tensor &k, const Tensor &v, int64_t dims, qs_kv_pool *p) {
  const int dt = dtype_of(k);
  if ((dt != QS_F16 && dt != QS_BF16) || v.scalar_type() != k.scalar_type() || k.dim() != dims || v.dim() != dims ||
      k.sizes() != v.sizes() || k.stride(-1) != 1 || v.stride(-1) != 1)
    return false;
  const int64_t o = dims - 4;  // 1 with a layer axis
  *p = qs_kv_pool{k.data_ptr(), v.data_ptr(), dt, o ? k.size(0) : 1, k.size(o), k.size(o + 1), k.size(o + 2), k.size(o + 3),
                  {o ? k.stride(0) : 0, k.stride(o), k.stride(o + 1), k.stride(o + 2)},
                  {o ? v.stride(0) : 0, v.stride(o), v.stride(o + 1), v.stride(o + 2)}};
  return true;
}

bool integer(PyObject *o, int64_t *v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) return PyErr_Clear(), false;
  return true;
}

// A new tensor, without the way through the dispatcher (0.3 us each).
Tensor fresh(const Args &a, at::IntArrayRef sizes, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, a.device), std::nullopt));
}
Tensor ints(const Args &a, at::IntArrayRef sizes) { return fresh(a, sizes, at::kInt); }

// A workspace from torch's allocator, given back when the call's launches are queued (what
// is next to have it on this stream comes after them).
struct Scratch {
  void *p;
  Scratch(const Args &a, int64_t bytes)
      : p(bytes ? c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(bytes, a.cuda_stream()) : nullptr) {}
  ~Scratch() {
    if (p) c10::cuda::CUDACachingAllocator::raw_delete(p);
  }
  Scratch(const Scratch &) = delete;
};

int *ip(const Tensor &t) { return static_cast<int *>(t.data_ptr()); }

PyObject *tuple3(const Tensor &a, const Tensor &b, const Tensor &c) {
  return Py_BuildValue("(NNN)", THPVariable_Wrap(a), THPVariable_Wrap(b), THPVariable_Wrap(c));
}

#define PLAIN(cond) \
  if (!(cond)) Py_RETURN_NONE

// (q, k_pages, v_pages, table, lengths, cu or None, window or None, sinks, scale or None, return_lse)
PyObject *attend(PyObject *const *in) {
  Args a;
  const Tensor *q = a.tensor(in[0]), *k = a.tensor(in[1]), *v = a.tensor(in[2]);
  const Tensor *table = a.ints(in[3], 2), *lengths = a.ints(in[4], 1);
  const bool many = in[5] != Py_None;
  const Tensor *cu = many ? a.ints(in[5], 1) : nullptr;
  PLAIN(a.ok);
  int64_t window = 0, sinks;
  PLAIN(in[6] == Py_None || (integer(in[6], &window) && window >= 1));
  PLAIN(integer(in[7], &sinks) && sinks >= 0 && PyBool_Check(in[9]));
  qs_kv_pool pool;
  PLAIN(q->dim() == 3 && q->scalar_type() == k->scalar_type() && pool_of(*k, *v, 4, &pool) && in_pieces(*q));
  const int64_t rows = table->size(0), width = table->size(1), tokens = q->size(0), heads = q->size(1), dim = q->size(2);
  PLAIN(dim == pool.dim && dim > 0 && pool.heads > 0 && heads % pool.heads == 0 && lengths->size(0) == rows &&
        (many ? cu->size(0) == rows + 1 : tokens == rows));
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (in[8] != Py_None) {
    PLAIN(PyFloat_CheckExact(in[8]));
    scale = PyFloat_AS_DOUBLE(in[8]);
  }
  const int64_t nb = many ? qs_attn_window_workspace_bytes(tokens, rows, heads, pool.heads, dim, pool.page, width, window, sinks)
                          : qs_attn_decode_workspace_bytes(rows, heads, pool.heads, dim, pool.page, width, window, sinks);
  PLAIN(nb >= 0);
  const bool want_lse = in[9] == Py_True;
  const Scratch ws(a, nb);
  const Tensor out = fresh(a, {tokens, heads, dim}, q->scalar_type());
  const Tensor lse = want_lse ? fresh(a, {tokens, heads}, at::kFloat) : Tensor();
  float *lp = want_lse ? static_cast<float *>(lse.data_ptr()) : nullptr;
  const int st =
      many ? qs_attn_window(q->data_ptr(), q->stride(0), q->stride(1), &pool, tokens, rows, heads, width, ip(*table),
                            ip(*lengths), ip(*cu), static_cast<float>(scale), window, sinks, out.data_ptr(), lp, ws.p, nb,
                            a.stream())
           : qs_attn_decode(q->data_ptr(), q->stride(0), q->stride(1), &pool, rows, heads, width, ip(*table), ip(*lengths),
                            static_cast<float>(scale), window, sinks, out.data_ptr(), lp, ws.p, nb, a.stream());
  PLAIN(st == QS_OK);
  if (!want_lse) return THPVariable_Wrap(out);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
}

// (k, v, table, lengths, refcount, parents)
PyObject *fork_pages(PyObject *const *in) {
  Args a;
  const Tensor *k = a.tensor(in[0]), *v = a.tensor(in[1]), *table = a.ints(in[2], 2), *lengths = a.ints(in[3], 1),
               *count = a.ints(in[4], 1), *parents = a.ints(in[5], 1);
  PLAIN(a.ok);
  qs_kv_pool pool;
  const int64_t rows = table->size(0), width = table->size(1);
  PLAIN(pool_of(*k, *v, 5, &pool) && lengths->size(0) == rows && parents->size(0) == rows && count->size(0) == pool.pages);
  const int64_t nb = qs_cache_workspace_bytes(rows, pool.pages);
  PLAIN(nb >= 0);
  const Scratch ws(a, nb);
  const Tensor t = ints(a, {rows, width}), n = ints(a, {rows}),
               c = ints(a, {pool.pages});
  PLAIN(qs_cache_fork(&pool, rows, width, ip(*table), ip(*lengths), ip(*count), ip(*parents), ip(t), ip(n), ip(c),
                      ws.p, nb, a.stream()) == QS_OK);
  return tuple3(t, n, c);
}

// (k, v, table, lengths, refcount)
PyObject *compact_pages(PyObject *const *in) {
  Args a;
  const Tensor *k = a.tensor(in[0]), *v = a.tensor(in[1]), *table = a.ints(in[2], 2), *lengths = a.ints(in[3], 1),
               *count = a.ints(in[4], 1);
  PLAIN(a.ok);
  qs_kv_pool pool;
  const int64_t rows = table->size(0), width = table->size(1);
  PLAIN(pool_of(*k, *v, 5, &pool) && lengths->size(0) == rows && count->size(0) == pool.pages);
  const int64_t nb = qs_cache_workspace_bytes(rows, pool.pages);
  PLAIN(nb >= 0);
  const Scratch ws(a, nb);
  const Tensor t = ints(a, {rows, width}),
               c = ints(a, {pool.pages}), used = ints(a, {1});
  PLAIN(qs_cache_compact(&pool, rows, width, ip(*table), ip(*lengths), ip(*count), ip(t), ip(c), ip(used), ws.p, nb,
                         a.stream()) == QS_OK);
  return tuple3(t, c, used);
}

// (table, lengths, refcount, new_tokens, page_size)
PyObject *extend_pages(PyObject *const *in) {
  Args a;
  const Tensor *table = a.ints(in[0], 2), *lengths = a.ints(in[1], 1), *count = a.ints(in[2], 1), *add = a.ints(in[3], 1);
  int64_t page;
  PLAIN(a.ok && integer(in[4], &page));
  const int64_t rows = table->size(0), width = table->size(1), pages = count->size(0);
  PLAIN(lengths->size(0) == rows && add->size(0) == rows);
  const int64_t nb = qs_cache_workspace_bytes(rows, pages);
  PLAIN(nb >= 0);
  const Scratch ws(a, nb);
  const Tensor t = ints(a, {rows, width}), n = ints(a, {rows}),
               c = ints(a, {pages});
  PLAIN(qs_cache_extend(page, pages, rows, width, ip(*table), ip(*lengths), ip(*count), ip(*add), ip(t), ip(n), ip(c),
                        ws.p, nb, a.stream()) == QS_OK);
  return tuple3(t, n, c);
}

// (k, v, k_pages, v_pages, table, lengths, cu or None)
PyObject *write_kv(PyObject *const *in) {
  Args a;
  const Tensor *k = a.tensor(in[0]), *v = a.tensor(in[1]), *kp = a.tensor(in[2]), *vp = a.tensor(in[3]),
               *table = a.ints(in[4], 2), *lengths = a.ints(in[5], 1),
               *cu = in[6] == Py_None ? nullptr : a.ints(in[6], 1);
  PLAIN(a.ok);
  qs_kv_pool pool;
  const int64_t rows = table->size(0), width = table->size(1);
  PLAIN(pool_of(*kp, *vp, 4, &pool) && lengths->size(0) == rows && (!cu || cu->size(0) == rows + 1));
  PLAIN(k->dim() == 3 && k->sizes() == v->sizes() && k->scalar_type() == kp->scalar_type() &&
        v->scalar_type() == kp->scalar_type() && k->size(1) == pool.heads && k->size(2) == pool.dim && pool.dim > 0 &&
        in_pieces(*k) && in_pieces(*v));
  PLAIN(qs_cache_write(&pool, rows, width, ip(*table), ip(*lengths), cu ? ip(*cu) : nullptr, k->data_ptr(), k->stride(0),
                       k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), k->size(0), a.stream()) == QS_OK);
  Py_RETURN_TRUE;
}

// (logits, scores, n or None, finished or None, pad)
PyObject *beam_select(PyObject *const *in) {
  Args a;
  const Tensor *logits = a.tensor(in[0]), *scores = a.tensor(in[1]),
               *finished = in[3] == Py_None ? nullptr : a.tensor(in[3]);
  PLAIN(a.ok);
  const int dt = dtype_of(*logits);
  PLAIN(dt >= 0 && logits->dim() == 3 && logits->stride(2) == 1 && scores->scalar_type() == at::kFloat &&
        scores->dim() == 2 && scores->is_contiguous());
  const int64_t batch = logits->size(0), beams = logits->size(1), vocab = logits->size(2);
  int64_t n = beams, pad;
  PLAIN((in[2] == Py_None || integer(in[2], &n)) && integer(in[4], &pad) && pad == static_cast<int>(pad));
  PLAIN(scores->size(0) == batch && scores->size(1) == beams);
  if (finished)
    PLAIN((finished->scalar_type() == at::kBool || finished->scalar_type() == at::kByte) && finished->is_contiguous() &&
          finished->sizes() == scores->sizes());
  const int64_t nb = qs_beam_workspace_bytes(batch, beams, vocab, n);
  PLAIN(nb >= 0);
  const Scratch ws(a, nb);
  const Tensor out = fresh(a, {batch, n}, at::kFloat), parents = ints(a, {batch, n}), tokens = ints(a, {batch, n});
  PLAIN(qs_beam_select(logits->data_ptr(), dt, logits->stride(0), logits->stride(1), batch, beams, vocab,
                       static_cast<const float *>(scores->data_ptr()),
                       finished ? static_cast<const uint8_t *>(finished->data_ptr()) : nullptr, n, static_cast<int>(pad),
                       static_cast<float *>(out.data_ptr()), ip(parents), ip(tokens), ws.p, nb,
                       a.stream()) == QS_OK);
  return tuple3(out, parents, tokens);
}

// What torch throws (out of memory, say) becomes the Python exception it is elsewhere.
template <PyObject *(*F)(PyObject *const *), Py_ssize_t COUNT>
PyObject *entry(PyObject *, PyObject *const *in, Py_ssize_t count) {
  if (count != COUNT) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", COUNT, count);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  return F(in);
  END_HANDLE_TH_ERRORS
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t COUNT>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, COUNT>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    method<attend, 10>("attend"),           method<fork_pages, 6>("fork_pages"), method<compact_pages, 5>("compact_pages"),
    method<extend_pages, 5>("extend_pages"), method<write_kv, 7>("write_kv"),     method<beam_select, 5>("beam_select"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
