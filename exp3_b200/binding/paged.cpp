// exp3_b200._paged: the paged cache's three calls from torch tensors to the C ABI.
//
// A decode step makes these calls once a layer on a few rows each, where the GPU needs a few
// microseconds; checking ten tensors and handing forty arguments through ctypes took longer than
// that (17 us of host time for one paged_decode_attention, against 8 us with this module). The
// checks are those of exp3_b200.paged, whose functions call this module and document it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "fpx.h"

namespace {

// Bound once by exp3_b200.paged: the library's functions, and the exception that it raises.
decltype(&fpx_paged_append) g_append;
decltype(&fpx_paged_gather) g_gather;
decltype(&fpx_paged_decode_attention) g_decode;
decltype(&fpx_paged_decode_workspace_bytes) g_workspace;
decltype(&fpx_status_string) g_status;
PyObject *g_error;

struct Refusal {
  PyObject *type;
  std::string text;
};
[[noreturn]] void refuse(std::string text) { throw Refusal{g_error ? g_error : PyExc_RuntimeError, std::move(text)}; }
[[noreturn]] void wrong_type(std::string text) { throw Refusal{PyExc_TypeError, std::move(text)}; }

const at::Tensor *tensor(PyObject *o, const char *name, bool may_be_none = false) {
  if (may_be_none && o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) wrong_type(std::string(name) + " must be a tensor");
  return &THPVariable_Unpack(o);
}

struct Device {
  bool known = false;
  c10::Device value{c10::kCPU};
  void add(const at::Tensor *t) {
    if (!t) return;
    if (!t->is_cuda()) refuse("fpx ops run on CUDA tensors only (there is no CPU path)");
    if (known && t->device() != value) refuse("all tensors of a call must be on one CUDA device");
    value = t->device();
    known = true;
  }
};

// Address and strides of a bf16 tensor [B, L, heads, d].
struct Rows {
  void *data = nullptr;
  int64_t b = 0, l = 0, h = 0;
};
Rows rows(const at::Tensor &t, at::IntArrayRef shape, const char *name, bool output = false) {
  if (t.scalar_type() != at::kBFloat16) wrong_type("q, k, v and their outputs must be bfloat16");
  if (t.sizes() != shape) {
    std::string text = std::string(name) + " must be [";
    for (size_t i = 0; i < shape.size(); ++i) text += (i ? ", " : "") + std::to_string(shape[i]);
    refuse(text + "]");
  }
  const auto s = t.strides();
  if (s[3] != 1 && shape[3] > 1) refuse("the last dimension must be contiguous");
  if (output)
    for (int i = 0; i < 3; ++i)
      if (s[i] == 0 && shape[i] > 1) refuse(std::string(name) + " must not be an expanded tensor");
  return {t.data_ptr(), s[0], s[1], s[2]};
}

int to_int(int64_t v) {
  if (v < INT32_MIN || v > INT32_MAX) refuse("a size is beyond 32 bits");
  return (int)v;
}

struct Where {
  int format, dim, heads, pages, page_size, max_pages;
  void *pool;
  const int32_t *table, *starts, *counts;
  int64_t stride;
};
const int32_t *index_tensor(const at::Tensor *t, int64_t batch) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kInt) wrong_type("page_table, starts and counts must be int32");
  if (t->dim() != 1 || t->size(0) != batch || !t->is_contiguous()) refuse("starts and counts must be [B], contiguous");
  return static_cast<const int32_t *>(t->data_ptr());
}
void pool_form(const at::Tensor &pool, Where &w) {
  if (pool.dim() != 4) refuse("a pool is [pages, Hkv, page_size, row]");
  const int64_t row = pool.size(3);
  const auto type = pool.scalar_type();
  if (type == at::kBFloat16) {
    w.format = FPX_PAGES_BF16;
    w.dim = row == 256 ? 128 : row == 512 ? 256 : 0;
  } else if (type == at::kByte) {
    w.format = FPX_PAGES_INT4;
    w.dim = row == 146 ? 128 : row == 290 ? 256 : 0;
  } else {
    wrong_type("a pool is bfloat16, or uint8 in the 4-bit form");
  }
  if (!w.dim) refuse("a pool's rows of " + std::to_string(row) + " elements are of no compiled head dim");
  if (!pool.is_contiguous()) refuse("a pool must be contiguous");
}
Where where(const at::Tensor &pool, const at::Tensor &table, const at::Tensor &starts, const at::Tensor *counts, int64_t batch,
            int64_t heads, int64_t dim) {
  Where w{};
  pool_form(pool, w);
  if (w.dim != dim || pool.size(1) != heads)
    refuse("the pool holds " + std::to_string(pool.size(1)) + " KV heads of " + std::to_string(w.dim) + ", the call " +
           std::to_string(heads) + " of " + std::to_string(dim));
  if (table.scalar_type() != at::kInt) wrong_type("page_table, starts and counts must be int32");
  if (table.dim() != 2 || table.size(0) != batch || (table.size(1) > 1 && table.stride(1) != 1))
    refuse("page_table must be [B, max_pages] with contiguous rows");
  w.pages = to_int(pool.size(0));
  w.heads = to_int(heads);
  w.page_size = to_int(pool.size(2));
  w.pool = pool.data_ptr();
  w.table = static_cast<const int32_t *>(table.data_ptr());
  w.max_pages = to_int(table.size(1));
  w.stride = batch > 1 ? table.stride(0) : table.size(1);
  w.starts = index_tensor(&starts, batch);
  w.counts = index_tensor(counts, batch);
  return w;
}

// Runs a C call on the device's current stream, with the device as the current one (its default stream has no device
// of its own to be bound to).
template <class F>
void on_stream(const Device &dev, const char *name, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev.value.index()) guard.set_device(dev.value);
  const int rc = f((fpx_stream_t)c10::cuda::getCurrentCUDAStream(dev.value.index()).stream());
  if (rc) refuse(std::string(name) + " failed with status " + std::to_string(rc) + " (" + g_status(rc) + ")");
}
at::Tensor empty(at::IntArrayRef shape, const Device &dev, at::ScalarType type) {
  return at::detail::empty_cuda(shape, type, dev.value, c10::nullopt);
}

// paged_decode_attention(q, pool, page_table, starts, scale, counts, out, lse, ws)
PyObject *decode(PyObject *const *a) {
  const at::Tensor &q = *tensor(a[0], "q"), &pool = *tensor(a[1], "pool"), &table = *tensor(a[2], "page_table"),
                   &starts = *tensor(a[3], "starts");
  const double scale = PyFloat_AsDouble(a[4]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  const at::Tensor *counts = tensor(a[5], "counts", true), *out = tensor(a[6], "out", true), *lse = tensor(a[7], "lse", true),
                   *ws = tensor(a[8], "ws", true);
  if (q.dim() == 4 && q.size(1) > FPX_PAGED_MAX_ROWS)
    refuse(std::to_string(q.size(1)) + " query rows a sequence: one call takes " + std::to_string(FPX_PAGED_MAX_ROWS) +
           " (paged_gather and prefill_attention take longer continuations)");
  // its bytes count from its address on, which strides of their own would not give
  if (ws && !ws->is_contiguous()) refuse("ws must be contiguous");
  Device dev;
  for (const at::Tensor *t : {&q, &pool, &table, &starts, counts, out, lse, ws}) dev.add(t);
  if (q.dim() != 4) refuse("q must be [B, Lq, H, d]");
  const int64_t B = q.size(0), L = q.size(1), H = q.size(2), d = q.size(3);
  const Rows qr = rows(q, q.sizes(), "q");
  const Where w = where(pool, table, starts, counts, B, pool.dim() == 4 ? pool.size(1) : 0, d);
  at::Tensor made;
  if (!out) {
    made = empty(q.sizes(), dev, at::kBFloat16);
    out = &made;
  }
  const Rows o = rows(*out, q.sizes(), "out", true);
  if (lse && (lse->scalar_type() != at::kFloat || !lse->is_contiguous() || lse->sizes() != q.sizes().slice(0, 3)))
    refuse("lse must be a contiguous fp32 [B, Lq, H]");
  if (B && L) {
    at::Tensor scratch;
    on_stream(dev, "fpx_paged_decode_attention", [&](fpx_stream_t stream) {
      const auto call = [&](const at::Tensor *space) {
        return g_decode(w.format, qr.data, qr.b, qr.l, qr.h, to_int(B), to_int(L), to_int(H), w.heads, w.dim, scale, w.pool, w.pages,
                        w.page_size, w.table, w.stride, w.max_pages, w.starts, w.counts, o.data, o.b, o.l, o.h,
                        lse ? static_cast<float *>(lse->data_ptr()) : nullptr, space ? space->data_ptr() : nullptr,
                        space ? (size_t)space->nbytes() : 0, stream);
      };
      int rc = call(ws);  // short tables need no workspace: without one the call says so before it does anything
      if (rc == FPX_ERR_WORKSPACE && !ws) {
        scratch = empty({(int64_t)g_workspace(w.format, to_int(B), to_int(L), to_int(H), w.heads, w.dim)}, dev, at::kByte);
        rc = call(&scratch);
      }
      return rc;
    });
  }
  return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(a[6]);
}

// paged_gather(pool, page_table, starts, counts, length, k_out, v_out)
PyObject *gather(PyObject *const *a) {
  const at::Tensor &pool = *tensor(a[0], "pool"), &table = *tensor(a[1], "page_table"), &starts = *tensor(a[2], "starts");
  const at::Tensor *counts = tensor(a[3], "counts", true), *k = tensor(a[5], "k_out", true), *v = tensor(a[6], "v_out", true);
  const int64_t L = PyLong_AsLongLong(a[4]);
  if (L == -1 && PyErr_Occurred()) return nullptr;
  Device dev;
  for (const at::Tensor *t : {&pool, &table, &starts, counts, k, v}) dev.add(t);
  Where form{};
  pool_form(pool, form);
  if (starts.dim() != 1) refuse("starts and counts must be [B], contiguous");
  if (L < 0) refuse("length must not be negative");
  const int64_t B = starts.size(0), heads = pool.size(1);
  const Where w = where(pool, table, starts, counts, B, heads, form.dim);
  if (!k != !v) refuse("give both of k_out and v_out, or neither");
  const int64_t shape[4] = {B, L, heads, w.dim};
  at::Tensor mk, mv;
  if (!k) {
    mk = empty(shape, dev, at::kBFloat16);
    mv = empty(shape, dev, at::kBFloat16);
  }
  const Rows kr = rows(k ? *k : mk, shape, "k_out", true), vr = rows(v ? *v : mv, shape, "v_out", true);
  if (B && L)
    on_stream(dev, "fpx_paged_gather", [&](fpx_stream_t stream) {
      return g_gather(w.format, w.pool, w.pages, w.page_size, w.table, w.stride, w.max_pages, w.starts, w.counts, to_int(B), to_int(L),
                      w.heads, w.dim, kr.data, kr.b, kr.l, kr.h, vr.data, vr.b, vr.l, vr.h, !k, stream);
    });
  PyObject *pk = k ? Py_NewRef(a[5]) : THPVariable_Wrap(mk), *pv = v ? Py_NewRef(a[6]) : THPVariable_Wrap(mv);
  PyObject *both = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return both;
}

// paged_append(k, v, pool, page_table, starts, counts, q, rope, q_out, k_out)
PyObject *append(PyObject *const *a) {
  const at::Tensor &k = *tensor(a[0], "k"), &v = *tensor(a[1], "v"), &pool = *tensor(a[2], "pool"), &table = *tensor(a[3], "page_table"),
                   &starts = *tensor(a[4], "starts");
  const at::Tensor *counts = tensor(a[5], "counts", true), *q = tensor(a[6], "q", true), *rope = tensor(a[7], "rope", true),
                   *q_out = tensor(a[8], "q_out", true), *k_out = tensor(a[9], "k_out", true);
  Device dev;
  for (const at::Tensor *t : {&k, &v, &pool, &table, &starts, counts, q, rope, q_out, k_out}) dev.add(t);
  if (k.dim() != 4) refuse("k and v must be [B, L, Hkv, d]");
  const int64_t B = k.size(0), L = k.size(1), heads = k.size(2), d = k.size(3);
  const Rows kr = rows(k, k.sizes(), "k"), vr = rows(v, k.sizes(), "v");
  const Where w = where(pool, table, starts, counts, B, heads, d);
  int rope_len = 0, rotary = 0;
  if (rope) {
    if (rope->scalar_type() != at::kFloat || rope->dim() != 2 || !rope->is_contiguous())
      refuse("rope must be a contiguous fp32 [positions, rotary] table");
    rope_len = to_int(rope->size(0));
    rotary = to_int(rope->size(1));
  }
  int64_t H = 0;
  Rows qr, qo, ko;
  at::Tensor made;
  if (!q) {
    if (q_out) refuse("q_out without q");
  } else {
    if (q->dim() != 4) refuse("q must be [B, L, H, d]");
    H = q->size(2);
    const int64_t shape[4] = {B, L, H, d};
    qr = rows(*q, shape, "q");
    if (!q_out) made = empty(shape, dev, at::kBFloat16);
    qo = rows(q_out ? *q_out : made, shape, "q_out", true);
  }
  if (k_out) ko = rows(*k_out, k.sizes(), "k_out", true);
  if (B && L)
    on_stream(dev, "fpx_paged_append", [&](fpx_stream_t stream) {
      return g_append(w.format, qr.data, qr.b, qr.l, qr.h, kr.data, kr.b, kr.l, kr.h, vr.data, vr.b, vr.l, vr.h, to_int(B), to_int(L),
                      to_int(H), w.heads, w.dim, rope ? static_cast<const float *>(rope->data_ptr()) : nullptr, rope_len, rotary,
                      w.pool, w.pages, w.page_size, w.table, w.stride, w.max_pages, w.starts, w.counts, qo.data, qo.b, qo.l, qo.h,
                      ko.data, ko.b, ko.l, ko.h, made.defined(), stream);
    });
  return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(a[8]);
}

// check_where(pool, page_table, starts, counts, batch, kv_heads, head_dim) -> format: the checks alone, on any device
PyObject *check_where(PyObject *const *a) {
  const at::Tensor &pool = *tensor(a[0], "pool"), &table = *tensor(a[1], "page_table"), &starts = *tensor(a[2], "starts");
  const Where w = where(pool, table, starts, tensor(a[3], "counts", true), PyLong_AsLongLong(a[4]), PyLong_AsLongLong(a[5]),
                        PyLong_AsLongLong(a[6]));
  return PyLong_FromLong(w.format);
}

// bind(append, gather, decode_attention, decode_workspace_bytes, status_string: addresses; error: exception class)
PyObject *bind(PyObject *const *a) {
  void *f[5];
  for (int i = 0; i < 5; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a function's address is null");
      return nullptr;
    }
  }
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_gather = reinterpret_cast<decltype(g_gather)>(f[1]);
  g_decode = reinterpret_cast<decltype(g_decode)>(f[2]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(f[3]);
  g_status = reinterpret_cast<decltype(g_status)>(f[4]);
  Py_XSETREF(g_error, Py_NewRef(a[5]));
  Py_RETURN_NONE;
}

// No C++ exception leaves a call.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t count) {
  if (count != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are needed, %zd given", N, count);
    return nullptr;
  }
  if (F != bind && !g_error) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal &r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

template <PyObject *(*F)(PyObject *const *), int N>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {method<decode, 9>("paged_decode_attention"), method<gather, 7>("paged_gather"),
                           method<append, 10>("paged_append"), method<check_where, 7>("check_where"), method<bind, 6>("bind"),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged() {
  PyObject *module = PyModule_Create(&g_module);
  if (module && PyModule_AddStringConstant(module, "TORCH_VERSION", FPX_TORCH_VERSION) < 0) Py_CLEAR(module);
  return module;
}
