// The operators' way from torch tensors to the C ABI, for plain tensors: what the raw-pointer entry points cannot see (types,
// shapes, strides, devices) is checked here, and the launch goes to the current stream of the tensors' device.
//
// In Python the same checks, four data_ptr() and two ctypes calls took 4.4 of the 7.1 us of a batch-1 call whose kernel takes 4.6.
//
// True: launched.  False: nothing was done, and the caller takes the general path, which names the error where there is one. That
// path also takes everything that is not a plain tensor: subclasses, wrapped tensors (vmap, grad transforms, functionalisation),
// lazily conjugated, negated or zero tensors, and any call under a torch-function mode.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstdint>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b200_q4f16.h"

namespace {

// The library that the package has loaded (its own or the one that the environment names).
struct Entry {
  decltype(&b200_set_stream) set_stream = nullptr;
  decltype(&b200_q4f16_matmul) matmul = nullptr;
  decltype(&b200_q4f16_matmul_layout) matmul_layout = nullptr;
  decltype(&b200_q4f16_dequantize) dequantize = nullptr;
  decltype(&b200_paged_rope_append) paged_rope_append = nullptr;
  decltype(&b200_paged_attention) paged_attention = nullptr;
  decltype(&b200_token_logprobs) token_logprobs = nullptr;
} g_entry;

const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  static const c10::DispatchKeySet special({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                            c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                            c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor,
                                            c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
  if (!t.defined() || t.key_set().has_any(special) || !t.is_cuda() || t.layout() != c10::kStrided || !t.has_storage()) return nullptr;
  return &t;
}

const at::Tensor* plain_matrix(PyObject* o, at::ScalarType type) {
  const at::Tensor* t = plain(o);
  return t && t->scalar_type() == type && t->dim() == 2 && t->is_contiguous() ? t : nullptr;
}

// The tensors' device if it is everyone's and the current one, else -1.
int common_device(std::initializer_list<const at::Tensor*> ts) {
  const int dev = (*ts.begin())->get_device();
  for (const at::Tensor* t : ts)
    if (t->get_device() != dev) return -1;
  return c10::cuda::current_device() == dev ? dev : -1;
}

PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "matmul(x, wq, scales, out, layout)");
    return nullptr;
  }
  // -1: no layout given.  Any other number that is no layout is for the general path, which refuses it.
  int overflow = 0;
  const long layout = PyLong_AsLongAndOverflow(args[4], &overflow);
  if (layout == -1 && PyErr_Occurred()) return nullptr;
  if (overflow != 0 || layout < -1 || layout > INT32_MAX) Py_RETURN_FALSE;
  try {
    if (!g_entry.matmul || at::impl::torch_function_mode_enabled()) Py_RETURN_FALSE;
    const at::Tensor *x = plain_matrix(args[0], at::kHalf), *wq = plain_matrix(args[1], at::kUInt32),
                     *scales = plain_matrix(args[2], at::kHalf), *out = plain_matrix(args[3], at::kHalf);
    if (!x || !wq || !scales || !out) Py_RETURN_FALSE;
    const int dev = common_device({x, wq, scales, out});
    const int64_t M = x->size(0), K = x->size(1), N = wq->size(0);
    if (dev < 0 || K % 32 != 0 || wq->size(1) * 8 != K || scales->size(0) != N || scales->size(1) != K / 32 || out->size(0) != M ||
        out->size(1) != N)
      Py_RETURN_FALSE;
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    const void *px = x->const_data_ptr(), *pw = wq->const_data_ptr(), *ps = scales->const_data_ptr();
    void* py = out->mutable_data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    g_entry.set_stream(stream);
    rc = layout < 0 ? g_entry.matmul(px, pw, ps, py, M, N, K, stream)
                    : g_entry.matmul_layout(px, pw, ps, py, M, N, K, (int32_t)layout, stream);
    Py_END_ALLOW_THREADS
    return PyBool_FromLong(rc == 0);
  } catch (const std::exception&) {
    Py_RETURN_FALSE;
  }
}

PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "dequantize(wq, scales, out)");
    return nullptr;
  }
  try {
    if (!g_entry.dequantize || at::impl::torch_function_mode_enabled()) Py_RETURN_FALSE;
    const at::Tensor *wq = plain_matrix(args[0], at::kUInt32), *scales = plain_matrix(args[1], at::kHalf), *out = plain_matrix(args[2], at::kHalf);
    if (!wq || !scales || !out) Py_RETURN_FALSE;
    const int dev = common_device({wq, scales, out});
    const int64_t N = wq->size(0), K = wq->size(1) * 8;
    if (dev < 0 || K % 32 != 0 || scales->size(0) != N || scales->size(1) != K / 32 || out->size(0) != N || out->size(1) != K) Py_RETURN_FALSE;
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    const void *pw = wq->const_data_ptr(), *ps = scales->const_data_ptr();
    void* po = out->mutable_data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    g_entry.set_stream(stream);
    rc = g_entry.dequantize(pw, ps, po, N, K, stream);
    Py_END_ALLOW_THREADS
    return PyBool_FromLong(rc == 0);
  } catch (const std::exception&) {
    Py_RETURN_FALSE;
  }
}

// ---- the operators over the paged cache and the logits: a new result tensor, or None where the general path takes the call ----------

// An argument that may be None: false where it is neither that nor a plain contiguous tensor of that type and size.
bool optional_vector(PyObject* o, at::ScalarType type, int64_t size, const at::Tensor** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o);
  if (!t || t->scalar_type() != type || t->dim() != 1 || t->size(0) != size || !t->is_contiguous()) return false;
  *out = t;
  return true;
}
const void* pointer(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }

// A whole number that fits; false: something else, for the general path to name.
bool whole(PyObject* o, int64_t low, int64_t high, int64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0 && *out >= low && *out <= high;
}
bool number(PyObject* o, double* out) {
  if (PyFloat_CheckExact(o)) {
    *out = PyFloat_AS_DOUBLE(o);
    return true;
  }
  int64_t i;
  if (!whole(o, -(1 << 24), 1 << 24, &i)) return false;
  *out = (double)i;
  return true;
}

// The pages, the table and the lengths of a call with `tokens` rows of `type` on `dev`.
bool paged_cache(PyObject* const* args, int64_t tokens, at::ScalarType type, B200PagedCache* c, int dev) {
  const at::Tensor *k = plain(args[0]), *v = plain(args[1]), *table = plain(args[2]), *lengths, *starts;
  if (!k || !v || !table || (type != at::kHalf && type != at::kBFloat16)) return false;
  if (k->scalar_type() != type || v->scalar_type() != type || k->dim() != 4 || v->sizes() != k->sizes()) return false;
  const int64_t page = k->size(2), dim = k->size(3);
  for (const at::Tensor* t : {k, v})
    if (t->stride(3) != 1 || t->stride(2) != dim || (t->size(1) > 1 && t->stride(1) != page * dim)) return false;
  if (table->scalar_type() != at::kInt || table->dim() != 2 || (table->size(1) > 1 && table->stride(1) != 1)) return false;
  const int64_t batch = table->size(0), width = table->size(1);
  if (args[3] == Py_None || !optional_vector(args[3], at::kInt, batch, &lengths) || !optional_vector(args[4], at::kInt, batch + 1, &starts)) return false;
  for (const at::Tensor* t : {k, v, table, lengths})
    if (t->get_device() != dev) return false;
  if (starts ? starts->get_device() != dev : tokens != batch) return false;
  if (batch > INT32_MAX || width > INT32_MAX || k->size(1) > INT32_MAX || page > INT32_MAX || dim > INT32_MAX) return false;
  c->dtype = type == at::kHalf ? B200_F16 : B200_BF16;
  c->kv_heads = (int32_t)k->size(1);
  c->page_size = (int32_t)page;
  c->head_dim = (int32_t)dim;
  c->pages = k->size(0);
  // (the stride of a dimension of one entry says nothing)
  c->k_page_stride = k->size(0) > 1 ? k->stride(0) : k->size(1) * page * dim;
  c->v_page_stride = v->size(0) > 1 ? v->stride(0) : k->size(1) * page * dim;
  c->k_pages = const_cast<void*>(k->const_data_ptr());
  c->v_pages = const_cast<void*>(v->const_data_ptr());
  c->batch = (int32_t)batch;
  c->table_width = (int32_t)width;
  c->table_stride = batch > 1 ? table->stride(0) : width;
  c->tokens = tokens;
  c->max_query = 1;
  c->page_table = table->const_data_ptr();
  c->lengths = lengths->const_data_ptr();
  c->starts = pointer(starts);
  return true;
}

// The result: `given` where it is a fitting tensor, a new one where it is None, else undefined.
at::Tensor result_of(PyObject* given, at::IntArrayRef sizes, const at::Tensor& like) {
  if (given == Py_None) return at::empty(sizes, like.options().requires_grad(false));
  const at::Tensor* t = plain(given);
  if (!t || t->scalar_type() != like.scalar_type() || t->sizes() != sizes || !t->is_contiguous() || t->get_device() != like.get_device()) return {};
  return *t;
}

// paged_rope_append(qkv, cos, sin, k, v, table, lengths, starts, interleaved, positions, out)
PyObject* paged_rope_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11) {
    PyErr_SetString(PyExc_TypeError, "paged_rope_append() takes 11 arguments");
    return nullptr;
  }
  try {
    if (!g_entry.paged_rope_append || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor *qkv = plain(args[0]), *cos = plain_matrix(args[1], at::kFloat), *sin = plain_matrix(args[2], at::kFloat), *positions;
    if (!qkv || !cos || !sin || qkv->dim() != 2 || (qkv->size(1) > 1 && qkv->stride(1) != 1) || cos->sizes() != sin->sizes()) Py_RETURN_NONE;
    const int dev = common_device({qkv, cos, sin});
    const int64_t tokens = qkv->size(0);
    B200PagedCache c = {};
    if (dev < 0 || !PyBool_Check(args[8]) || !paged_cache(args + 3, tokens, qkv->scalar_type(), &c, dev)) Py_RETURN_NONE;
    if (!optional_vector(args[9], at::kInt, tokens, &positions) || (positions && positions->get_device() != dev)) Py_RETURN_NONE;
    if (c.head_dim == 0 || qkv->size(1) % c.head_dim || cos->size(1) > c.head_dim) Py_RETURN_NONE;
    const int64_t heads = qkv->size(1) / c.head_dim - 2 * (int64_t)c.kv_heads;
    if (heads <= 0 || heads > INT32_MAX) Py_RETURN_NONE;
    const at::Tensor out = result_of(args[10], {tokens, heads, c.head_dim}, *qkv);
    if (!out.defined()) Py_RETURN_NONE;
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    const int64_t stride = tokens > 1 ? qkv->stride(0) : qkv->size(1);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_entry.paged_rope_append(&c, qkv->const_data_ptr(), stride, (int32_t)heads, cos->const_data_ptr(), sin->const_data_ptr(), cos->size(0),
                                   (int32_t)(2 * cos->size(1)), args[8] == Py_True, pointer(positions), out.mutable_data_ptr(), stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// paged_attention(q, k, v, table, lengths, starts, max_query, scale, causal, window, cap, slopes, prefix, out, scratch)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 15) {
    PyErr_SetString(PyExc_TypeError, "paged_attention() takes 15 arguments");
    return nullptr;
  }
  try {
    if (!g_entry.paged_attention || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor *q = plain(args[0]), *slopes, *prefix, *scratch = plain(args[14]);
    if (!q || !scratch || q->dim() != 3 || !scratch->is_contiguous()) Py_RETURN_NONE;
    const int dev = common_device({q, scratch});
    const int64_t tokens = q->size(0), heads = q->size(1);
    B200PagedCache c = {};
    if (dev < 0 || tokens == 0 || heads > INT32_MAX || !paged_cache(args + 1, tokens, q->scalar_type(), &c, dev)) Py_RETURN_NONE;
    if (q->size(2) != c.head_dim || q->stride(2) != 1 || (heads > 1 && q->stride(1) != c.head_dim)) Py_RETURN_NONE;
    if (!optional_vector(args[11], at::kFloat, heads, &slopes) || !optional_vector(args[12], at::kInt, c.batch, &prefix)) Py_RETURN_NONE;
    if ((slopes && slopes->get_device() != dev) || (prefix && prefix->get_device() != dev)) Py_RETURN_NONE;
    B200PagedAttention a = {};
    int64_t most = tokens, window;
    double scale = 1.0 / std::sqrt((double)c.head_dim), cap;
    if (c.starts) {
      if (args[6] != Py_None && !whole(args[6], 0, INT32_MAX, &most)) Py_RETURN_NONE;
      if (most > INT32_MAX) Py_RETURN_NONE;
      c.max_query = (int32_t)most;
    }
    if (args[7] != Py_None && !number(args[7], &scale)) Py_RETURN_NONE;
    if (!PyBool_Check(args[8]) || !whole(args[9], 0, INT32_MAX, &window) || !number(args[10], &cap)) Py_RETURN_NONE;
    const at::Tensor out = result_of(args[13], q->sizes(), *q);
    if (!out.defined()) Py_RETURN_NONE;
    a.q = q->const_data_ptr();
    a.q_stride = tokens > 1 ? q->stride(0) : heads * c.head_dim;
    a.out = out.mutable_data_ptr();
    a.heads = (int32_t)heads;
    a.causal = args[8] == Py_True;
    a.window = (int32_t)window;
    a.scale = (float)scale;
    a.cap = (float)cap;
    a.slopes = pointer(slopes);
    a.prefix = pointer(prefix);
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_entry.paged_attention(&c, &a, scratch->mutable_data_ptr(), (int64_t)scratch->nbytes(), stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// token_logprobs(logits, tokens, top): (logprob, entropy, top_logprob, top_token), the last two None without top
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "token_logprobs(logits, tokens, top)");
    return nullptr;
  }
  try {
    if (!g_entry.token_logprobs || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor *x = plain(args[0]), *tokens;
    int64_t top;
    if (!x || x->dim() != 2 || (x->size(1) > 1 && x->stride(1) != 1) || !whole(args[2], 0, 1 << 20, &top)) Py_RETURN_NONE;
    const int64_t rows = x->size(0), V = x->size(1);
    if (args[1] == Py_None || !optional_vector(args[1], at::kInt, rows, &tokens) || rows == 0) Py_RETURN_NONE;
    const int dev = common_device({x, tokens});
    const at::ScalarType t = x->scalar_type();
    if (dev < 0 || top > V || (t != at::kHalf && t != at::kBFloat16 && t != at::kFloat)) Py_RETURN_NONE;
    const auto fp32 = x->options().dtype(at::kFloat).requires_grad(false);
    const at::Tensor logprob = at::empty({rows}, fp32), entropy = at::empty({rows}, fp32);
    at::Tensor best, best_token;
    if (top) {
      best = at::empty({rows, top}, fp32);
      best_token = at::empty({rows, top}, fp32.dtype(at::kInt));
    }
    void *p0 = logprob.mutable_data_ptr(), *p1 = entropy.mutable_data_ptr(), *p2 = top ? best.mutable_data_ptr() : nullptr,
         *p3 = top ? best_token.mutable_data_ptr() : nullptr;
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_entry.token_logprobs(x->const_data_ptr(), t == at::kHalf ? B200_F16 : t == at::kBFloat16 ? B200_BF16 : B200_F32,
                                rows > 1 ? x->stride(0) : V, tokens->const_data_ptr(), p0, p1, p2, p3, rows, V, (int32_t)top, stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) Py_RETURN_NONE;
    // (THPVariable_Wrap gives None for an undefined tensor)
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(logprob), THPVariable_Wrap(entropy), THPVariable_Wrap(best), THPVariable_Wrap(best_token));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// bind(set_stream, matmul, matmul_layout, dequantize, paged_rope_append, paged_attention, token_logprobs): addresses of the loaded
// library's entry points.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kEntries = 7;
  void* p[kEntries] = {};
  for (Py_ssize_t i = 0; n == kEntries && i < n; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  bool all = n == kEntries;
  for (void* q : p) all = all && q;
  if (!all) {
    PyErr_SetString(PyExc_TypeError, "bind() takes the addresses of seven entry points");
    return nullptr;
  }
  g_entry.paged_rope_append = reinterpret_cast<decltype(g_entry.paged_rope_append)>(p[4]);
  g_entry.paged_attention = reinterpret_cast<decltype(g_entry.paged_attention)>(p[5]);
  g_entry.token_logprobs = reinterpret_cast<decltype(g_entry.token_logprobs)>(p[6]);
  g_entry.set_stream = reinterpret_cast<decltype(g_entry.set_stream)>(p[0]);
  g_entry.matmul = reinterpret_cast<decltype(g_entry.matmul)>(p[1]);
  g_entry.matmul_layout = reinterpret_cast<decltype(g_entry.matmul_layout)>(p[2]);
  g_entry.dequantize = reinterpret_cast<decltype(g_entry.dequantize)>(p[3]);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(matmul)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize)), METH_FASTCALL, nullptr},
    {"paged_rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_rope_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(token_logprobs)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_call", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_call() { return PyModule_Create(&kModule); }
