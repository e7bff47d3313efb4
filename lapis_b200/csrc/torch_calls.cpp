// CPython entry points of the device-resident layer: tensor checks, address and stream lookup and the call into
// liblapis_b200.so in native code.
//
// A small call is bound by the host: at 10,000 rows the SpMV kernel takes 2-3 us and the launch 2 us, while the same
// checks written in Python with a ctypes call took 11 us (3.5 us of it torch.cuda.current_stream()).
// Every function returns the library's status, or -1 when an operand is not the kind of tensor it takes; the caller
// (lapis_b200/device.py) then names the operand in the exception it raises.  Those of lapis_b200/attention.py and experts.py make their results
// here (torch.empty took 3.3 us where it was measured, at::empty 0.8) and return them where all went well.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/Exception.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/lapis_b200.h"

namespace {

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool is(const at::Tensor *t, at::ScalarType st) {
  return t != nullptr && t->is_cuda() && t->scalar_type() == st && t->is_contiguous();
}
// Two extents, further ones being 1: a row-major matrix.
bool is_matrix(const at::Tensor *t) {
  for (int64_t d = 2; d < t->dim(); ++d)
    if (t->size(d) != 1) return false;
  return t->dim() >= 2;
}
bool is_index(const at::Tensor *t) {
  return t != nullptr && t->is_cuda() && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->is_contiguous();
}
void *addr(const at::Tensor *t) { return t->numel() == 0 ? nullptr : t->data_ptr(); }
template <typename T>
T *addr_of(const at::Tensor *t) {
  return static_cast<T *>(addr(t));
}
void *stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
lapis_b200_csr_t handle(PyObject *o) { return static_cast<lapis_b200_csr_t>(PyLong_AsVoidPtr(o)); }
PyObject *status(int code) { return PyLong_FromLong(code); }
// Calls the library without the interpreter lock: a launch waits where the stream's queue is full.
template <typename... P, typename... A>
PyObject *call(int (*fn)(P...), A... args) {
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = fn(static_cast<P>(args)...);
  Py_END_ALLOW_THREADS
  return status(code);
}

// What Python calls.  torch reports some operands by a C++ exception (a tensor without storage has no address, a sparse
// one no contiguity), which must not leave a C function; an argument that is no integer leaves a Python one.
template <PyObject *(*CALL)(PyObject *const *), Py_ssize_t ARGS>
PyObject *entry(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
  if (nargs != ARGS) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    PyObject *result = CALL(a);
    if (PyErr_Occurred() == nullptr) return result;
    Py_XDECREF(result);
  } catch (const c10::Error &e) {
    if (PyErr_Occurred() == nullptr) PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    if (PyErr_Occurred() == nullptr) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// spmv(handle, nrows, ncols, x, y, accumulate)
PyObject *py_spmv(PyObject *const *a) {
  const int accumulate = PyObject_IsTrue(a[5]);
  if (accumulate < 0) return nullptr;
  const at::Tensor *x = tensor(a[3]), *y = tensor(a[4]);
  if (!is(x, at::kDouble) || !is(y, at::kDouble)) return status(-1);
  if (y->numel() != PyLong_AsLongLong(a[1]) || x->numel() != PyLong_AsLongLong(a[2])) return status(-1);
  return call(lapis_b200_spmv_f64, handle(a[0]), addr_of<double>(x), addr_of<double>(y), accumulate, stream());
}

// spmm(handle, nrows, ncols, B, C, accumulate)
PyObject *py_spmm(PyObject *const *a) {
  const int accumulate = PyObject_IsTrue(a[5]);
  if (accumulate < 0) return nullptr;
  const at::Tensor *B = tensor(a[3]), *C = tensor(a[4]);
  if (!is(B, at::kDouble) || !is(C, at::kDouble) || !is_matrix(B) || !is_matrix(C)) return status(-1);
  if (C->size(0) != PyLong_AsLongLong(a[1]) || B->size(0) != PyLong_AsLongLong(a[2]) || B->size(1) != C->size(1)) return status(-1);
  return call(lapis_b200_spmm_f64, handle(a[0]), B->size(1), addr_of<double>(B), addr_of<double>(C), accumulate, stream());
}

// spmm_dcsr(i1, p2, i2, val, B, C, ncols)
PyObject *py_spmm_dcsr(PyObject *const *a) {
  const at::Tensor *i1 = tensor(a[0]), *p2 = tensor(a[1]), *i2 = tensor(a[2]), *val = tensor(a[3]), *B = tensor(a[4]), *C = tensor(a[5]);
  const long long ncols = PyLong_AsLongLong(a[6]);
  if (!is_index(i1) || !is_index(p2) || !is_index(i2) || i1->scalar_type() != p2->scalar_type() ||
      i2->scalar_type() != p2->scalar_type() || !is(val, at::kDouble) || !is(B, at::kDouble) || !is(C, at::kDouble))
    return status(-1);
  if (B->dim() != 2 || C->dim() != 2 || B->size(0) != ncols || B->size(1) != C->size(1) || p2->numel() != i1->numel() + 1)
    return status(-1);
  return call(lapis_b200_spmm_dcsr_f64, (int)p2->element_size(), C->size(0), ncols, i1->numel(), B->size(1), addr(i1), addr(p2),
              addr(i2), addr_of<double>(val), addr_of<double>(B), addr_of<double>(C), stream());
}

// bspmm(pos, crd, val, B, C, n2, accumulate)
PyObject *py_bspmm(PyObject *const *a) {
  const int accumulate = PyObject_IsTrue(a[6]);
  if (accumulate < 0) return nullptr;
  const at::Tensor *pos = tensor(a[0]), *crd = tensor(a[1]), *val = tensor(a[2]), *B = tensor(a[3]), *C = tensor(a[4]);
  const long long n2 = PyLong_AsLongLong(a[5]);
  if (!is_index(pos) || !is_index(crd) || pos->scalar_type() != crd->scalar_type() || !is(val, at::kFloat) || !is(B, at::kFloat) ||
      !is(C, at::kFloat) || B->dim() != 3 || C->dim() != 3)
    return status(-1);
  const int64_t n1 = pos->numel() - 1, dh = B->size(1), nh = B->size(2);
  if (B->size(0) != n2 || val->numel() != crd->numel() * nh || C->size(0) != n1 || C->size(1) != dh || C->size(2) != nh) return status(-1);
  return call(lapis_b200_bspmm_csrv_f32, (int)pos->element_size(), n1, n2, nh, dh, addr(pos), addr(crd), addr_of<float>(val),
              addr_of<float>(B), addr_of<float>(C), accumulate, stream());
}

// bgemm(A, B, C): [M,K]x[K,N] or [b,M,K]x[b,K,N]
PyObject *py_bgemm(PyObject *const *a) {
  const at::Tensor *A = tensor(a[0]), *B = tensor(a[1]), *C = tensor(a[2]);
  if (!is(A, at::kFloat) || !is(B, at::kFloat) || !is(C, at::kFloat)) return status(-1);
  const int64_t d = A->dim();
  if ((d != 2 && d != 3) || B->dim() != d || C->dim() != d) return status(-1);
  const int64_t batch = d == 3 ? A->size(0) : 1, M = A->size(d - 2), K = A->size(d - 1), N = B->size(d - 1);
  if (B->size(d - 2) != K || C->size(d - 2) != M || C->size(d - 1) != N || (d == 3 && (B->size(0) != batch || C->size(0) != batch)))
    return status(-1);
  return call(lapis_b200_bgemm_f32, batch, M, N, K, addr_of<float>(A), addr_of<float>(B), addr_of<float>(C), stream());
}

// ---- attention (lapis_b200/attention.py) ----

// LAPIS_F32 ... of a tensor's elements, or -1.
int type_of(const at::Tensor *t) {
  switch (t->scalar_type()) {
    case at::kFloat: return LAPIS_F32;
    case at::kHalf: return LAPIS_F16;
    case at::kBFloat16: return LAPIS_BF16;
    default: return -1;
  }
}
bool on_device(const at::Tensor *t) { return t->is_cuda() && t->device().index() == c10::cuda::current_device(); }
// Heads of tokens, [tokens, heads, dim], whose values lie next to one another.
bool heads_of(PyObject *o, int type, int64_t tokens, int64_t dim, lapis_b200_heads *h) {
  const at::Tensor *t = tensor(o);
  if (t == nullptr || t->dim() != 3 || !on_device(t) || type_of(t) != type || t->size(0) != tokens || t->size(2) != dim) return false;
  if (dim > 1 && t->stride(2) != 1 && t->numel() > 0) return false;
  *h = {addr(t), t->size(1), t->stride(0), t->stride(1)};
  return true;
}
at::Tensor result(const at::Tensor *like, at::IntArrayRef sizes) { return at::empty(sizes, like->options()); }
at::Tensor result(const at::Tensor *like, at::ScalarType type, at::IntArrayRef sizes) { return at::empty(sizes, like->options().dtype(type)); }
// The status of a call where it is not 0; otherwise the results, one as itself, several as a tuple.
template <typename... R>
PyObject *results(PyObject *code, const R &...r) {
  if (code == nullptr || PyLong_AsLong(code) != 0) return code;
  Py_DECREF(code);
  if constexpr (sizeof...(R) == 1) return THPVariable_Wrap(r...);
  return Py_BuildValue(sizeof...(R) == 2 ? "(NN)" : "(NNN)", THPVariable_Wrap(r)...);
}
bool indices_of(PyObject *o, int64_t count, int *idx_bytes, const void **p) {
  const at::Tensor *t = tensor(o);
  if (!is_index(t) || !on_device(t) || t->dim() != 1 || (count >= 0 && t->numel() != count)) return false;
  if (*idx_bytes != 0 && *idx_bytes != (int)t->element_size()) return false;
  *idx_bytes = (int)t->element_size();
  *p = addr(t);
  return true;
}
bool lists_of(PyObject *pos, PyObject *crd, lapis_b200_page_lists *l) {
  *l = {};
  if (!indices_of(pos, -1, &l->idx_bytes, &l->d_pos) || !indices_of(crd, -1, &l->idx_bytes, &l->d_crd)) return false;
  l->rows = tensor(pos)->numel() - 1;
  l->entries = tensor(crd)->numel();
  return l->rows >= 0;
}
// a: q_weight, k_weight, cos, sin, eps, interleaved
bool norm_rope_of(PyObject *const *a, int type, int64_t dim, lapis_b200_norm_rope *how) {
  const at::Tensor *w[2] = {tensor(a[0]), tensor(a[1])}, *cos = tensor(a[2]), *sin = tensor(a[3]);
  for (const at::Tensor *t : w)
    if (t == nullptr || !on_device(t) || !t->is_contiguous() || t->dim() != 1 || t->numel() != dim || t->scalar_type() != w[0]->scalar_type())
      return false;
  for (const at::Tensor *t : {cos, sin})
    if (!is(t, at::kFloat) || !on_device(t) || t->dim() != 2 || t->size(0) != cos->size(0) || t->size(1) != cos->size(1)) return false;
  const int weight_type = type_of(w[0]);
  if (weight_type != LAPIS_F32 && weight_type != type) return false;
  if (2 * cos->size(1) > dim) return false;
  const double eps = PyFloat_AsDouble(a[4]);
  const int interleaved = PyObject_IsTrue(a[5]);
  *how = {addr(w[0]), addr(w[1]), weight_type, addr_of<float>(cos), addr_of<float>(sin), cos->size(0), 2 * cos->size(1), interleaved, eps};
  return true;
}
const lapis_b200_kv_cache *cache_of(PyObject *o) { return static_cast<const lapis_b200_kv_cache *>(PyLong_AsVoidPtr(o)); }

// qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps, interleaved, place) -> q, k
PyObject *py_qk_norm_rope(PyObject *const *a) {
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]);
  if (q == nullptr || q->dim() != 3) return status(-1);
  const int64_t tokens = q->size(0), dim = q->size(2);
  const int type = type_of(q);
  lapis_b200_heads hq, hk;
  lapis_b200_norm_rope how;
  int idx_bytes = 0;
  const void *place;
  if (type < 0 || !heads_of(a[0], type, tokens, dim, &hq) || !heads_of(a[1], type, tokens, dim, &hk) || !norm_rope_of(a + 2, type, dim, &how) ||
      !indices_of(a[8], tokens, &idx_bytes, &place))
    return status(-1);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor q_out = result(q, q->sizes()), k_out = result(k, k->sizes());
  return results(call(lapis_b200_qk_norm_rope, type, tokens, dim, &hq, &hk, &how, idx_bytes, place, addr(&q_out), addr(&k_out), stream()), q_out, k_out);
}

// qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, eps, interleaved, place) -> of q, of k, of the weights [2, dim]
PyObject *py_qk_norm_rope_backward(PyObject *const *a) {
  const at::Tensor *q = tensor(a[2]), *k = tensor(a[3]);
  if (q == nullptr || q->dim() != 3) return status(-1);
  const int64_t tokens = q->size(0), dim = q->size(2);
  const int type = type_of(q);
  lapis_b200_heads hdq, hdk, hq, hk;
  lapis_b200_norm_rope how;
  int idx_bytes = 0;
  const void *place;
  if (type < 0 || !heads_of(a[0], type, tokens, dim, &hdq) || !heads_of(a[1], type, tokens, dim, &hdk) ||
      !heads_of(a[2], type, tokens, dim, &hq) || !heads_of(a[3], type, tokens, dim, &hk) || !norm_rope_of(a + 4, type, dim, &how) ||
      !indices_of(a[10], tokens, &idx_bytes, &place) || hdq.heads != hq.heads || hdk.heads != hk.heads)
    return status(-1);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor q_grad = result(q, q->sizes()), k_grad = result(k, k->sizes()), weights = result(q, at::kFloat, {2, dim});
  float *const dqw = addr_of<float>(&weights);
  return results(call(lapis_b200_qk_norm_rope_backward, type, tokens, dim, &hdq, &hdk, &hq, &hk, &how, idx_bytes, place, addr(&q_grad), addr(&k_grad), dqw,
                      dqw == nullptr ? nullptr : dqw + dim, stream()),
                 q_grad, k_grad, weights);
}

// kv_append(cache, k, v, pos, crd, row, place)
PyObject *py_kv_append(PyObject *const *a) {
  const lapis_b200_kv_cache *cache = cache_of(a[0]);
  const at::Tensor *k = tensor(a[1]);
  if (cache == nullptr || k == nullptr || k->dim() != 3) return status(-1);
  const int64_t tokens = k->size(0);
  const int type = type_of(k);
  lapis_b200_heads hk, hv;
  lapis_b200_page_lists lists;
  const void *row, *place;
  if (type < 0 || !heads_of(a[1], type, tokens, cache->dim, &hk) || !heads_of(a[2], type, tokens, cache->dim, &hv) ||
      hk.heads != cache->heads || hv.heads != cache->heads || !lists_of(a[3], a[4], &lists) ||
      !indices_of(a[5], tokens, &lists.idx_bytes, &row) || !indices_of(a[6], tokens, &lists.idx_bytes, &place))
    return status(-1);
  return call(lapis_b200_kv_append, type, tokens, nullptr, &hk, &hv, nullptr, cache, &lists, row, place, nullptr, stream());
}

// kv_append_norm_rope(cache, q, k, v, q_weight, k_weight, cos, sin, eps, interleaved, pos, crd, row, place) -> q
PyObject *py_kv_append_norm_rope(PyObject *const *a) {
  const lapis_b200_kv_cache *cache = cache_of(a[0]);
  const at::Tensor *q = tensor(a[1]), *k = tensor(a[2]);
  if (cache == nullptr || k == nullptr || k->dim() != 3) return status(-1);
  const int64_t tokens = k->size(0);
  const int type = type_of(k);
  lapis_b200_heads hq, hk, hv;
  lapis_b200_norm_rope how;
  lapis_b200_page_lists lists;
  const void *row, *place;
  if (type < 0 || !heads_of(a[1], type, tokens, cache->dim, &hq) || !heads_of(a[2], type, tokens, cache->dim, &hk) ||
      !heads_of(a[3], type, tokens, cache->dim, &hv) || hk.heads != cache->heads || hv.heads != cache->heads || !norm_rope_of(a + 4, type, cache->dim, &how) || !lists_of(a[10], a[11], &lists) ||
      !indices_of(a[12], tokens, &lists.idx_bytes, &row) || !indices_of(a[13], tokens, &lists.idx_bytes, &place))
    return status(-1);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor q_out = result(q, q->sizes());
  return results(call(lapis_b200_kv_append, type, tokens, &hq, &hk, &hv, &how, cache, &lists, row, place, addr(&q_out), stream()), q_out);
}

// kv_read(cache, pos, crd, row, place, type: LAPIS_F32, LAPIS_F16 or LAPIS_BF16) -> k, v
PyObject *py_kv_read(PyObject *const *a) {
  const lapis_b200_kv_cache *cache = cache_of(a[0]);
  const at::Tensor *row_of = tensor(a[3]);
  const long type = PyLong_AsLong(a[5]);
  if (cache == nullptr || row_of == nullptr || type < LAPIS_F32 || type > LAPIS_BF16) return status(-1);
  const int64_t tokens = row_of->numel();
  lapis_b200_page_lists lists;
  const void *row, *place;
  if (!lists_of(a[1], a[2], &lists) || !indices_of(a[3], tokens, &lists.idx_bytes, &row) || !indices_of(a[4], tokens, &lists.idx_bytes, &place))
    return status(-1);
  const at::ScalarType scalar = type == LAPIS_F32 ? at::kFloat : type == LAPIS_F16 ? at::kHalf : at::kBFloat16;
  const at::Tensor k = result(row_of, scalar, {tokens, cache->heads, cache->dim}), v = result(row_of, scalar, {tokens, cache->heads, cache->dim});
  return results(call(lapis_b200_kv_read, cache, &lists, tokens, row, place, type, addr(&k), addr(&v), stream()), k, v);
}

// paged_attention(cache, q, pos, crd, length, scale, window, return_lse) -> out, or out and lse
PyObject *py_paged_attention(PyObject *const *a) {
  const lapis_b200_kv_cache *cache = cache_of(a[0]);
  const at::Tensor *q = tensor(a[1]);
  if (cache == nullptr || q == nullptr || q->dim() != 3) return status(-1);
  const int64_t requests = q->size(0);
  const int type = type_of(q);
  lapis_b200_heads hq;
  lapis_b200_page_lists lists;
  const void *length;
  const double scale = PyFloat_AsDouble(a[5]);
  const long long window = PyLong_AsLongLong(a[6]);
  const int with_lse = PyObject_IsTrue(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (type < 0 || !heads_of(a[1], type, requests, cache->dim, &hq) || !lists_of(a[2], a[3], &lists) ||
      !indices_of(a[4], requests, &lists.idx_bytes, &length))
    return status(-1);
  const at::Tensor out = result(q, q->sizes());
  if (!with_lse)
    return results(call(lapis_b200_paged_attention, type, requests, &hq, cache, &lists, length, scale, window, addr(&out), nullptr, stream()), out);
  const at::Tensor lse = result(q, at::kFloat, {requests, hq.heads});
  return results(call(lapis_b200_paged_attention, type, requests, &hq, cache, &lists, length, scale, window, addr(&out), addr_of<float>(&lse), stream()),
                 out, lse);
}

// ---- a layer of experts (lapis_b200/experts.py) ----

// Rows [rows, dim] of a type whose values lie next to one another.
bool rows_of(const at::Tensor *t, int type, int64_t rows, int64_t dim) {
  if (t == nullptr || t->dim() != 2 || !on_device(t) || type_of(t) != type || t->size(0) != rows || t->size(1) != dim) return false;
  return dim <= 1 || t->stride(1) == 1 || t->numel() == 0;
}
bool matrix_of(PyObject *o, at::ScalarType type, int64_t rows, int64_t columns, const at::Tensor **t) {
  *t = tensor(o);
  return is(*t, type) && on_device(*t) && (*t)->dim() == 2 && (*t)->size(0) == rows && (*t)->size(1) == columns;
}
// a: pos, crd, place
bool expert_lists_of(PyObject *const *a, lapis_b200_expert_lists *l) {
  const at::Tensor *pos = tensor(a[0]), *crd = tensor(a[1]), *place = tensor(a[2]);
  for (const at::Tensor *t : {pos, crd, place})
    if (!is(t, at::kInt) || !on_device(t)) return false;
  if (pos->dim() != 1 || pos->numel() < 1 || crd->dim() != 1 || place->dim() != 2 || crd->numel() != place->numel()) return false;
  *l = {place->size(0), place->size(1), pos->numel() - 1, addr_of<int32_t>(pos), addr_of<int32_t>(crd), addr_of<int32_t>(place)};
  return true;
}

// route(logits, k, normalise) -> weights, expert
PyObject *py_route(PyObject *const *a) {
  const at::Tensor *logits = tensor(a[0]);
  const long long k = PyLong_AsLongLong(a[1]);
  const int normalise = PyObject_IsTrue(a[2]);
  if (PyErr_Occurred()) return nullptr;
  if (logits == nullptr || logits->dim() != 2 || k < 0 || k > logits->size(1)) return status(-1);
  const int64_t tokens = logits->size(0), experts = logits->size(1);
  const int type = type_of(logits);
  if (type < 0 || !rows_of(logits, type, tokens, experts)) return status(-1);
  const at::Tensor weights = result(logits, at::kFloat, {tokens, k}), expert = result(logits, at::kInt, {tokens, k});
  return results(call(lapis_b200_route, type, tokens, experts, addr(logits), logits->stride(0), k, normalise, addr_of<float>(&weights),
                      addr_of<int32_t>(&expert), stream()),
                 weights, expert);
}

// route_backward(dweights, logits, expert, normalise) -> of the logits
PyObject *py_route_backward(PyObject *const *a) {
  const at::Tensor *logits = tensor(a[1]), *dweights, *expert;
  const int normalise = PyObject_IsTrue(a[3]);
  if (PyErr_Occurred()) return nullptr;
  if (logits == nullptr || logits->dim() != 2) return status(-1);
  const int64_t tokens = logits->size(0), experts = logits->size(1);
  const int type = type_of(logits);
  const at::Tensor *chosen = tensor(a[2]);
  if (chosen == nullptr || chosen->dim() != 2 || chosen->size(1) > experts) return status(-1);
  const int64_t k = chosen->size(1);
  if (type < 0 || !rows_of(logits, type, tokens, experts) || !matrix_of(a[0], at::kFloat, tokens, k, &dweights) ||
      !matrix_of(a[2], at::kInt, tokens, k, &expert))
    return status(-1);
  const at::Tensor dlogits = result(logits, {tokens, experts});
  return results(call(lapis_b200_route_backward, type, tokens, experts, addr(logits), logits->stride(0), k, normalise, addr_of<int32_t>(expert),
                      addr_of<float>(dweights), addr(&dlogits), stream()),
                 dlogits);
}

// expert_lists(expert, experts) -> pos, crd, place
PyObject *py_expert_lists(PyObject *const *a) {
  const at::Tensor *expert = tensor(a[0]);
  const long long experts = PyLong_AsLongLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if (!is_index(expert) || !on_device(expert) || expert->dim() != 2 || experts < 0 || experts > (1 << 20)) return status(-1);
  const int64_t tokens = expert->size(0), k = expert->size(1);
  const at::Tensor pos = result(expert, at::kInt, {experts + 1}), crd = result(expert, at::kInt, {tokens * k}), place = result(expert, at::kInt, {tokens, k});
  return results(call(lapis_b200_expert_lists_make, (int)expert->element_size(), tokens, k, experts, addr(expert), addr_of<int32_t>(&pos),
                      addr_of<int32_t>(&crd), addr_of<int32_t>(&place), stream()),
                 pos, crd, place);
}

// expert_gather(x, pos, crd, place) -> rows
PyObject *py_expert_gather(PyObject *const *a) {
  const at::Tensor *x = tensor(a[0]);
  lapis_b200_expert_lists l;
  if (x == nullptr || x->dim() != 2 || !expert_lists_of(a + 1, &l)) return status(-1);
  const int type = type_of(x);
  const int64_t dim = x->size(1);
  if (type < 0 || !rows_of(x, type, l.tokens, dim)) return status(-1);
  const at::Tensor rows = result(x, {l.tokens * l.k, dim});
  return results(call(lapis_b200_expert_gather, type, dim, addr(x), x->stride(0), &l, addr(&rows), stream()), rows);
}

// expert_combine(rows, weights or None, pos, crd, place) -> out
PyObject *py_expert_combine(PyObject *const *a) {
  const at::Tensor *rows = tensor(a[0]), *weights = nullptr;
  lapis_b200_expert_lists l;
  if (rows == nullptr || rows->dim() != 2 || !expert_lists_of(a + 2, &l)) return status(-1);
  const int type = type_of(rows);
  const int64_t dim = rows->size(1);
  if (type < 0 || !rows_of(rows, type, l.tokens * l.k, dim) || (a[1] != Py_None && !matrix_of(a[1], at::kFloat, l.tokens, l.k, &weights))) return status(-1);
  const at::Tensor out = result(rows, {l.tokens, dim});
  return results(call(lapis_b200_expert_combine, type, dim, addr(rows), rows->stride(0), &l, weights == nullptr ? nullptr : addr_of<float>(weights),
                      addr(&out), stream()),
                 out);
}

// expert_combine_backward(dout, rows, weights, pos, crd, place) -> of rows, of weights
PyObject *py_expert_combine_backward(PyObject *const *a) {
  const at::Tensor *dout = tensor(a[0]), *rows = tensor(a[1]), *weights;
  lapis_b200_expert_lists l;
  if (rows == nullptr || rows->dim() != 2 || !expert_lists_of(a + 3, &l)) return status(-1);
  const int type = type_of(rows);
  const int64_t dim = rows->size(1);
  if (type < 0 || !rows_of(rows, type, l.tokens * l.k, dim) || !rows_of(dout, type, l.tokens, dim) || !matrix_of(a[2], at::kFloat, l.tokens, l.k, &weights))
    return status(-1);
  const at::Tensor drows = result(rows, rows->sizes()), dweights = result(weights, weights->sizes());
  return results(call(lapis_b200_expert_combine_backward, type, dim, addr(dout), dout->stride(0), addr(rows), rows->stride(0), &l, addr_of<float>(weights),
                      addr(&drows), addr_of<float>(&dweights), stream()),
                 drows, dweights);
}

// int4_matmul(weights, x) -> y, int4_matmul_lists(weights, x, fetch, pos, crd, place) -> y
const lapis_b200_int4 *int4_of(PyObject *o) { return static_cast<const lapis_b200_int4 *>(PyLong_AsVoidPtr(o)); }
PyObject *int4_product(const lapis_b200_int4 *w, PyObject *rows, int fetch, const lapis_b200_expert_lists *l) {
  const at::Tensor *x = tensor(rows);
  if (PyErr_Occurred()) return nullptr;
  if (w == nullptr || x == nullptr || x->dim() != 2) return status(-1);
  const int type = type_of(x);
  const int64_t given = x->size(0);
  if (type < 0 || !rows_of(x, type, given, w->columns)) return status(-1);
  const at::Tensor y = result(x, {l == nullptr ? given : l->tokens * l->k, w->gated ? w->outputs / 2 : w->outputs});
  return results(call(lapis_b200_int4_matmul, type, w, given, addr(x), x->stride(0), l, fetch, addr(&y), stream()), y);
}
PyObject *py_int4_matmul(PyObject *const *a) { return int4_product(int4_of(a[0]), a[1], 0, nullptr); }
PyObject *py_int4_matmul_lists(PyObject *const *a) {
  const int fetch = PyObject_IsTrue(a[2]);
  lapis_b200_expert_lists l;
  if (PyErr_Occurred()) return nullptr;
  if (!expert_lists_of(a + 3, &l)) return status(-1);
  return int4_product(int4_of(a[0]), a[1], fetch, &l);
}

template <PyObject *(*CALL)(PyObject *const *), Py_ssize_t ARGS>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<CALL, ARGS>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<py_spmv, 6>("spmv"),   method<py_spmm, 6>("spmm"),   method<py_spmm_dcsr, 7>("spmm_dcsr"),
                         method<py_bspmm, 7>("bspmm"), method<py_bgemm, 3>("bgemm"),
                         method<py_qk_norm_rope, 9>("qk_norm_rope"), method<py_qk_norm_rope_backward, 11>("qk_norm_rope_backward"),
                         method<py_kv_append, 7>("kv_append"), method<py_kv_append_norm_rope, 14>("kv_append_norm_rope"),
                         method<py_kv_read, 6>("kv_read"), method<py_paged_attention, 8>("paged_attention"),
                         method<py_route, 3>("route"), method<py_route_backward, 4>("route_backward"), method<py_expert_lists, 2>("expert_lists"),
                         method<py_expert_gather, 4>("expert_gather"), method<py_expert_combine, 5>("expert_combine"),
                         method<py_expert_combine_backward, 6>("expert_combine_backward"), method<py_int4_matmul, 2>("int4_matmul"),
                         method<py_int4_matmul_lists, 6>("int4_matmul_lists"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
