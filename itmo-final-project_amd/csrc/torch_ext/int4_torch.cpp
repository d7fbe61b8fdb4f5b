// int4_hip._int4_torch: the Python entry points' call path in native code for
// plain operands.
//
// A one-row product of a small linear takes 3.6 us on the GPU; checking five
// tensors, allocating the output and marshalling sixteen ctypes arguments in
// Python took 13 us of host time per call, so eager calls were bound by it.
// These functions do the same checks, allocation and C-ABI call (the addresses
// come from the library that _lib.py has loaded).  They return None, having done
// nothing, for everything else: other types, dtypes, strides or devices,
// invalid arguments, tensor subclasses, tracing, functorch transforms and
// dispatch or function modes.  The Python code then runs as it always did and
// raises the errors it always raised.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <array>
#include <map>
#include <vector>

#include "int4_hip.h"

namespace {

struct Api {
  decltype(&w4a16_gemm) gemm;
  decltype(&w4a16_workspace_bytes) workspace_bytes;
  decltype(&w4a16_gemm_grouped) gemm_grouped;
  decltype(&w4a16_grouped_workspace_bytes) grouped_workspace_bytes;
  decltype(&w4_quantize_grouped) quantize_grouped;
  decltype(&w4_quantize) quantize;
  decltype(&w4_dequantize) dequantize;
  decltype(&w4_paged_append) paged_append;
  decltype(&w4_paged_attention_workspace_bytes) paged_attention_workspace_bytes;
  decltype(&w4_paged_attention) paged_attention;
  decltype(&w4_paged_evict_scratch_words) paged_evict_scratch_words;
  decltype(&w4_paged_evict) paged_evict;
  decltype(&w4_token_logprobs_workspace_bytes) token_logprobs_workspace_bytes;
  decltype(&w4_token_logprobs) token_logprobs;
  decltype(&w4_paged8_append) paged8_append;
  decltype(&w4_paged8_read) paged8_read;
  decltype(&w4_paged8_attention_workspace_bytes) paged8_attention_workspace_bytes;
  decltype(&w4_paged8_attention) paged8_attention;
  decltype(&w4_verify_drafts_workspace_bytes) verify_drafts_workspace_bytes;
  decltype(&w4_verify_drafts) verify_drafts;
};
Api api{};
PyObject* py_workspace = nullptr;  // (device index, stream, bytes) -> (address, bytes)
PyObject* py_check = nullptr;      // raises for a nonzero status

// Nothing that has to see the individual operations is active on this thread.
bool quiet() {
  return api.gemm != nullptr && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         at::impl::PythonTorchFunctionTLS::stack_len() == 0 && !torch::jit::tracer::isTracing();
}

const c10::DispatchKeySet kWrapped =
    c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                         c10::DispatchKey::Python, c10::DispatchKey::Functionalize});

// The tensor behind a plain GPU tensor or parameter, else null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != c10::kStrided || t.is_neg() || t.key_set().has_any(kWrapped))
    return nullptr;
  return &t;
}

int act_code(at::ScalarType t) {
  return t == at::kBFloat16 ? W4_DTYPE_BF16 : t == at::kHalf ? W4_DTYPE_FP16 : -1;
}

// Group size of a valid dense weight triple on `dev` for K activations, else 0.
int64_t weight_group(const at::Tensor* q, const at::Tensor* s, const at::Tensor* z, c10::Device dev, int64_t K) {
  if (!q || !s || !z || q->device() != dev || s->device() != dev || z->device() != dev) return 0;
  if (q->scalar_type() != at::kInt || q->dim() != 2 || s->scalar_type() != at::kHalf ||
      z->scalar_type() != at::kHalf || s->dim() != 2 || s->sizes() != z->sizes())
    return 0;
  if (q->size(0) * 8 != K || s->size(1) != q->size(1) || s->size(0) < 1) return 0;
  if (!q->is_contiguous() || !s->is_contiguous() || !z->is_contiguous()) return 0;
  const int64_t G = K / s->size(0);
  return G * s->size(0) == K && G >= 8 && (G & (G - 1)) == 0 ? G : 0;
}

bool current(c10::Device dev) { return c10::hip::current_device() == dev.index(); }

// The stream's workspace (kept and grown by the Python side); false: exception set.
bool workspace(c10::Device dev, void* stream, size_t bytes, void** ptr, size_t* size) {
  *ptr = nullptr;
  *size = 0;
  if (bytes == 0) return true;
  PyObject* r = PyObject_CallFunction(py_workspace, "iKK", (int)dev.index(), (unsigned long long)(uintptr_t)stream,
                                      (unsigned long long)bytes);
  if (!r) return false;
  unsigned long long p = 0, n = 0;
  const bool ok = PyArg_ParseTuple(r, "KK", &p, &n);
  Py_DECREF(r);
  *ptr = reinterpret_cast<void*>(p);
  *size = n;
  return ok;
}

// false: exception set.
bool check(int rc, const char* what) {
  if (rc == W4_OK) return true;
  PyObject* r = PyObject_CallFunction(py_check, "is", rc, what);
  Py_XDECREF(r);
  if (r) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", what, rc);
  return false;
}

at::Tensor empty(c10::IntArrayRef sizes, at::ScalarType dtype, c10::Device dev) {
  return at::empty(sizes, at::TensorOptions().dtype(dtype).device(dev));
}

PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !quiet()) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0]);
  if (!x || x->dim() < 1 || !x->is_contiguous()) Py_RETURN_NONE;
  const int dt = act_code(x->scalar_type());
  const int64_t K = x->size(-1);
  const c10::Device dev = x->device();
  if (dt < 0 || K < 8 || x->numel() == 0 || !current(dev)) Py_RETURN_NONE;
  const at::Tensor *q = plain(args[1]), *s = plain(args[2]), *z = plain(args[3]);
  const int64_t G = weight_group(q, s, z, dev, K);
  if (G == 0 || G > INT32_MAX) Py_RETURN_NONE;
  const int64_t M = x->numel() / K, N = q->size(1);
  if (N == 0) Py_RETURN_NONE;
  std::vector<int64_t> sizes(x->sizes().begin(), x->sizes().end());
  sizes.back() = N;
  at::Tensor y = empty(sizes, x->scalar_type(), dev);
  // a pure function of the shape (and the CU count of the one GPU type): memoised
  static std::map<std::array<int64_t, 4>, size_t> memo;
  const std::array<int64_t, 4> key{M, N, K, G};
  auto it = memo.find(key);
  if (it == memo.end()) {
    if (memo.size() > 4096) memo.clear();
    it = memo.emplace(key, api.workspace_bytes(M, N, K, (int)G)).first;
  }
  const size_t need = it->second;  // the callback below may let another thread at the memo
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, need, &ws, &ws_bytes)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.gemm(x->const_data_ptr(), dt, M, N, K, K, 1, static_cast<const int32_t*>(q->const_data_ptr()),
                static_cast<const uint16_t*>(s->const_data_ptr()), static_cast<const uint16_t*>(z->const_data_ptr()),
                (int)G, y.mutable_data_ptr(), N, ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4a16_gemm")) return nullptr;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (xs, weights, out or None) -> list of outputs
PyObject* matmul_grouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !quiet()) Py_RETURN_NONE;
  auto seq = [](PyObject* o) { return PyList_CheckExact(o) || PyTuple_CheckExact(o); };
  if (!seq(args[0]) || !seq(args[1]) || (args[2] != Py_None && !seq(args[2]))) Py_RETURN_NONE;
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(args[0]);
  if (count < 1 || count > W4_MAX_GROUPED || PySequence_Fast_GET_SIZE(args[1]) != count ||
      (args[2] != Py_None && PySequence_Fast_GET_SIZE(args[2]) < count))
    Py_RETURN_NONE;
  // Owned: the workspace callback and the launch let other threads run, which may
  // take the operands out of the caller's lists.
  struct Item {
    at::Tensor x, q, s, z, out;
    int64_t K, N, G;
  };
  std::array<Item, W4_MAX_GROUPED> it;
  int64_t M = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    Item& a = it[i];
    const at::Tensor* x = plain(PySequence_Fast_GET_ITEM(args[0], i));
    if (!x || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 || ((uintptr_t)x->const_data_ptr() % 16) != 0)
      Py_RETURN_NONE;
    a.x = *x;
    a.K = x->size(-1);
    const int64_t rows = x->numel() / a.K;
    if (i == 0) M = rows;
    if (rows != M || x->scalar_type() != it[0].x.scalar_type() || x->device() != it[0].x.device()) Py_RETURN_NONE;
    PyObject* w = PySequence_Fast_GET_ITEM(args[1], i);
    if (!seq(w) || PySequence_Fast_GET_SIZE(w) != 3) Py_RETURN_NONE;
    const at::Tensor *q = plain(PySequence_Fast_GET_ITEM(w, 0)), *s = plain(PySequence_Fast_GET_ITEM(w, 1)),
                     *z = plain(PySequence_Fast_GET_ITEM(w, 2));
    a.G = weight_group(q, s, z, x->device(), a.K);
    if (a.G == 0 || a.G > INT32_MAX) Py_RETURN_NONE;
    a.q = *q;
    a.s = *s;
    a.z = *z;
    a.N = q->size(1);
    if (a.N == 0) Py_RETURN_NONE;
    if (args[2] != Py_None) {
      const at::Tensor* out = plain(PySequence_Fast_GET_ITEM(args[2], i));
      if (!out || x->dim() != 2 || out->dim() != 2 || out->size(0) != M || out->size(1) != a.N ||
          !out->is_contiguous() || out->scalar_type() != x->scalar_type() || out->device() != x->device())
        Py_RETURN_NONE;
      a.out = *out;
    }
  }
  const c10::Device dev = it[0].x.device();
  const int dt = act_code(it[0].x.scalar_type());
  if (dt < 0 || !current(dev)) Py_RETURN_NONE;
  w4a16_problem probs[W4_MAX_GROUPED];
  for (Py_ssize_t i = 0; i < count; ++i) {
    Item& a = it[i];
    if (!a.out.defined()) {
      std::vector<int64_t> sizes(a.x.sizes().begin(), a.x.sizes().end());
      sizes.back() = a.N;
      a.out = empty(sizes, a.x.scalar_type(), dev);
    }
    probs[i] = w4a16_problem{a.x.const_data_ptr(),
                             static_cast<const int32_t*>(a.q.const_data_ptr()),
                             static_cast<const uint16_t*>(a.s.const_data_ptr()),
                             static_cast<const uint16_t*>(a.z.const_data_ptr()),
                             a.out.mutable_data_ptr(),
                             a.N,
                             a.K,
                             (int32_t)a.G,
                             0};
  }
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, api.grouped_workspace_bytes(probs, (int)count, M), &ws, &ws_bytes)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.gemm_grouped(probs, (int)count, dt, M, ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4a16_gemm_grouped")) return nullptr;
  PyObject* list = PyList_New(count);
  if (!list) return nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) PyList_SET_ITEM(list, i, THPVariable_Wrap(std::move(it[i].out)));
  return list;
  END_HANDLE_TH_ERRORS
}

struct Quant {
  const at::Tensor* w;
  int64_t N, K, G;
  at::Tensor q, s, z;
};

// A weight that quantize_int4 accepts, as it is (any strides).
bool quant_item(PyObject* o, int64_t group, Quant* a) {
  a->w = plain(o);
  if (!a->w || a->w->dim() != 2 || a->w->numel() == 0 || act_code(a->w->scalar_type()) < 0) return false;
  a->N = a->w->size(0);
  a->K = a->w->size(1);
  a->G = group == -1 ? a->K : group;
  return a->G > 0 && a->K % a->G == 0 && a->G % 8 == 0 && (a->G & (a->G - 1)) == 0;
}

void quant_outputs(Quant* a) {
  const c10::Device dev = a->w->device();
  a->q = empty({a->K / 8, a->N}, at::kInt, dev);
  a->s = empty({a->K / a->G, a->N}, at::kHalf, dev);
  a->z = empty({a->K / a->G, a->N}, at::kHalf, dev);
}

PyObject* quant_triple(Quant* a) {
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(a->q)), THPVariable_Wrap(std::move(a->s)),
                       THPVariable_Wrap(std::move(a->z)));
}

// The group size an int names, or 0 (never valid) if it is no int or does not fit 32 bits.
int64_t group_arg(PyObject* o) {
  if (!PyLong_CheckExact(o)) return 0;
  int overflow = 0;
  const long long g = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow || g < -1 || g > INT32_MAX ? 0 : g;
}

PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !quiet()) Py_RETURN_NONE;
  Quant a;
  if (!quant_item(args[0], group_arg(args[1]), &a) || !current(a.w->device())) Py_RETURN_NONE;
  if (a.G > INT32_MAX) Py_RETURN_NONE;
  quant_outputs(&a);
  void* const stream = c10::hip::getCurrentHIPStream(a.w->device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.quantize(a.w->const_data_ptr(), act_code(a.w->scalar_type()), a.N, a.K, a.w->stride(0), a.w->stride(1),
                    (int)a.G, static_cast<int32_t*>(a.q.mutable_data_ptr()),
                    static_cast<uint16_t*>(a.s.mutable_data_ptr()), static_cast<uint16_t*>(a.z.mutable_data_ptr()),
                    stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_quantize")) return nullptr;
  return quant_triple(&a);
  END_HANDLE_TH_ERRORS
}

PyObject* quantize_grouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !quiet() || !PyList_CheckExact(args[0])) Py_RETURN_NONE;
  const int64_t group = group_arg(args[1]);
  const Py_ssize_t count = PyList_GET_SIZE(args[0]);
  if (count < 1 || count > W4_MAX_GROUPED) Py_RETURN_NONE;
  std::array<Quant, W4_MAX_GROUPED> it;
  for (Py_ssize_t i = 0; i < count; ++i)
    if (!quant_item(PyList_GET_ITEM(args[0], i), group, &it[i]) || it[i].G > INT32_MAX ||
        it[i].w->scalar_type() != it[0].w->scalar_type() || it[i].w->device() != it[0].w->device())
      Py_RETURN_NONE;
  const c10::Device dev = it[0].w->device();
  if (!current(dev)) Py_RETURN_NONE;
  w4_quantize_problem probs[W4_MAX_GROUPED];
  for (Py_ssize_t i = 0; i < count; ++i) {
    Quant& a = it[i];
    quant_outputs(&a);
    probs[i] = w4_quantize_problem{a.w->const_data_ptr(),
                                   static_cast<int32_t*>(a.q.mutable_data_ptr()),
                                   static_cast<uint16_t*>(a.s.mutable_data_ptr()),
                                   static_cast<uint16_t*>(a.z.mutable_data_ptr()),
                                   a.N,
                                   a.K,
                                   a.w->stride(0),
                                   a.w->stride(1),
                                   (int32_t)group,
                                   0};
  }
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.quantize_grouped(probs, (int)count, act_code(it[0].w->scalar_type()), stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_quantize_grouped")) return nullptr;
  PyObject* list = PyList_New(count);
  if (!list) return nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* t = quant_triple(&it[i]);
    if (!t) {
      Py_DECREF(list);
      return nullptr;
    }
    PyList_SET_ITEM(list, i, t);
  }
  return list;
  END_HANDLE_TH_ERRORS
}

PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !quiet() || !THPDtype_Check(args[3])) Py_RETURN_NONE;
  const at::Tensor *q = plain(args[0]), *s = plain(args[1]), *z = plain(args[2]);
  const at::ScalarType dtype = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
  const int dt = dtype == at::kFloat ? W4_DTYPE_FP32 : act_code(dtype);
  if (!q || dt < 0 || q->dim() != 2 || !current(q->device())) Py_RETURN_NONE;
  const int64_t K = q->size(0) * 8, N = q->size(1), G = weight_group(q, s, z, q->device(), K);
  if (G == 0 || G > INT32_MAX || N == 0) Py_RETURN_NONE;
  at::Tensor out = empty({N, K}, dtype, q->device());
  void* const stream = c10::hip::getCurrentHIPStream(q->device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.dequantize(static_cast<const int32_t*>(q->const_data_ptr()),
                      static_cast<const uint16_t*>(s->const_data_ptr()),
                      static_cast<const uint16_t*>(z->const_data_ptr()), N, K, (int)G, dt, out.mutable_data_ptr(),
                      stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_dequantize")) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- paged cache and log probabilities
// Each takes the arguments of the Python function of its name, all of them by position.

// A derivative is asked for: gradients are recorded, or the tensor holds a tangent.
bool tracked(const at::Tensor* t) {
  return (t->requires_grad() && c10::GradMode::is_enabled()) || t->_fw_grad(/*level=*/0).defined();
}

// The cache of plain, dense tensors; false: not plain.
struct Cache {
  const at::Tensor *k, *v, *weight, *table;
  w4_paged_cache c;
};
bool cache_of(PyObject* k, PyObject* v, PyObject* table, PyObject* weight, Cache* out) {
  out->k = plain(k);
  out->v = plain(v);
  out->table = plain(table);
  out->weight = nullptr;
  if (!out->k || !out->v || !out->table) return false;
  if (weight != Py_None && !(out->weight = plain(weight))) return false;
  const at::Tensor &kt = *out->k, &vt = *out->v, &tt = *out->table;
  const c10::Device dev = kt.device();
  if (act_code(kt.scalar_type()) < 0 || kt.dim() != 4 || vt.scalar_type() != kt.scalar_type() ||
      vt.sizes() != kt.sizes() || vt.device() != dev || !kt.is_contiguous() || !vt.is_contiguous() || tracked(&kt) ||
      tracked(&vt))
    return false;
  if (tt.scalar_type() != at::kInt || tt.dim() != 2 || tt.device() != dev || !tt.is_contiguous() || tt.size(1) < 1)
    return false;
  if (out->weight) {
    const at::Tensor& w = *out->weight;
    if (w.scalar_type() != at::kFloat || w.dim() != 3 || w.sizes() != kt.sizes().slice(0, 3) || w.device() != dev ||
        !w.is_contiguous() || tracked(&w))
      return false;
  }
  out->c = w4_paged_cache{kt.mutable_data_ptr(),
                          vt.mutable_data_ptr(),
                          out->weight ? static_cast<float*>(out->weight->mutable_data_ptr()) : nullptr,
                          static_cast<const int32_t*>(tt.const_data_ptr()),
                          kt.size(0),
                          kt.size(1),
                          kt.size(2),
                          kt.size(3),
                          tt.size(0),
                          tt.size(1)};
  const int64_t d = out->c.head_dim, S = out->c.page_size;
  return (d == 64 || d == 128) && S >= 8 && S <= 1024 && (S & (S - 1)) == 0 && current(dev);
}

// [n, width] like the cache, rows dense and 16-byte aligned.
bool rows_fit(const at::Tensor* t, int64_t n, int64_t width, const at::Tensor& like) {
  return t && t->dim() == 2 && t->size(0) == n && t->size(1) == width && t->scalar_type() == like.scalar_type() &&
         t->device() == like.device() && t->stride(1) == 1 && t->stride(0) % 8 == 0 &&
         (uintptr_t)t->const_data_ptr() % 16 == 0 && !tracked(t);
}

bool index_fit(const at::Tensor* t, int64_t n, c10::Device dev) {
  return t && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->device() == dev &&
         t->is_contiguous();
}

bool angles_fit(const at::Tensor* cos, const at::Tensor* sin, int64_t d, c10::Device dev) {
  for (const at::Tensor* t : {cos, sin})
    if (!t || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) != d / 2 || t->size(0) < 1 ||
        t->device() != dev || !t->is_contiguous() || (uintptr_t)t->const_data_ptr() % 16 != 0 || tracked(t))
      return false;
  return cos->size(0) == sin->size(0);
}

const int32_t* ints(const at::Tensor* t) { return static_cast<const int32_t*>(t->const_data_ptr()); }
const float* floats(const at::Tensor* t) { return static_cast<const float*>(t->const_data_ptr()); }

// (k, v, cos, sin, k_pages, v_pages, table, rows, slots, positions, weight) -> True
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache p;
  if (n != 11 || !api.paged_append || !quiet() || !cache_of(args[4], args[5], args[6], args[10], &p)) Py_RETURN_NONE;
  const at::Tensor *k = plain(args[0]), *v = plain(args[1]), *cos = plain(args[2]), *sin = plain(args[3]);
  const at::Tensor *rows = plain(args[7]), *slots = plain(args[8]), *positions = plain(args[9]);
  if (!k || k->dim() != 2) Py_RETURN_NONE;
  const int64_t T = k->size(0), width = p.c.kv_heads * p.c.head_dim;
  const c10::Device dev = p.k->device();
  if (!rows_fit(k, T, width, *p.k) || !rows_fit(v, T, width, *p.k) || !angles_fit(cos, sin, p.c.head_dim, dev) ||
      !index_fit(rows, T, dev) || !index_fit(slots, T, dev) || !index_fit(positions, T, dev))
    Py_RETURN_NONE;
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged_append(&p.c, act_code(p.k->scalar_type()), k->const_data_ptr(), v->const_data_ptr(), k->stride(0),
                        v->stride(0), T, ints(rows), ints(slots), ints(positions), floats(cos), floats(sin),
                        cos->size(0), stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged_append")) return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (q, k, v, cos, sin, k_pages, v_pages, table, lengths, positions, weight) -> out
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache p;
  if (n != 11 || !api.paged_attention || !quiet() || !cache_of(args[5], args[6], args[7], args[10], &p)) Py_RETURN_NONE;
  const at::Tensor *q = plain(args[0]), *k = plain(args[1]), *v = plain(args[2]), *cos = plain(args[3]),
                   *sin = plain(args[4]), *lengths = plain(args[8]), *positions = plain(args[9]);
  if (!q || q->dim() != 2) Py_RETURN_NONE;
  const int64_t B = p.c.rows, d = p.c.head_dim, width = p.c.kv_heads * d;
  const c10::Device dev = p.k->device();
  if (q->size(1) < 1 || q->size(1) % width != 0 || !rows_fit(q, B, q->size(1), *p.k) ||
      !rows_fit(k, B, width, *p.k) || !rows_fit(v, B, width, *p.k) || !angles_fit(cos, sin, d, dev) ||
      !index_fit(lengths, B, dev) || !index_fit(positions, B, dev) || B < 1)
    Py_RETURN_NONE;
  const int64_t heads = q->size(1) / d;
  at::Tensor out = empty({B, q->size(1)}, p.k->scalar_type(), dev), scores;
  if (p.weight) scores = empty({B * heads * p.c.width * p.c.page_size}, at::kFloat, dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, api.paged_attention_workspace_bytes(B, heads, p.c.kv_heads, d), &ws, &ws_bytes))
    return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged_attention(&p.c, act_code(p.k->scalar_type()), q->const_data_ptr(), k->const_data_ptr(),
                           v->const_data_ptr(), q->stride(0), k->stride(0), v->stride(0), heads, ints(lengths),
                           ints(positions), floats(cos), floats(sin), cos->size(0), out.mutable_data_ptr(),
                           scores.defined() ? static_cast<float*>(scores.mutable_data_ptr()) : nullptr, ws, ws_bytes,
                           stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged_attention")) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A Python int that fits; else -1.
int64_t count_arg(PyObject* o) {
  if (!PyLong_CheckExact(o)) return -1;
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow || v < 0 ? -1 : v;
}

// (k_pages, v_pages, weight, table, lengths, new_table, keep, recent) -> new lengths
PyObject* paged_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache p;
  if (n != 8 || !api.paged_evict || !quiet() || args[2] == Py_None ||
      !cache_of(args[0], args[1], args[3], args[2], &p))
    Py_RETURN_NONE;
  const at::Tensor *lengths = plain(args[4]), *to = plain(args[5]);
  const int64_t keep = count_arg(args[6]), recent = count_arg(args[7]), B = p.c.rows;
  const c10::Device dev = p.k->device();
  if (!index_fit(lengths, B, dev) || !to || to->scalar_type() != at::kInt || to->dim() != 2 || to->size(0) != B ||
      to->device() != dev || !to->is_contiguous() || keep < 1 || recent < 0 || recent > keep || B < 1 ||
      keep > to->size(1) * p.c.page_size)
    Py_RETURN_NONE;
  at::Tensor lens = empty({B}, at::kInt, dev),
             scratch = empty({(int64_t)api.paged_evict_scratch_words(&p.c, keep)}, at::kInt, dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged_evict(&p.c, act_code(p.k->scalar_type()), ints(lengths), ints(to), to->size(1), keep, recent,
                       static_cast<int32_t*>(scratch.mutable_data_ptr()),
                       static_cast<int32_t*>(lens.mutable_data_ptr()), stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged_evict")) return nullptr;
  return THPVariable_Wrap(std::move(lens));
  END_HANDLE_TH_ERRORS
}

// (logits, tokens or None, top) -> (logprob or None, entropy, top_logprob, top_token)
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !api.token_logprobs || !quiet()) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0]);
  if (!x || x->dim() != 2 || tracked(x)) Py_RETURN_NONE;
  const int dt = x->scalar_type() == at::kFloat ? W4_DTYPE_FP32 : act_code(x->scalar_type());
  const int64_t R = x->size(0), V = x->size(1), top = count_arg(args[2]);
  const c10::Device dev = x->device();
  if (dt < 0 || R < 1 || V < 1 || top < 0 || top > 64 || top > V || x->stride(1) != 1 || x->stride(0) < 0 ||
      !current(dev))
    Py_RETURN_NONE;
  const at::Tensor* tokens = args[1] == Py_None ? nullptr : plain(args[1]);
  if (args[1] != Py_None && (!tokens || tokens->scalar_type() != at::kLong || tokens->dim() != 1 ||
                             tokens->size(0) != R || tokens->device() != dev || !tokens->is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor logprob, entropy = empty({R}, at::kFloat, dev), top_logprob = empty({R, top}, at::kFloat, dev),
             top_token = empty({R, top}, at::kLong, dev);
  if (tokens) logprob = empty({R}, at::kFloat, dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, api.token_logprobs_workspace_bytes(R, V, top), &ws, &ws_bytes)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.token_logprobs(x->const_data_ptr(), dt, R, V, x->stride(0),
                          tokens ? static_cast<const int64_t*>(tokens->const_data_ptr()) : nullptr, top,
                          logprob.defined() ? static_cast<float*>(logprob.mutable_data_ptr()) : nullptr,
                          static_cast<float*>(entropy.mutable_data_ptr()),
                          static_cast<float*>(top_logprob.mutable_data_ptr()),
                          static_cast<int64_t*>(top_token.mutable_data_ptr()), ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_token_logprobs")) return nullptr;
  PyObject* first = Py_None;
  if (logprob.defined()) first = THPVariable_Wrap(std::move(logprob));
  else Py_INCREF(first);
  return Py_BuildValue("(NNNN)", first, THPVariable_Wrap(std::move(entropy)), THPVariable_Wrap(std::move(top_logprob)),
                       THPVariable_Wrap(std::move(top_token)));
  END_HANDLE_TH_ERRORS
}

// The 8-bit cache of plain, dense tensors (k_pages, v_pages, k_scale, v_scale, table); false: not plain.
bool cache8_of(PyObject* const* o, w4_paged8_cache* c) {
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i) {
    t[i] = plain(o[i]);
    if (!t[i] || t[i]->device() != t[0]->device() || !t[i]->is_contiguous() || tracked(t[i])) return false;
  }
  const at::Tensor &k = *t[0], &ks = *t[2], &table = *t[4];
  const at::ScalarType type = k.scalar_type();
  if ((type != at::kChar && type != at::kFloat8_e4m3fn) || k.dim() != 4 || t[1]->scalar_type() != type ||
      t[1]->sizes() != k.sizes() || ks.scalar_type() != at::kFloat || t[3]->scalar_type() != at::kFloat ||
      ks.dim() != 3 || t[3]->sizes() != ks.sizes() || ks.size(0) != k.size(0) || ks.size(1) != k.size(1) ||
      ks.size(2) < 1 || table.scalar_type() != at::kInt || table.dim() != 2 || table.size(1) < 1)
    return false;
  const int64_t S = k.size(2), d = k.size(3), block = S / ks.size(2);
  if ((d != 64 && d != 128) || S < 8 || S > 1024 || (S & (S - 1)) != 0 || block * ks.size(2) != S || block < 8 ||
      block > 64 || (block & (block - 1)) != 0)
    return false;
  *c = w4_paged8_cache{k.mutable_data_ptr(),
                       t[1]->mutable_data_ptr(),
                       static_cast<float*>(ks.mutable_data_ptr()),
                       static_cast<float*>(t[3]->mutable_data_ptr()),
                       ints(&table),
                       k.size(0),
                       k.size(1),
                       S,
                       d,
                       block,
                       table.size(0),
                       table.size(1),
                       type == at::kChar ? W4_CODE_INT8 : W4_CODE_E4M3,
                       0};
  return current(k.device());
}

// The operands of new tokens (k, v, cos, sin) and (lengths, offsets, positions); false: not plain, or not fitting.
bool new_fit(const at::Tensor* const kv[4], const at::Tensor* const at3[3], const w4_paged8_cache& c, c10::Device dev) {
  const at::Tensor* k = kv[0];
  if (!k || k->dim() != 2 || act_code(k->scalar_type()) < 0 || k->device() != dev) return false;
  const int64_t T = k->size(0), width = c.kv_heads * c.head_dim;
  return rows_fit(k, T, width, *k) && rows_fit(kv[1], T, width, *k) && angles_fit(kv[2], kv[3], c.head_dim, dev) &&
         index_fit(at3[0], c.rows, dev) && index_fit(at3[1], c.rows + 1, dev) && index_fit(at3[2], T, dev);
}

// (k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions) -> True
PyObject* paged_append8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  w4_paged8_cache c;
  if (n != 12 || !api.paged8_append || !quiet() || !cache8_of(args + 4, &c)) Py_RETURN_NONE;
  const c10::Device dev = THPVariable_Unpack(args[4]).device();
  const at::Tensor* const kv[4] = {plain(args[0]), plain(args[1]), plain(args[2]), plain(args[3])};
  const at::Tensor* const at3[3] = {plain(args[9]), plain(args[10]), plain(args[11])};
  if (!new_fit(kv, at3, c, dev)) Py_RETURN_NONE;
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged8_append(&c, act_code(kv[0]->scalar_type()), kv[0]->const_data_ptr(), kv[1]->const_data_ptr(),
                         kv[0]->stride(0), kv[1]->stride(0), kv[0]->size(0), ints(at3[0]), ints(at3[1]), ints(at3[2]),
                         floats(kv[2]), floats(kv[3]), kv[2]->size(0), stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged8_append")) return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (k_pages, v_pages, k_scale, v_scale, table, starts, offsets, tokens, dtype) -> (k, v)
PyObject* paged_read8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  w4_paged8_cache c;
  if (n != 9 || !api.paged8_read || !quiet() || !THPDtype_Check(args[8]) || !cache8_of(args, &c)) Py_RETURN_NONE;
  const c10::Device dev = THPVariable_Unpack(args[0]).device();
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[8])->scalar_type;
  const int dt = type == at::kFloat ? W4_DTYPE_FP32 : act_code(type);
  const int64_t T = count_arg(args[7]);
  const at::Tensor *starts = plain(args[5]), *offsets = plain(args[6]);
  if (dt < 0 || T < 0 || T > (1 << 24) || !index_fit(starts, c.rows, dev) || !index_fit(offsets, c.rows + 1, dev))
    Py_RETURN_NONE;
  at::Tensor k = empty({T, c.kv_heads * c.head_dim}, type, dev), v = empty({T, c.kv_heads * c.head_dim}, type, dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged8_read(&c, dt, ints(starts), ints(offsets), T, k.mutable_data_ptr(), v.mutable_data_ptr(), stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged8_read")) return nullptr;
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions, longest or None,
// window or None, sinks) -> out
PyObject* paged_attention8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  w4_paged8_cache c;
  if (n != 16 || !api.paged8_attention || !quiet() || !cache8_of(args + 5, &c)) Py_RETURN_NONE;
  const c10::Device dev = THPVariable_Unpack(args[5]).device();
  const at::Tensor* q = plain(args[0]);
  const at::Tensor* const kv[4] = {plain(args[1]), plain(args[2]), plain(args[3]), plain(args[4])};
  const at::Tensor* const at3[3] = {plain(args[10]), plain(args[11]), plain(args[12])};
  const int64_t longest = args[13] == Py_None ? 0 : count_arg(args[13]);
  const int64_t window = args[14] == Py_None ? 0 : count_arg(args[14]), sinks = count_arg(args[15]);
  if (!q || q->dim() != 2 || longest < 0 || sinks < 0 || window < (args[14] == Py_None ? 0 : 1) || !new_fit(kv, at3, c, dev))
    Py_RETURN_NONE;
  const at::Tensor& k = *kv[0];
  const int64_t T = k.size(0), width = c.kv_heads * c.head_dim;
  if (T < 1 || T > (1 << 24) || q->size(1) < 1 || q->size(1) % width != 0 || !rows_fit(q, T, q->size(1), k))
    Py_RETURN_NONE;
  const int64_t heads = q->size(1) / c.head_dim;
  at::Tensor out = empty({T, q->size(1)}, k.scalar_type(), dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, api.paged8_attention_workspace_bytes(c.rows, T, heads, c.kv_heads, c.head_dim), &ws, &ws_bytes))
    return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.paged8_attention(&c, act_code(k.scalar_type()), q->const_data_ptr(), k.const_data_ptr(),
                            kv[1]->const_data_ptr(), q->stride(0), k.stride(0), kv[1]->stride(0), heads, T, longest,
                            window, sinks, ints(at3[0]), ints(at3[1]), ints(at3[2]), floats(kv[2]), floats(kv[3]),
                            kv[2]->size(0), out.mutable_data_ptr(), ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_paged8_attention")) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (target, draft or None, tokens, accept, sample, counts or None) -> (accepted, token)
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !api.verify_drafts || !quiet()) Py_RETURN_NONE;
  const at::Tensor* p = plain(args[0]);
  if (!p || p->dim() != 3 || tracked(p)) Py_RETURN_NONE;
  const int dt = p->scalar_type() == at::kFloat ? W4_DTYPE_FP32 : act_code(p->scalar_type());
  const int64_t B = p->size(0), K = p->size(1) - 1, V = p->size(2);
  const c10::Device dev = p->device();
  if (dt < 0 || B < 1 || K < 0 || K > 64 || V < 1 || p->stride(2) != 1 || !current(dev)) Py_RETURN_NONE;
  const at::Tensor* d = args[1] == Py_None ? nullptr : plain(args[1]);
  if (args[1] != Py_None && (!d || d->dim() != 3 || d->scalar_type() != p->scalar_type() || d->size(0) != B ||
                             d->size(1) != K || d->size(2) != V || d->device() != dev || d->stride(2) != 1 || tracked(d)))
    Py_RETURN_NONE;
  const at::Tensor *x = plain(args[2]), *u = plain(args[3]), *r = plain(args[4]);
  const at::Tensor* counts = args[5] == Py_None ? nullptr : plain(args[5]);
  auto grid = [&](const at::Tensor* t, at::ScalarType type) {
    return t && t->scalar_type() == type && t->dim() == 2 && t->size(0) == B && t->size(1) == K && t->device() == dev &&
           t->is_contiguous() && !tracked(t);
  };
  if (!grid(x, at::kLong) || !grid(u, at::kFloat) || !r || r->scalar_type() != at::kFloat || r->dim() != 1 ||
      r->size(0) != B || r->device() != dev || !r->is_contiguous() || tracked(r) ||
      (args[5] != Py_None && !index_fit(counts, B, dev)))
    Py_RETURN_NONE;
  at::Tensor accepted = empty({B}, at::kLong, dev), token = empty({B}, at::kLong, dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  void* ws;
  size_t ws_bytes;
  if (!workspace(dev, stream, api.verify_drafts_workspace_bytes(B, V), &ws, &ws_bytes)) return nullptr;
  if (K == 0) d = nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.verify_drafts(p->const_data_ptr(), d ? d->const_data_ptr() : nullptr, dt, B, K, V, p->stride(0), p->stride(1),
                         d ? d->stride(0) : 0, d ? d->stride(1) : 0, static_cast<const int64_t*>(x->const_data_ptr()),
                         counts ? ints(counts) : nullptr, floats(u), floats(r),
                         static_cast<int64_t*>(accepted.mutable_data_ptr()),
                         static_cast<int64_t*>(token.mutable_data_ptr()), ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (!check(rc, "w4_verify_drafts")) return nullptr;
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(accepted)), THPVariable_Wrap(std::move(token)));
  END_HANDLE_TH_ERRORS
}

// (addresses of the 8-bit cache's and the verification's C-ABI functions in Api's order)
PyObject* init_paged8(PyObject*, PyObject* args) {
  unsigned long long p[6];
  if (!PyArg_ParseTuple(args, "(KKKKKK)", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5])) return nullptr;
  api.paged8_append = reinterpret_cast<decltype(api.paged8_append)>(p[0]);
  api.paged8_read = reinterpret_cast<decltype(api.paged8_read)>(p[1]);
  api.paged8_attention_workspace_bytes = reinterpret_cast<decltype(api.paged8_attention_workspace_bytes)>(p[2]);
  api.paged8_attention = reinterpret_cast<decltype(api.paged8_attention)>(p[3]);
  api.verify_drafts_workspace_bytes = reinterpret_cast<decltype(api.verify_drafts_workspace_bytes)>(p[4]);
  api.verify_drafts = reinterpret_cast<decltype(api.verify_drafts)>(p[5]);
  Py_RETURN_NONE;
}

// (addresses of the paged cache's and the log probabilities' C-ABI functions in Api's order)
PyObject* init_paged(PyObject*, PyObject* args) {
  unsigned long long p[7];
  if (!PyArg_ParseTuple(args, "(KKKKKKK)", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6])) return nullptr;
  api.paged_append = reinterpret_cast<decltype(api.paged_append)>(p[0]);
  api.paged_attention_workspace_bytes = reinterpret_cast<decltype(api.paged_attention_workspace_bytes)>(p[1]);
  api.paged_attention = reinterpret_cast<decltype(api.paged_attention)>(p[2]);
  api.paged_evict_scratch_words = reinterpret_cast<decltype(api.paged_evict_scratch_words)>(p[3]);
  api.paged_evict = reinterpret_cast<decltype(api.paged_evict)>(p[4]);
  api.token_logprobs_workspace_bytes = reinterpret_cast<decltype(api.token_logprobs_workspace_bytes)>(p[5]);
  api.token_logprobs = reinterpret_cast<decltype(api.token_logprobs)>(p[6]);
  Py_RETURN_NONE;
}

// (addresses of the C-ABI functions in Api's order, workspace, check)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long p[7];
  PyObject *w, *c;
  if (!PyArg_ParseTuple(args, "(KKKKKKK)OO", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &w, &c)) return nullptr;
  Py_INCREF(w);
  Py_INCREF(c);
  Py_XDECREF(py_workspace);
  Py_XDECREF(py_check);
  py_workspace = w;
  py_check = c;
  api.workspace_bytes = reinterpret_cast<decltype(api.workspace_bytes)>(p[1]);
  api.gemm_grouped = reinterpret_cast<decltype(api.gemm_grouped)>(p[2]);
  api.grouped_workspace_bytes = reinterpret_cast<decltype(api.grouped_workspace_bytes)>(p[3]);
  api.quantize_grouped = reinterpret_cast<decltype(api.quantize_grouped)>(p[4]);
  api.quantize = reinterpret_cast<decltype(api.quantize)>(p[5]);
  api.dequantize = reinterpret_cast<decltype(api.dequantize)>(p[6]);
  api.gemm = reinterpret_cast<decltype(api.gemm)>(p[0]);
  Py_RETURN_NONE;
}

#define W4_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr},
                         {"init_paged", init_paged, METH_VARARGS, nullptr},
                         W4_FAST(paged_append),
                         W4_FAST(paged_attention),
                         W4_FAST(paged_evict),
                         W4_FAST(token_logprobs),
                         {"init_paged8", init_paged8, METH_VARARGS, nullptr},
                         W4_FAST(paged_append8),
                         W4_FAST(paged_read8),
                         W4_FAST(paged_attention8),
                         W4_FAST(verify_drafts),
                         W4_FAST(matmul),
                         W4_FAST(matmul_grouped),
                         W4_FAST(quantize),
                         W4_FAST(quantize_grouped),
                         W4_FAST(dequantize),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_int4_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__int4_torch() {
  PyObject* m = PyModule_Create(&module);
  // the torch whose headers this was built from: tensors are read through them
  if (m && PyModule_AddStringConstant(m, "torch_version", W4_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
