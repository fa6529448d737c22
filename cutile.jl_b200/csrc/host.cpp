// Native call path of the Python package: one C function per entry point takes the tensors as they are, checks the
// ordinary form of the call (CUDA tensors of the expected types and shapes, no launch keywords) and enqueues it through
// the C ABI.
//
// What bounds the small calls is the host: in Python a softmax of 64 x 1000 elements spent about 9 us on reading
// shapes, strides, pointers and the current stream (torch.cuda.current_stream 1.2 us, a shape or stride 0.1-0.3 us) and
// on the ctypes conversion of 11 arguments (1.2 us), against 2.4-3.1 us for the launch itself.  The same through this
// file takes about 0.3 us on top of the launch.
//
// Every function returns None when a call is not of the ordinary form; the Python wrapper then runs its full argument
// checks, which either raise the precise error or make the call themselves.  A status other than CTB_OK raises CtbError
// (through the Python function installed by setup()).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/cutile_b200.h"

namespace {

constexpr int kMaxDevices = 64;
ctb_ctx* g_ctx[kMaxDevices] = {};  // written under the GIL
PyObject* g_context = nullptr;     // _lib.context(device) -> c_void_p
PyObject* g_check = nullptr;       // _lib.check(status): raises CtbError

using at::Tensor;

const Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

struct Call {  // device, context and current stream of a call; ok() is false with a Python error set
  ctb_ctx* ctx = nullptr;
  void* stream = nullptr;
  explicit Call(const Tensor& t) {
    const int dev = t.get_device();
    if (dev < 0 || dev >= kMaxDevices) return;
    if (!g_ctx[dev]) {
      PyObject* h = PyObject_CallFunction(g_context, "i", dev);
      PyObject* v = h ? PyObject_GetAttrString(h, "value") : nullptr;
      if (v) g_ctx[dev] = static_cast<ctb_ctx*>(PyLong_AsVoidPtr(v));
      Py_XDECREF(v);
      Py_XDECREF(h);
      if (!g_ctx[dev] && !PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "cutile_b200: no context");
    }
    ctx = g_ctx[dev];
    if (ctx) stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  }
  bool ok() const { return ctx != nullptr; }
};

// Py_None ("not the ordinary form") and the result of a call with status s
PyObject* decline() { Py_RETURN_NONE; }
PyObject* done(int s, PyObject* result_owned) {
  if (s == CTB_OK) return result_owned;
  Py_XDECREF(result_owned);
  PyObject* r = PyObject_CallFunction(g_check, "i", s);  // raises
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "cutile_b200: call failed");
  return nullptr;
}
PyObject* yes() { Py_RETURN_TRUE; }

template <class F>
int without_gil(F f) {
  struct Release {  // the lock is taken again also when f throws: data_ptr() does for a tensor without storage (vmap, fake)
    PyThreadState* state = PyEval_SaveThread();
    ~Release() { PyEval_RestoreThread(state); }
  } release;
  return f();
}

bool as_int(PyObject* o, long long* v) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0 && *v >= INT32_MIN && *v <= INT32_MAX;
}
bool ints(PyObject* const* a, int n, long long* v) {
  for (int i = 0; i < n; ++i)
    if (!as_int(a[i], v + i)) return false;
  return true;
}
bool as_float(PyObject* o, float* v) {
  if (!PyFloat_Check(o)) return false;
  *v = (float)PyFloat_AS_DOUBLE(o);
  return true;
}
int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CTB_F32;
    case at::kHalf: return CTB_F16;
    case at::kBFloat16: return CTB_BF16;
    default: return -1;
  }
}
// 2-D with contiguous rows -> leading dimension
bool rows(const Tensor& t, int64_t* ld, int64_t* m, int64_t* n) {
  if (t.dim() != 2) return false;
  *m = t.size(0);
  *n = t.size(1);
  if (*n > 1 && t.stride(1) != 1) return false;
  *ld = *m > 1 ? t.stride(0) : std::max<int64_t>(*n, t.stride(0));
  return true;
}
bool vec_f32(const Tensor* t, int64_t n) { return t && t->scalar_type() == at::kFloat && t->numel() == n && t->is_contiguous(); }

// softmax(output, input, variant, tile)
PyObject* softmax(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor *out, *in;
  long long v[2];
  int64_t ldo, mo, no, ldi, m, k;
  if (n != 4 || !(out = cuda_tensor(a[0])) || !(in = cuda_tensor(a[1])) || !ints(a + 2, 2, v) || !rows(*out, &ldo, &mo, &no) ||
      !rows(*in, &ldi, &m, &k) || mo != m || no != k || out->scalar_type() != in->scalar_type() || dtype_of(*in) < 0)
    return decline();
  Call c(*in);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_softmax(c.ctx, c.stream, out->data_ptr(), in->data_ptr(), k, m, ldo, ldi, (int)v[0], (int)v[1], dtype_of(*in));
  });
  return done(s, yes());
}

// vadd(a, b, c, tile_x, tile_y, gather, dims): dims = 1: dense 1-D arrays; 2: 2-D arrays with contiguous rows
PyObject* vadd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[3];
  long long v[4];
  if (n != 7 || !ints(a + 3, 4, v)) return decline();
  int64_t ld[3], m = 1, k = 0;
  for (int i = 0; i < 3; ++i) {
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->scalar_type() != t[0]->scalar_type() || t[i]->sizes() != t[0]->sizes() ||
        t[i]->dim() != v[3])
      return decline();
    if (v[3] == 1) {
      if (!t[i]->is_contiguous()) return decline();
      k = ld[i] = t[i]->numel();
    } else if (!rows(*t[i], ld + i, &m, &k)) {
      return decline();
    }
  }
  const int dt = dtype_of(*t[0]);
  if (dt < 0) return decline();
  Call c(*t[0]);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_vadd(c.ctx, c.stream, t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), k, m, ld[0], ld[1], ld[2], (int)v[0],
                    (int)v[1], (int)v[2], dt);
  });
  return done(s, yes());
}

// transpose(x, y, tm, tn)
PyObject* transpose(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor *x, *y;
  long long v[2];
  int64_t ldx, N, M, ldy, My, Ny;
  if (n != 4 || !(x = cuda_tensor(a[0])) || !(y = cuda_tensor(a[1])) || !ints(a + 2, 2, v) || !rows(*x, &ldx, &N, &M) ||
      !rows(*y, &ldy, &My, &Ny) || My != M || Ny != N || x->scalar_type() != y->scalar_type() || dtype_of(*x) < 0)
    return decline();
  Call c(*x);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_transpose(c.ctx, c.stream, x->data_ptr(), y->data_ptr(), M, N, ldx, ldy, (int)v[0], (int)v[1], dtype_of(*x));
  });
  return done(s, yes());
}

// layernorm_fwd(X, W, B, Y, Mean, Rstd, eps, tile)
PyObject* layernorm_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[6];
  if (n != 8) return decline();
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = cuda_tensor(a[i]))) return decline();
  int64_t ldx, M, N, ldy, My, Ny;
  float eps;
  long long tile;
  if (t[0]->scalar_type() != at::kFloat || t[3]->scalar_type() != at::kFloat || !rows(*t[0], &ldx, &M, &N) ||
      !rows(*t[3], &ldy, &My, &Ny) || My != M || Ny != N || !vec_f32(t[1], N) || !vec_f32(t[2], N) || !vec_f32(t[4], M) ||
      !vec_f32(t[5], M) || !as_float(a[6], &eps) || !as_int(a[7], &tile))
    return decline();
  Call c(*t[0]);
  if (!c.ok()) return nullptr;
  auto p = [&](int i) { return static_cast<float*>(t[i]->data_ptr()); };
  const int s = without_gil([&] {
    return ctb_layernorm_fwd(c.ctx, c.stream, p(0), p(1), p(2), p(3), p(4), p(5), N, M, ldx, ldy, eps, (int)tile);
  });
  return done(s, yes());
}

// layernorm_bwd(DX, DY, DW, DB, X, W, Mean, Rstd, group_size_m, tile)
PyObject* layernorm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[8];
  if (n != 10) return decline();
  for (int i = 0; i < 8; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->scalar_type() != at::kFloat) return decline();
  int64_t ld[3], M, N, m, k;
  long long v[2];
  if (!ints(a + 8, 2, v) || !rows(*t[4], ld, &M, &N) || !rows(*t[1], ld + 1, &m, &k) || m != M || k != N ||
      !rows(*t[0], ld + 2, &m, &k) || m != M || k != N || !vec_f32(t[5], N) || !vec_f32(t[6], M) || !vec_f32(t[7], M))
    return decline();
  for (int i = 2; i < 4; ++i)
    if (t[i]->dim() != 2 || t[i]->size(0) != v[0] || t[i]->size(1) != N || !t[i]->is_contiguous()) return decline();
  Call c(*t[4]);
  if (!c.ok()) return nullptr;
  auto p = [&](int i) { return static_cast<float*>(t[i]->data_ptr()); };
  const int s = without_gil([&] {
    return ctb_layernorm_bwd_dx_partial_dwdb(c.ctx, c.stream, p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), nullptr, N, M,
                                             ld[0], ld[1], ld[2], (int)v[0], (int)v[1]);
  });
  return done(s, yes());
}

// layernorm_dwdb(DW, DB, FINAL_DW, FINAL_DB, tile_m, tile_n)
PyObject* layernorm_dwdb(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[4];
  long long v[2];
  if (n != 6 || !ints(a + 4, 2, v)) return decline();
  for (int i = 0; i < 4; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->scalar_type() != at::kFloat || !t[i]->is_contiguous()) return decline();
  if (t[0]->dim() != 2 || t[1]->sizes() != t[0]->sizes()) return decline();
  const int64_t G = t[0]->size(0), N = t[0]->size(1);
  if (t[2]->numel() != N || t[3]->numel() != N) return decline();
  Call c(*t[0]);
  if (!c.ok()) return nullptr;
  auto p = [&](int i) { return static_cast<float*>(t[i]->data_ptr()); };
  const int s = without_gil([&] {
    return ctb_layernorm_bwd_dwdb(c.ctx, c.stream, p(0), p(1), p(2), p(3), N, (int)G, (int)v[0], (int)v[1]);
  });
  return done(s, yes());
}

// matmul(A, B, C, tm, tn, tk): A [K, M], B [N, K], C [N, M]
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[3];
  long long v[3];
  if (n != 6 || !ints(a + 3, 3, v)) return decline();
  int64_t ld[3], d0[3], d1[3];
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->scalar_type() != t[0]->scalar_type() || !rows(*t[i], ld + i, d0 + i, d1 + i))
      return decline();
  const int dt = dtype_of(*t[0]);
  const int64_t K = d0[0], M = d1[0], N = d0[1];
  if (dt < 0 || d1[1] != K || d0[2] != N || d1[2] != M) return decline();
  Call c(*t[0]);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_gemm(c.ctx, c.stream, t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), M, N, K, ld[0], ld[1], ld[2], dt,
                    (int)v[0], (int)v[1], (int)v[2]);
  });
  return done(s, yes());
}

// batch_matmul(A, B, C, tm, tn, tk): A [batch, K, M], B [batch, N, K], C [batch, N, M]
PyObject* batch_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[3];
  long long v[3];
  if (n != 6 || !ints(a + 3, 3, v)) return decline();
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->scalar_type() != t[0]->scalar_type() || t[i]->dim() != 3 || t[i]->stride(2) != 1)
      return decline();
  const int dt = dtype_of(*t[0]);
  const int64_t nb = t[0]->size(0), K = t[0]->size(1), M = t[0]->size(2), N = t[1]->size(1);
  if (dt < 0 || t[1]->size(0) != nb || t[2]->size(0) != nb || t[1]->size(2) != K || t[2]->size(1) != N || t[2]->size(2) != M)
    return decline();
  Call c(*t[0]);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_gemm_batched(c.ctx, c.stream, t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), M, N, K, nb, t[0]->stride(1),
                            t[1]->stride(1), t[2]->stride(1), t[0]->stride(0), t[1]->stride(0), t[2]->stride(0), dt, (int)v[0],
                            (int)v[1], (int)v[2]);
  });
  return done(s, yes());
}

// fmha(Q, K, V, Out or None, qk_scale or None, input_pos, tile_m, tile_n, group, causal) -> Out
PyObject* fmha(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[3];
  long long v[4];
  if (n != 10 || !ints(a + 5, 4, v) || !PyBool_Check(a[9])) return decline();
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || t[i]->dim() != 4 || !t[i]->is_contiguous() || t[i]->scalar_type() != t[0]->scalar_type())
      return decline();
  const Tensor &Q = *t[0], &K = *t[1], &V = *t[2];
  const int dt = dtype_of(Q);
  const int64_t B = Q.size(0), H = Q.size(1), Sq = Q.size(2), D = Q.size(3), KVH = K.size(1), Skv = K.size(2), Dv = V.size(3);
  if (dt < 0 || K.size(0) != B || K.size(3) != D || V.size(0) != B || V.size(1) != KVH || V.size(2) != Skv || D <= 0)
    return decline();
  float scale;
  if (a[4] == Py_None) scale = (float)(1.0 / std::sqrt((double)D));
  else if (!as_float(a[4], &scale)) return decline();
  const bool causal = a[9] == Py_True;
  Call c(Q);
  if (!c.ok()) return nullptr;
  Tensor made;
  const Tensor* out;
  if (a[3] == Py_None) {
    made = at::empty({B, H, Sq, Dv}, Q.options());
    out = &made;
  } else {
    if (!(out = cuda_tensor(a[3])) || out->scalar_type() != Q.scalar_type() || out->dim() != 4 || !out->is_contiguous() ||
        out->size(0) != B || out->size(1) != H || out->size(2) != Sq || out->size(3) != Dv)
      return decline();
  }
  const int s = without_gil([&] {
    return ctb_fmha_fwd(c.ctx, c.stream, Q.data_ptr(), K.data_ptr(), V.data_ptr(), out->data_ptr(), D, Dv, Sq, Skv, H, KVH, B,
                        scale, (int32_t)v[0], (int)v[1], (int)v[2], (int)v[3], causal ? 1 : 0, dt);
  });
  if (s != CTB_OK || a[3] != Py_None) return done(s, s == CTB_OK ? Py_NewRef(a[3]) : nullptr);
  return THPVariable_Wrap(std::move(made));
}

// Three strides of [batch, seq, heads, D], or of [tokens, heads, D] as one batch.
bool token_strides(const Tensor& t, int64_t* s) {
  const int64_t n = t.dim();
  if ((n != 3 && n != 4) || t.stride(n - 1) != 1) return false;
  s[0] = n == 4 ? t.stride(0) : 0;
  s[1] = t.stride(n - 3);
  s[2] = t.stride(n - 2);
  return true;
}
int index_bits(const Tensor& t) { return t.scalar_type() == at::kInt ? 32 : t.scalar_type() == at::kLong ? 64 : 0; }
bool frequencies_of(const Tensor* f, const Tensor& like) {
  return f && f->scalar_type() == at::kDouble && f->dim() == 1 && f->size(0) > 0 && f->is_contiguous() && f->device() == like.device();
}
// A new array, without the dispatcher: at::empty takes 0.6 us more.
Tensor new_array(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
// at::empty_like's layout: the order of the dimensions in memory stays.
Tensor new_like(const Tensor& x) {
  for (int64_t i = 1; i < x.dim(); ++i)
    if (x.stride(i - 1) < x.stride(i)) return at::empty_like(x);
  return new_array(x.sizes(), x.scalar_type(), x);
}
// A result where one is given, else a new array with the layout of its input.
const Tensor* result_like(PyObject* given, const Tensor& x, Tensor* made) {
  if (given == Py_None) {
    *made = new_like(x);
    return made;
  }
  const Tensor* out = cuda_tensor(given);
  return out && out->device() == x.device() && out->scalar_type() == x.scalar_type() && out->sizes() == x.sizes() ? out : nullptr;
}
PyObject* given_or(PyObject* given, Tensor& made) { return given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(std::move(made)); }

// rope(q, k or None, positions, frequencies, interleaved, scale, out_q or None, out_k or None, inverse) -> (out_q, out_k or None)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return decline();
  const Tensor *q = cuda_tensor(a[0]), *k = a[1] == Py_None ? nullptr : cuda_tensor(a[1]), *pos = cuda_tensor(a[2]), *f = cuda_tensor(a[3]);
  float scale;
  int64_t s[12] = {};
  if (!q || (!k && a[1] != Py_None) || !pos || !PyBool_Check(a[4]) || !as_float(a[5], &scale) || !PyBool_Check(a[8]) || dtype_of(*q) < 0 ||
      !token_strides(*q, s + 3) || !frequencies_of(f, *q) || pos->device() != q->device() || !pos->is_contiguous() || !index_bits(*pos))
    return decline();
  const int64_t d = q->dim();
  if (pos->dim() != d - 2 || pos->sizes() != q->sizes().slice(0, d - 2)) return decline();
  if (k && (k->device() != q->device() || k->scalar_type() != q->scalar_type() || k->dim() != d || k->size(d - 1) != q->size(d - 1) ||
            k->sizes().slice(0, d - 2) != q->sizes().slice(0, d - 2) || !token_strides(*k, s + 9)))
    return decline();
  Call c(*q);
  if (!c.ok()) return nullptr;
  Tensor made[2];
  const Tensor* out[2] = {result_like(a[6], *q, &made[0]), nullptr};
  if (!out[0] || !token_strides(*out[0], s)) return decline();
  if (k && (!(out[1] = result_like(a[7], *k, &made[1])) || !token_strides(*out[1], s + 6))) return decline();
  const int r = without_gil([&] {
    return ctb_rope(c.ctx, c.stream, out[0]->data_ptr(), q->data_ptr(), k ? out[1]->data_ptr() : nullptr, k ? k->data_ptr() : nullptr,
                    pos->data_ptr(), index_bits(*pos), static_cast<const double*>(f->data_ptr()), d == 4 ? q->size(0) : 1, q->size(d - 3),
                    q->size(d - 2), k ? k->size(d - 2) : 0, q->size(d - 1), 2 * f->size(0), s, a[4] == Py_True, a[8] == Py_True, scale,
                    dtype_of(*q));
  });
  if (r != CTB_OK) return done(r, nullptr);
  return Py_BuildValue("(NN)", given_or(a[6], made[0]), k ? given_or(a[7], made[1]) : Py_NewRef(Py_None));
}

// A kvcache.KvCache (a tuple of k, v, k_scale or None, v_scale or None) in its ordinary form.
bool cache_of(PyObject* o, const Tensor& like, ctb_kv_cache* c) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
  const Tensor* t[4];
  for (int i = 0; i < 4; ++i) {
    PyObject* x = PyTuple_GET_ITEM(o, i);
    t[i] = x == Py_None ? nullptr : cuda_tensor(x);
    if ((!t[i] && (i < 2 || x != Py_None)) || (t[i] && t[i]->device() != like.device())) return false;
  }
  const Tensor &k = *t[0], &v = *t[1];
  if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) return false;
  switch (k.scalar_type()) {
    case at::kHalf: c->dtype = CTB_F16; break;
    case at::kBFloat16: c->dtype = CTB_BF16; break;
    case at::kFloat8_e4m3fn: c->dtype = CTB_E4M3; break;
    case at::kChar: c->dtype = CTB_I8; break;
    default: return false;
  }
  const bool bytes = c->dtype == CTB_E4M3 || c->dtype == CTB_I8;
  const int64_t D = k.size(3), page = k.size(2);
  for (const Tensor* x : {&k, &v})
    if (x->stride(3) != 1 || x->stride(2) != D || x->stride(1) != page * D) return false;
  for (int i = 2; i < 4; ++i) {
    if ((t[i] != nullptr) != bytes) return false;
    if (bytes && (t[i]->scalar_type() != at::kFloat || t[i]->sizes() != k.sizes().slice(0, 3) || t[i]->stride(2) != 1 || t[i]->stride(1) != page))
      return false;
  }
  c->k = k.data_ptr();
  c->v = v.data_ptr();
  c->k_scale = bytes ? static_cast<float*>(t[2]->data_ptr()) : nullptr;
  c->v_scale = bytes ? static_cast<float*>(t[3]->data_ptr()) : nullptr;
  c->pages = k.size(0);
  c->kv_heads = k.size(1);
  c->page_size = page;
  c->head_dim = D;
  c->k_page_stride = k.stride(0);
  c->v_page_stride = v.stride(0);
  c->k_scale_page_stride = bytes ? t[2]->stride(0) : 0;
  c->v_scale_page_stride = bytes ? t[3]->stride(0) : 0;
  return true;
}
// [tokens, heads, D] of the type and device of `like`, heads contiguous.
bool token_rows(const Tensor* t, const Tensor& like, int64_t T, int64_t D, int64_t* s) {
  if (!t || t->dim() != 3 || t->size(0) != T || t->size(2) != D || t->stride(2) != 1 || t->scalar_type() != like.scalar_type() ||
      t->device() != like.device())
    return false;
  s[0] = t->stride(0);
  s[1] = t->stride(1);
  return true;
}

// kv_write(cache, slots, k, v, q, positions, frequencies, interleaved, scale, out_q) -> (out_q or None,); q .. frequencies, out_q: or None.
// Positions without frequencies turn nothing.
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return decline();
  const Tensor *slots = cuda_tensor(a[1]), *k = cuda_tensor(a[2]), *v = cuda_tensor(a[3]);
  const Tensor *q = a[4] == Py_None ? nullptr : cuda_tensor(a[4]), *pos = a[5] == Py_None ? nullptr : cuda_tensor(a[5]);
  const Tensor* f = a[6] == Py_None ? nullptr : cuda_tensor(a[6]);
  ctb_kv_cache cache;
  float scale;
  int64_t s[8] = {};
  if (!slots || !k || !v || (!q && a[4] != Py_None) || (!pos && a[5] != Py_None) || (!f && a[6] != Py_None) || !PyBool_Check(a[7]) ||
      !as_float(a[8], &scale) || dtype_of(*k) < 0 || k->dim() != 3 || !cache_of(a[0], *k, &cache))
    return decline();
  const int64_t T = k->size(0), D = cache.head_dim;
  auto list = [&](const Tensor& t) { return t.dim() == 1 && t.size(0) == T && t.is_contiguous() && t.device() == k->device() && index_bits(t); };
  if (!list(*slots) || !token_rows(k, *k, T, D, s + 4) || !token_rows(v, *k, T, D, s + 6) || k->size(1) != cache.kv_heads ||
      v->size(1) != cache.kv_heads || (f && !pos) || (f && !frequencies_of(f, *k)) || (pos && !list(*pos)) ||
      (q && (!f || !token_rows(q, *k, T, D, s + 2))) || (!q && a[9] != Py_None))
    return decline();
  Call c(*k);
  if (!c.ok()) return nullptr;
  Tensor made;
  const Tensor* out = nullptr;
  if (q && (!(out = result_like(a[9], *q, &made)) || !token_rows(out, *k, T, D, s))) return decline();
  const int r = without_gil([&] {
    return ctb_kv_write(c.ctx, c.stream, &cache, slots->data_ptr(), index_bits(*slots), q ? out->data_ptr() : nullptr, q ? q->data_ptr() : nullptr,
                        k->data_ptr(), v->data_ptr(), s, f ? pos->data_ptr() : nullptr, f ? index_bits(*pos) : 32,
                        f ? static_cast<const double*>(f->data_ptr()) : nullptr, T, q ? q->size(1) : 0, f ? 2 * f->size(0) : 0, a[7] == Py_True,
                        scale, dtype_of(*k));
  });
  if (r != CTB_OK) return done(r, nullptr);
  return Py_BuildValue("(N)", q ? given_or(a[9], made) : Py_NewRef(Py_None));
}

bool page_table_of(const Tensor* table, const Tensor* lengths, const Tensor& like, int64_t* ld) {
  if (!table || !lengths || table->device() != like.device() || lengths->device() != like.device() || table->scalar_type() != at::kInt ||
      lengths->scalar_type() != at::kInt || table->dim() != 2 || lengths->dim() != 1 || lengths->size(0) != table->size(0) ||
      !lengths->is_contiguous() || (table->size(1) > 1 && table->stride(1) != 1))
    return false;
  *ld = table->size(0) > 1 ? table->stride(0) : std::max(table->size(1), table->stride(0));
  return true;
}

// kv_read(cache, page_table, lengths, max_length, dtype or None) -> (K, V)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) return decline();
  const Tensor *table = cuda_tensor(a[1]), *lengths = cuda_tensor(a[2]);
  ctb_kv_cache cache;
  long long seq;
  int64_t ld;
  if (!table || !page_table_of(table, lengths, *table, &ld) || !as_int(a[3], &seq) || seq < 0 || !cache_of(a[0], *table, &cache)) return decline();
  at::ScalarType type;
  if (THPDtype_Check(a[4])) type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  else if (a[4] == Py_None && cache.dtype == CTB_F16) type = at::kHalf;
  else if (a[4] == Py_None && cache.dtype == CTB_BF16) type = at::kBFloat16;
  else return decline();
  if (type != at::kHalf && type != at::kBFloat16) return decline();
  Call c(*table);
  if (!c.ok()) return nullptr;
  Tensor K = new_array({table->size(0), cache.kv_heads, seq, cache.head_dim}, type, *table), V = new_array(K.sizes(), type, *table);
  const int r = without_gil([&] {
    return ctb_kv_read(c.ctx, c.stream, K.data_ptr(), V.data_ptr(), &cache, static_cast<const int32_t*>(table->data_ptr()),
                       static_cast<const int32_t*>(lengths->data_ptr()), table->size(0), seq, table->size(1), ld,
                       type == at::kHalf ? CTB_F16 : CTB_BF16);
  });
  if (r != CTB_OK) return done(r, nullptr);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(K)), THPVariable_Wrap(std::move(V)));
}

// fmha_paged(Q, cache, page_table, lengths, qk_scale or None, return_lse) -> Out or (Out, lse)
PyObject* fmha_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) return decline();
  const Tensor *q = cuda_tensor(a[0]), *table = cuda_tensor(a[2]), *lengths = cuda_tensor(a[3]);
  ctb_kv_cache cache;
  int64_t ld, s[2];
  float scale;
  if (!q || q->dim() != 3 || dtype_of(*q) < 0 || !PyBool_Check(a[5]) || !page_table_of(table, lengths, *q, &ld) || !cache_of(a[1], *q, &cache) ||
      !token_rows(q, *q, table->size(0), cache.head_dim, s))
    return decline();
  if (a[4] == Py_None) scale = (float)(1.0 / std::sqrt((double)cache.head_dim));
  else if (!as_float(a[4], &scale)) return decline();
  Call c(*q);
  if (!c.ok()) return nullptr;
  const int64_t B = q->size(0), H = q->size(1);
  Tensor out = new_array({B, H, cache.head_dim}, q->scalar_type(), *q), lse;
  const bool with_lse = a[5] == Py_True;
  if (with_lse) lse = new_array({B, H}, at::kFloat, *q);
  const int r = without_gil([&] {
    return ctb_fmha_paged(c.ctx, c.stream, out.data_ptr(), with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, q->data_ptr(), &cache,
                          static_cast<const int32_t*>(table->data_ptr()), static_cast<const int32_t*>(lengths->data_ptr()), B, H, s[0], s[1],
                          table->size(1), ld, scale, dtype_of(*q));
  });
  if (r != CTB_OK) return done(r, nullptr);
  if (!with_lse) return THPVariable_Wrap(std::move(out));
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
}

// moe_router(hidden, W_r, topk) -> (gates [topk, T] f16, ids [topk, T] int32)
PyObject* moe_router(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor *x, *w;
  long long topk;
  if (n != 3 || !(x = cuda_tensor(a[0])) || !(w = cuda_tensor(a[1])) || !as_int(a[2], &topk) || x->dim() != 2 || w->dim() != 2 ||
      x->scalar_type() != at::kHalf || w->scalar_type() != at::kHalf || !x->is_contiguous() || !w->is_contiguous() ||
      x->size(1) != w->size(1) || topk < 1)
    return decline();
  const int64_t T = x->size(0), H = x->size(1), E = w->size(0);
  Call c(*x);
  if (!c.ok()) return nullptr;
  Tensor ids = at::empty({topk, T}, x->options().dtype(at::kInt)), gates = at::empty({topk, T}, x->options());
  const int s = without_gil([&] {
    return ctb_moe_router(c.ctx, c.stream, x->data_ptr(), w->data_ptr(), static_cast<int32_t*>(ids.data_ptr()), gates.data_ptr(),
                          nullptr, T, H, E, (int)topk);
  });
  if (s != CTB_OK) return done(s, nullptr);
  PyObject* g = THPVariable_Wrap(std::move(gates));
  PyObject* i = g ? THPVariable_Wrap(std::move(ids)) : nullptr;
  PyObject* r = i ? PyTuple_Pack(2, g, i) : nullptr;
  Py_XDECREF(g);
  Py_XDECREF(i);
  return r;
}

// moe_ffn(hidden, w1, w2, gates, ids, tile_m, tile_n, tile_k) -> out [T, H] f16
PyObject* moe_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* t[5];
  long long v[3];
  if (n != 8 || !ints(a + 5, 3, v)) return decline();
  for (int i = 0; i < 5; ++i)
    if (!(t[i] = cuda_tensor(a[i])) || !t[i]->is_contiguous() || (i < 4 && t[i]->scalar_type() != at::kHalf)) return decline();
  const Tensor &x = *t[0], &w1 = *t[1], &w2 = *t[2], &g = *t[3], &ids = *t[4];
  const int bits = ids.scalar_type() == at::kInt ? 32 : ids.scalar_type() == at::kLong ? 64 : 0;
  if (!bits || x.dim() != 2 || w1.dim() != 3 || w2.dim() != 3 || g.dim() != 2 || ids.dim() != 2) return decline();
  const int64_t T = x.size(0), H = x.size(1), E = w2.size(0), I = w2.size(2), topk = ids.size(0);
  if (w2.size(1) != H || w1.size(0) != E || w1.size(1) != 2 * I || w1.size(2) != H || ids.size(1) != T || g.size(0) != topk ||
      g.size(1) != T)
    return decline();
  Call c(x);
  if (!c.ok()) return nullptr;
  Tensor out = at::empty({T, H}, x.options());
  const int s = without_gil([&] {
    return ctb_moe_ffn(c.ctx, c.stream, x.data_ptr(), w1.data_ptr(), w2.data_ptr(), g.data_ptr(), ids.data_ptr(), bits,
                       out.data_ptr(), T, H, I, E, topk, (int)v[0], (int)v[1], (int)v[2]);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return THPVariable_Wrap(std::move(out));
}

// ---- rows of scores -----------------------------------------------------------------------------------------------
// A tensor or None; false: something else.
bool maybe_tensor(PyObject* o, const Tensor** t) {
  *t = nullptr;
  return o == Py_None || (*t = cuda_tensor(o));
}
bool same_device(const Tensor* t, const Tensor& x) { return !t || t->get_device() == x.get_device(); }
bool maybe_f32(const Tensor* t, const Tensor& x, at::IntArrayRef shape) {
  return !t || (t->scalar_type() == at::kFloat && t->sizes() == shape && t->is_contiguous() && same_device(t, x));
}
int bits_of(const Tensor& t) { return t.scalar_type() == at::kInt ? 32 : t.scalar_type() == at::kLong ? 64 : 0; }
float* f32(const Tensor* t) { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }
void* data(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
// logits with contiguous rows and the gradient's array (a new one when none is given)
struct Rows {
  const Tensor* x = nullptr;
  int64_t ld = 0, T = 0, V = 0, ld_out = 0;
  int dtype = -1;
  Tensor out;
  bool take(PyObject* o) { return (x = cuda_tensor(o)) && rows(*x, &ld, &T, &V) && (dtype = dtype_of(*x)) >= 0; }
  bool take_out(PyObject* o) {
    const Tensor* t;
    if (!maybe_tensor(o, &t)) return false;
    if (t) {
      int64_t m, k;
      if (!rows(*t, &ld_out, &m, &k) || m != T || k != V || t->scalar_type() != x->scalar_type() || !same_device(t, *x)) return false;
      out = *t;
    }
    return true;
  }
  void make_out() {
    if (out.defined()) return;
    out = at::empty({T, V}, x->options());
    ld_out = V;
  }
};
PyObject* pack(std::initializer_list<Tensor*> list) {  // a tuple; None for undefined tensors
  PyObject* r = PyTuple_New((Py_ssize_t)list.size());
  Py_ssize_t i = 0;
  for (Tensor* t : list) {
    PyObject* o = !r ? nullptr : t->defined() ? THPVariable_Wrap(std::move(*t)) : Py_NewRef(Py_None);
    if (!o) {
      Py_XDECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// token_logprobs(logits, tokens or None, top, temperature, entropy) -> (logprobs, entropy, lse, top_logprobs, top_ids)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  const Tensor* tokens;
  long long top;
  float temperature;
  if (n != 5 || !r.take(a[0]) || !maybe_tensor(a[1], &tokens) || !as_int(a[2], &top) || top < 0 || !as_float(a[3], &temperature) ||
      !PyBool_Check(a[4]))
    return decline();
  const int bits = tokens ? bits_of(*tokens) : 64;
  if (!bits || (tokens && (tokens->dim() != 1 || tokens->size(0) != r.T || !tokens->is_contiguous() || !same_device(tokens, *r.x))))
    return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  const auto f = r.x->options().dtype(at::kFloat);
  // one allocation for the vectors: each of its own would be 1.3 us of a call of 11
  const int64_t step = (r.T + 3) / 4 * 4;
  const Tensor all = at::empty({3 * step}, f);
  auto vector = [&](int i) {
    Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), all.dtype());
    v.unsafeGetTensorImpl()->set_sizes_contiguous({r.T});
    v.unsafeGetTensorImpl()->set_storage_offset(i * step);
    return v;
  };
  Tensor lp, h, lse = vector(0), tlp, tid;
  if (tokens) lp = vector(1);
  if (a[4] == Py_True) h = vector(2);
  if (top) {
    tlp = at::empty({r.T, top}, f);
    tid = at::empty({r.T, top}, f.dtype(at::kInt));
  }
  const int s = without_gil([&] {
    auto p = [](const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; };
    return ctb_token_logprobs(c.ctx, c.stream, r.x->data_ptr(), data(tokens), bits, p(lp), p(h), p(lse), p(tlp),
                              tid.defined() ? static_cast<int32_t*>(tid.data_ptr()) : nullptr, r.V, r.T, r.ld, (int)top, temperature,
                              r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return pack({&lp, &h, &lse, &tlp, &tid});
}

// token_logprobs_bwd(logits, tokens, lse, entropy, d_logprobs, d_entropy, top_ids, d_top_logprobs, temperature, out) -> out
PyObject* token_logprobs_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  const Tensor* t[7];  // tokens, lse, entropy, d_logprobs, d_entropy, top_ids, d_top
  float temperature;
  if (n != 10 || !r.take(a[0]) || !as_float(a[8], &temperature) || !r.take_out(a[9])) return decline();
  for (int i = 0; i < 7; ++i)
    if (!maybe_tensor(a[1 + i], &t[i])) return decline();
  const int bits = t[0] ? bits_of(*t[0]) : 64;
  if (!bits || (t[0] && (t[0]->dim() != 1 || t[0]->size(0) != r.T || !t[0]->is_contiguous() || !same_device(t[0], *r.x))) || !t[1] ||
      (t[4] && !t[2]) || (t[6] && !t[5]))
    return decline();
  for (int i = 1; i < 5; ++i)
    if (!maybe_f32(t[i], *r.x, {r.T})) return decline();
  int64_t top = 0;
  if (t[6]) {
    if (t[5]->dim() != 2 || t[5]->scalar_type() != at::kInt || !t[5]->is_contiguous() || !same_device(t[5], *r.x)) return decline();
    top = t[5]->size(1);
    if (t[5]->size(0) != r.T || !maybe_f32(t[6], *r.x, {r.T, top})) return decline();
  }
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  r.make_out();
  const int s = without_gil([&] {
    return ctb_token_logprobs_bwd(c.ctx, c.stream, r.out.data_ptr(), r.x->data_ptr(), data(t[0]), bits, f32(t[1]), f32(t[2]), f32(t[3]),
                                  f32(t[4]), top ? static_cast<const int32_t*>(t[5]->data_ptr()) : nullptr, top ? f32(t[6]) : nullptr,
                                  r.V, r.T, r.ld_out, r.ld, (int)top, temperature, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return THPVariable_Wrap(std::move(r.out));
}

// a teacher's list: ids [T, entries], values [T, entries]
struct Teacher {
  const Tensor *ids = nullptr, *values = nullptr;
  int bits = 0, dtype = -1, entries = 0;
  bool take(PyObject* i, PyObject* v, const Rows& r) {
    if (!(ids = cuda_tensor(i)) || !(values = cuda_tensor(v)) || ids->dim() != 2 || ids->size(0) != r.T || ids->size(1) > 4096 ||
        values->sizes() != ids->sizes() || !ids->is_contiguous() || !values->is_contiguous() || !same_device(ids, *r.x) ||
        !same_device(values, *r.x))
      return false;
    bits = bits_of(*ids);
    dtype = dtype_of(*values);
    entries = (int)ids->size(1);
    return bits && dtype >= 0;
  }
};

// distill_fwd(logits, ids, values, teacher_lse or None, temperature) -> (loss, saved)
PyObject* distill_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  Teacher t;
  const Tensor* lse;
  float temperature;
  if (n != 5 || !r.take(a[0]) || !t.take(a[1], a[2], r) || !maybe_tensor(a[3], &lse) || !maybe_f32(lse, *r.x, {r.T}) ||
      !as_float(a[4], &temperature))
    return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  const auto f = r.x->options().dtype(at::kFloat);
  Tensor loss = at::empty({r.T}, f), saved = at::empty({r.T, 8}, f);
  const int s = without_gil([&] {
    return ctb_distill_fwd(c.ctx, c.stream, r.x->data_ptr(), t.ids->data_ptr(), t.bits, t.values->data_ptr(), t.dtype, f32(lse), f32(&loss),
                           f32(&saved), r.V, r.T, r.ld, t.entries, temperature, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return pack({&loss, &saved});
}

// distill_bwd(logits, ids, values, saved, d_loss, temperature, out) -> out
PyObject* distill_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  Teacher t;
  const Tensor *saved, *d;
  float temperature;
  if (n != 7 || !r.take(a[0]) || !t.take(a[1], a[2], r) || !(saved = cuda_tensor(a[3])) || !maybe_f32(saved, *r.x, {r.T, 8}) ||
      !(d = cuda_tensor(a[4])) || !maybe_f32(d, *r.x, {r.T}) || !as_float(a[5], &temperature) || !r.take_out(a[6]))
    return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  r.make_out();
  const int s = without_gil([&] {
    return ctb_distill_bwd(c.ctx, c.stream, r.out.data_ptr(), r.x->data_ptr(), t.ids->data_ptr(), t.bits, t.values->data_ptr(), t.dtype,
                           f32(saved), f32(d), r.V, r.T, r.ld_out, r.ld, t.entries, temperature, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return THPVariable_Wrap(std::move(r.out));
}

// distill_fwd_bwd(logits, ids, values, d_loss, teacher_lse or None, temperature, out) -> (loss, out)
PyObject* distill_fwd_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  Teacher t;
  const Tensor *lse, *d;
  float temperature;
  if (n != 7 || !r.take(a[0]) || !t.take(a[1], a[2], r) || !(d = cuda_tensor(a[3])) || !maybe_f32(d, *r.x, {r.T}) ||
      !maybe_tensor(a[4], &lse) || !maybe_f32(lse, *r.x, {r.T}) || !as_float(a[5], &temperature) || !r.take_out(a[6]))
    return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  r.make_out();
  const auto f = r.x->options().dtype(at::kFloat);
  Tensor loss = at::empty({r.T}, f), saved = at::empty({r.T, 8}, f);
  const int s = without_gil([&] {
    return ctb_distill_fwd_bwd(c.ctx, c.stream, r.out.data_ptr(), r.x->data_ptr(), t.ids->data_ptr(), t.bits, t.values->data_ptr(), t.dtype,
                               f32(lse), f32(&loss), f32(&saved), f32(d), r.V, r.T, r.ld_out, r.ld, t.entries, temperature, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return pack({&loss, &r.out});
}

int score_of(PyObject* o) {  // -1: neither
  if (!PyUnicode_Check(o)) return -1;
  if (PyUnicode_CompareWithASCIIString(o, "softmax") == 0) return CTB_SCORE_SOFTMAX;
  return PyUnicode_CompareWithASCIIString(o, "sigmoid") == 0 ? CTB_SCORE_SIGMOID : -1;
}

// moe_route(logits, topk, bias or None, score, groups, topk_groups, group_top, renormalize, scale, weights' dtype) -> (weights, ids)
PyObject* moe_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  const Tensor* bias;
  long long topk, g[3];
  float scale;
  if (n != 10 || !r.take(a[0]) || !as_int(a[1], &topk) || topk < 1 || topk > r.V || !maybe_tensor(a[2], &bias) ||
      !maybe_f32(bias, *r.x, {r.V}) || !ints(a + 4, 3, g) || !PyBool_Check(a[7]) || !as_float(a[8], &scale) || !THPDtype_Check(a[9]))
    return decline();
  const int score = score_of(a[3]);
  const at::ScalarType wt = reinterpret_cast<THPDtype*>(a[9])->scalar_type;
  const int wdtype = wt == at::kFloat ? CTB_F32 : wt == at::kHalf ? CTB_F16 : wt == at::kBFloat16 ? CTB_BF16 : -1;
  if (score < 0 || wdtype < 0) return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  Tensor w = at::empty({topk, r.T}, r.x->options().dtype(wt)), ids = at::empty({topk, r.T}, r.x->options().dtype(at::kInt));
  const int s = without_gil([&] {
    return ctb_moe_route(c.ctx, c.stream, r.x->data_ptr(), f32(bias), static_cast<int32_t*>(ids.data_ptr()), w.data_ptr(), wdtype, r.T, r.V,
                         r.ld, (int)topk, score, (int)g[0], (int)g[1], (int)g[2], a[7] == Py_True, scale, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return pack({&w, &ids});
}

// moe_route_bwd(logits, ids, d_weights, score, renormalize, scale, out) -> out
PyObject* moe_route_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Rows r;
  const Tensor *ids, *d;
  float scale;
  if (n != 7 || !r.take(a[0]) || !(ids = cuda_tensor(a[1])) || !(d = cuda_tensor(a[2])) || !PyBool_Check(a[4]) || !as_float(a[5], &scale) ||
      !r.take_out(a[6]))
    return decline();
  const int score = score_of(a[3]), bits = bits_of(*ids), wdtype = dtype_of(*d);
  if (score < 0 || !bits || wdtype < 0 || ids->dim() != 2 || ids->size(1) != r.T || ids->size(0) > r.V || d->sizes() != ids->sizes() ||
      !ids->is_contiguous() || !d->is_contiguous() || !same_device(ids, *r.x) || !same_device(d, *r.x))
    return decline();
  Call c(*r.x);
  if (!c.ok()) return nullptr;
  r.make_out();
  const int s = without_gil([&] {
    return ctb_moe_route_bwd(c.ctx, c.stream, r.out.data_ptr(), r.x->data_ptr(), ids->data_ptr(), bits, d->data_ptr(), wdtype, r.T, r.V,
                             r.ld_out, r.ld, (int)ids->size(0), score, a[4] == Py_True, scale, r.dtype);
  });
  if (s != CTB_OK) return done(s, nullptr);
  return THPVariable_Wrap(std::move(r.out));
}

// ---- host-level array expressions ---------------------------------------------------------------------------------
// Expr and Tiled of the Python module `tiled` are the types below.  A fused expression is built of ten to twenty nodes
// per call; as Python classes a node cost 0.5-0.8 us (constructor, isinstance tests) and the walk that turns the tree
// into a program about 20 us, more than the kernel of an ordinary array.  As C types a node costs about 0.1 us and the
// walk about 1 us.
struct Node {
  PyObject_HEAD
  PyObject* node;    // ("leaf", tensor) | ("const", float) | (unary name, Expr) | (binary name, Expr, Expr)
  PyObject* tensor;  // Tiled only
  PyObject *dict, *weak;
};
PyTypeObject* g_expr = nullptr;
PyTypeObject* g_tiled = nullptr;
PyObject* g_leaf_error = nullptr;  // tiled._leaf_error(tensor): raises what is wrong with a leaf, or returns None
struct OpName { const char* name; int code; PyObject* str; };
OpName g_ops[] = {{"leaf", CTB_TILED_INPUT, nullptr}, {"const", CTB_TILED_CONST, nullptr}, {"identity", CTB_TILED_IDENTITY, nullptr},
                  {"neg", CTB_TILED_NEG, nullptr}, {"abs", CTB_TILED_ABS, nullptr}, {"sqrt", CTB_TILED_SQRT, nullptr},
                  {"exp", CTB_TILED_EXP, nullptr}, {"exp2", CTB_TILED_EXP2, nullptr}, {"log", CTB_TILED_LOG, nullptr},
                  {"log2", CTB_TILED_LOG2, nullptr}, {"sin", CTB_TILED_SIN, nullptr}, {"cos", CTB_TILED_COS, nullptr},
                  {"tanh", CTB_TILED_TANH, nullptr}, {"inv", CTB_TILED_INV, nullptr}, {"abs2", CTB_TILED_ABS2, nullptr},
                  {"add", CTB_TILED_ADD, nullptr}, {"sub", CTB_TILED_SUB, nullptr}, {"mul", CTB_TILED_MUL, nullptr},
                  {"div", CTB_TILED_DIV, nullptr}, {"max", CTB_TILED_MAX, nullptr}, {"min", CTB_TILED_MIN, nullptr},
                  {"pow", CTB_TILED_POW, nullptr}};
PyObject* op_str(int code) {
  for (auto& o : g_ops)
    if (o.code == code) return o.str;
  return nullptr;
}
int op_code(PyObject* name) {  // -1: not an operation
  for (auto& o : g_ops)
    if (o.str == name) return o.code;
  for (auto& o : g_ops)
    if (PyUnicode_Check(name) && PyUnicode_Compare(o.str, name) == 0) return o.code;
  return -1;
}

bool is_expr(PyObject* o) { return PyObject_TypeCheck(o, g_expr); }

PyObject* new_node(PyTypeObject* type, PyObject* tuple_owned, PyObject* tensor) {
  if (!tuple_owned) return nullptr;
  Node* n = reinterpret_cast<Node*>(type->tp_alloc(type, 0));
  if (!n) {
    Py_DECREF(tuple_owned);
    return nullptr;
  }
  n->node = tuple_owned;
  n->tensor = Py_XNewRef(tensor);
  return reinterpret_cast<PyObject*>(n);
}

int leaf_ok(PyObject* t) {  // 0 with a Python error set when the tensor cannot be a leaf
  try {
    const Tensor* c = cuda_tensor(t);
    if (c && c->dim() <= 3 && c->is_contiguous()) return 1;
  } catch (const std::exception& e) {  // type slots call this too: nothing may pass them
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return 0;
  }
  PyObject* r = PyObject_CallFunctionObjArgs(g_leaf_error, t, nullptr);
  Py_XDECREF(r);
  return r != nullptr;
}
PyObject* make_leaf(PyObject* t) {
  if (!leaf_ok(t)) return nullptr;
  return new_node(g_tiled, PyTuple_Pack(2, op_str(CTB_TILED_INPUT), t), t);
}

PyObject* wrap(PyObject* x) {  // new reference
  if (is_expr(x)) return Py_NewRef(x);
  if (THPVariable_Check(x)) return make_leaf(x);
  if (PyFloat_Check(x) || PyLong_Check(x)) {
    PyObject* f = PyNumber_Float(x);
    if (!f) return nullptr;
    PyObject* r = new_node(g_expr, PyTuple_Pack(2, op_str(CTB_TILED_CONST), f), nullptr);
    Py_DECREF(f);
    return r;
  }
  PyErr_Format(PyExc_TypeError, "a Tiled broadcast takes Tiled arrays and numbers, not %s", Py_TYPE(x)->tp_name);
  return nullptr;
}
PyObject* make_binary(int code, PyObject* a, PyObject* b) {
  PyObject* l = wrap(a);
  PyObject* r = l ? wrap(b) : nullptr;
  PyObject* out = r ? new_node(g_expr, PyTuple_Pack(3, op_str(code), l, r), nullptr) : nullptr;
  Py_XDECREF(l);
  Py_XDECREF(r);
  return out;
}
template <int CODE>
PyObject* nb_binary(PyObject* a, PyObject* b) { return make_binary(CODE, a, b); }
PyObject* nb_power(PyObject* a, PyObject* b, PyObject* mod) {
  if (!is_expr(a) || mod != Py_None) Py_RETURN_NOTIMPLEMENTED;
  return make_binary(CTB_TILED_POW, a, b);
}
template <int CODE>
PyObject* nb_unary(PyObject* a) { return new_node(g_expr, PyTuple_Pack(2, op_str(CODE), a), nullptr); }

int expr_init(PyObject* self, PyObject* args, PyObject* kw) {
  if (kw && PyDict_Size(kw)) {
    PyErr_SetString(PyExc_TypeError, "Expr takes no keyword arguments");
    return -1;
  }
  Py_XSETREF(reinterpret_cast<Node*>(self)->node, Py_NewRef(args));
  return 0;
}
int tiled_init(PyObject* self, PyObject* args, PyObject* kw) {
  static const char* names[] = {"tensor", nullptr};
  PyObject* t;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "O", const_cast<char**>(names), &t) || !leaf_ok(t)) return -1;
  PyObject* n = PyTuple_Pack(2, op_str(CTB_TILED_INPUT), t);
  if (!n) return -1;
  Py_XSETREF(reinterpret_cast<Node*>(self)->node, n);
  Py_XSETREF(reinterpret_cast<Node*>(self)->tensor, Py_NewRef(t));
  return 0;
}
int node_traverse(PyObject* self, visitproc visit, void* arg) {
  Py_VISIT(Py_TYPE(self));
  Py_VISIT(reinterpret_cast<Node*>(self)->node);
  Py_VISIT(reinterpret_cast<Node*>(self)->tensor);
  Py_VISIT(reinterpret_cast<Node*>(self)->dict);
  return 0;
}
int node_clear(PyObject* self) {
  Py_CLEAR(reinterpret_cast<Node*>(self)->node);
  Py_CLEAR(reinterpret_cast<Node*>(self)->tensor);
  Py_CLEAR(reinterpret_cast<Node*>(self)->dict);
  return 0;
}
void node_dealloc(PyObject* self) {
  PyTypeObject* type = Py_TYPE(self);
  PyObject_GC_UnTrack(self);
  Py_TRASHCAN_BEGIN(self, node_dealloc)
  if (reinterpret_cast<Node*>(self)->weak) PyObject_ClearWeakRefs(self);
  node_clear(self);
  type->tp_free(self);
  Py_DECREF(type);
  Py_TRASHCAN_END
}
PyObject* expr_wrap(PyObject*, PyObject* x) { return wrap(x); }
// For copies and pickles: a new object of the type, its attributes, then the members above (no __init__ runs).
PyObject* node_reduce(PyObject* self, PyObject*) {
  Node* n = reinterpret_cast<Node*>(self);
  PyObject* module = PyImport_ImportModule("copyreg");
  PyObject* make = module ? PyObject_GetAttrString(module, "__newobj__") : nullptr;
  PyObject* members = make ? PyDict_New() : nullptr;
  bool ok = members && (!n->node || PyDict_SetItemString(members, "node", n->node) == 0) &&
            (!n->tensor || PyDict_SetItemString(members, "tensor", n->tensor) == 0);
  PyObject* r = ok ? Py_BuildValue("O(O)(OO)", make, Py_TYPE(self), n->dict ? n->dict : Py_None, members) : nullptr;
  Py_XDECREF(members);
  Py_XDECREF(make);
  Py_XDECREF(module);
  return r;
}
PyMemberDef kNodeMembers[] = {{"node", Py_T_OBJECT_EX, offsetof(Node, node), 0, "the operation and its operands"},
                              {"__dictoffset__", Py_T_PYSSIZET, offsetof(Node, dict), Py_READONLY, nullptr},
                              {"__weaklistoffset__", Py_T_PYSSIZET, offsetof(Node, weak), Py_READONLY, nullptr},
                              {nullptr, 0, 0, 0, nullptr}};
PyMemberDef kTiledMembers[] = {{"tensor", Py_T_OBJECT_EX, offsetof(Node, tensor), 0, "the array"}, {nullptr, 0, 0, 0, nullptr}};
PyGetSetDef kExprGetSet[] = {{"__dict__", PyObject_GenericGetDict, PyObject_GenericSetDict, nullptr, nullptr},
                             {nullptr, nullptr, nullptr, nullptr, nullptr}};
PyMethodDef kExprMethods[] = {{"__reduce__", node_reduce, METH_NOARGS, nullptr},
                              {"wrap", expr_wrap, METH_O | METH_STATIC, "an Expr of an Expr, a tensor or a number"},
                              {nullptr, nullptr, 0, nullptr}};
template <class F>
void* slot(F f) { return reinterpret_cast<void*>(f); }
PyType_Slot kExprSlots[] = {
    {Py_tp_doc, const_cast<char*>("A node of a broadcast expression: (\"leaf\", tensor) | (\"const\", value) | (unary name, Expr) | "
                                  "(binary name, Expr, Expr).")},
    {Py_tp_init, slot(expr_init)}, {Py_tp_dealloc, slot(node_dealloc)}, {Py_tp_traverse, slot(node_traverse)},
    {Py_tp_clear, slot(node_clear)}, {Py_tp_members, kNodeMembers}, {Py_tp_methods, kExprMethods}, {Py_tp_getset, kExprGetSet},
    {Py_nb_add, slot(nb_binary<CTB_TILED_ADD>)}, {Py_nb_subtract, slot(nb_binary<CTB_TILED_SUB>)},
    {Py_nb_multiply, slot(nb_binary<CTB_TILED_MUL>)}, {Py_nb_true_divide, slot(nb_binary<CTB_TILED_DIV>)},
    {Py_nb_power, slot(nb_power)}, {Py_nb_negative, slot(nb_unary<CTB_TILED_NEG>)},
    {Py_nb_absolute, slot(nb_unary<CTB_TILED_ABS>)}, {0, nullptr}};
PyType_Spec kExprSpec = {"cutile_b200.tiled.Expr", sizeof(Node), 0, Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE | Py_TPFLAGS_HAVE_GC,
                         kExprSlots};
PyType_Slot kTiledSlots[] = {{Py_tp_doc, const_cast<char*>("``ct.Tiled(A)``: an array leaf.")}, {Py_tp_init, slot(tiled_init)},
                             {Py_tp_dealloc, slot(node_dealloc)}, {Py_tp_traverse, slot(node_traverse)},
                             {Py_tp_clear, slot(node_clear)}, {Py_tp_members, kTiledMembers}, {0, nullptr}};
PyType_Spec kTiledSpec = {"cutile_b200.tiled.Tiled", sizeof(Node), 0, Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE | Py_TPFLAGS_HAVE_GC,
                          kTiledSlots};

// unary(name, x), binary(name, a, b): the function forms (sin, tmax, ...)
PyObject* unary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "one argument expected");
    return nullptr;
  }
  PyObject* x = wrap(a[1]);
  if (!x) return nullptr;
  PyObject* t = PyTuple_Pack(2, a[0], x);
  Py_DECREF(x);
  return new_node(g_expr, t, nullptr);
}
PyObject* binary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "two arguments expected");
    return nullptr;
  }
  return make_binary(op_code(a[0]), a[1], a[2]);
}

// The tree as a postfix program over its distinct tensors and constants; false: more than the kernel takes (the Python
// path then reports it).
struct Walk {
  int32_t prog[2 * CTB_TILED_MAX_OPS];
  int n_ops = 0, n_in = 0, n_const = 0;
  PyObject* in[CTB_TILED_MAX_INPUTS];
  float consts[CTB_TILED_MAX_CONSTS];
  double exact[CTB_TILED_MAX_CONSTS];
  bool put(int op, int arg) {
    if (n_ops == CTB_TILED_MAX_OPS) return false;
    prog[2 * n_ops] = op;
    prog[2 * n_ops + 1] = arg;
    ++n_ops;
    return true;
  }
  bool walk(PyObject* e, int depth = 0) {
    PyObject* t = is_expr(e) ? reinterpret_cast<Node*>(e)->node : nullptr;
    if (!t || !PyTuple_Check(t) || PyTuple_GET_SIZE(t) < 2 || depth > CTB_TILED_MAX_OPS) return false;
    const int code = op_code(PyTuple_GET_ITEM(t, 0));
    const Py_ssize_t size = PyTuple_GET_SIZE(t);
    PyObject* x = PyTuple_GET_ITEM(t, 1);
    if (code == CTB_TILED_INPUT) {
      int i = 0;
      while (i < n_in && in[i] != x) ++i;
      if (i == CTB_TILED_MAX_INPUTS) return false;
      if (i == n_in) in[n_in++] = x;
      return put(CTB_TILED_INPUT, i);
    }
    if (code == CTB_TILED_CONST) {
      if (!PyFloat_Check(x)) return false;
      const double v = PyFloat_AS_DOUBLE(x);
      int i = 0;
      while (i < n_const && std::memcmp(&exact[i], &v, sizeof v)) ++i;  // 0.0 and -0.0 are two constants
      if (i == CTB_TILED_MAX_CONSTS) return false;
      if (i == n_const) {
        exact[n_const] = v;
        consts[n_const++] = (float)v;
      }
      return put(CTB_TILED_CONST, i);
    }
    if (code < 0 || size != (code >= CTB_TILED_ADD ? 3 : 2)) return false;
    for (Py_ssize_t k = 1; k < size; ++k)
      if (!walk(PyTuple_GET_ITEM(t, k), depth + 1)) return false;
    return put(code, 0);
  }
};
// Julia shape (first dimension contiguous) padded to three dimensions
void jshape(const Tensor& t, int64_t (&s)[3]) {
  const int d = (int)t.dim();
  for (int k = 0; k < 3; ++k) s[k] = k < d ? t.size(d - 1 - k) : 1;
}

// assign(dest, expr): dest .= expr
PyObject* assign(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor* dest;
  Walk w;
  if (n != 2 || !(dest = cuda_tensor(a[0])) || dest->dim() > 3 || !dest->is_contiguous() || dtype_of(*dest) < 0) return decline();
  PyObject* expr = wrap(a[1]);  // holds the operands until the call below is enqueued
  if (!expr) return nullptr;
  struct Hold {
    PyObject* o;
    ~Hold() { Py_DECREF(o); }
  } hold{expr};
  if (!w.walk(expr)) return decline();
  int64_t shape[3], strides[3 * CTB_TILED_MAX_INPUTS];
  const void* ptrs[CTB_TILED_MAX_INPUTS];
  jshape(*dest, shape);
  for (int i = 0; i < w.n_in; ++i) {
    const Tensor* t = cuda_tensor(w.in[i]);
    if (!t || t->dim() > 3 || !t->is_contiguous() || t->scalar_type() != dest->scalar_type() || t->device() != dest->device())
      return decline();
    int64_t s[3], run = 1;
    jshape(*t, s);
    for (int k = 0; k < 3; ++k) {
      if (s[k] != 1 && s[k] != shape[k]) return decline();
      strides[3 * i + k] = s[k] == 1 ? 0 : run;
      run *= s[k];
    }
    ptrs[i] = t->data_ptr();
  }
  Call c(*dest);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_tiled_broadcast(c.ctx, c.stream, dest->data_ptr(), shape, ptrs, strides, w.n_in, w.prog, w.n_ops, w.consts,
                               w.n_const, dtype_of(*dest));
  });
  return done(s, yes());
}

// mapreduce(f, op, tensor or Tiled, dims: None, int or tuple) -> the reduced tensor
PyObject* mapreduce(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return decline();
  PyObject* src = PyObject_TypeCheck(a[2], g_tiled) ? reinterpret_cast<Node*>(a[2])->tensor : a[2];
  const Tensor* t = src ? cuda_tensor(src) : nullptr;
  const int f = op_code(a[0]), op = op_code(a[1]);
  if (!t || t->dim() > 3 || !t->is_contiguous() || dtype_of(*t) < 0 || f < CTB_TILED_IDENTITY || f > CTB_TILED_ABS2 ||
      op < CTB_TILED_ADD)
    return decline();
  const int d = (int)t->dim();
  int mask = 0;
  long long v;
  auto add = [&](PyObject* o) {
    if (!as_int(o, &v) || v < 1) return false;
    if (v <= d) mask |= 1 << (v - 1);
    return true;
  };
  if (a[3] == Py_None) {
    mask = (1 << d) - 1;
  } else if (PyTuple_Check(a[3])) {
    for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(a[3]); ++k)
      if (!add(PyTuple_GET_ITEM(a[3], k))) return decline();
  } else if (!add(a[3])) {
    return decline();
  }
  int64_t shape[3], out[3];
  jshape(*t, shape);
  for (int k = 0; k < d; ++k) out[d - 1 - k] = (mask >> k) & 1 ? 1 : shape[k];
  Call c(*t);
  if (!c.ok()) return nullptr;
  Tensor dest = a[3] == Py_None ? at::empty({}, t->options()) : at::empty(at::IntArrayRef(out, d), t->options());
  const int s = without_gil([&] {
    return ctb_tiled_mapreduce(c.ctx, c.stream, dest.data_ptr(), t->data_ptr(), shape, mask, f, op, dtype_of(*t));
  });
  if (s != CTB_OK) return done(s, nullptr);
  return THPVariable_Wrap(std::move(dest));
}

// fft(x complex64 [batch, N], out or None, (W0, W1, W2, T0, T1) of make_twiddles, N, F0, F1, F2, D) -> out
PyObject* fft(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const Tensor *x, *out, *tab[2];
  long long v[5];
  if (n != 8 || !(x = cuda_tensor(a[0])) || !PyTuple_Check(a[2]) || PyTuple_GET_SIZE(a[2]) != 5 || !ints(a + 3, 5, v))
    return decline();
  const int64_t N = v[0], F0 = v[1], F1 = v[2], F2 = v[3];
  if (x->scalar_type() != at::kComplexFloat || x->dim() != 2 || x->size(1) != N || !x->is_contiguous() || x->is_conj())
    return decline();
  const int64_t want[2] = {2 * F0 * F1 * F2, 2 * F1 * F2};
  for (int i = 0; i < 2; ++i)
    if (!(tab[i] = cuda_tensor(PyTuple_GET_ITEM(a[2], 3 + i))) || !vec_f32(tab[i], want[i])) return decline();
  Tensor made;
  if (a[1] == Py_None) {
    made = at::empty(x->sizes(), x->options());
    out = &made;
  } else if (!(out = cuda_tensor(a[1])) || out->scalar_type() != at::kComplexFloat || out->sizes() != x->sizes() ||
             !out->is_contiguous() || out->is_conj()) {
    return decline();
  }
  Call c(*x);
  if (!c.ok()) return nullptr;
  const int s = without_gil([&] {
    return ctb_fft_plan(c.ctx, c.stream, x->data_ptr(), out->data_ptr(), tab[0]->data_ptr(), tab[1]->data_ptr(), N, (int)F0,
                        (int)F1, (int)F2, x->size(0), 1, (int)v[4]);
  });
  if (s != CTB_OK || a[1] != Py_None) return done(s, s == CTB_OK ? Py_NewRef(a[1]) : nullptr);
  return THPVariable_Wrap(std::move(made));
}

PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "setup(context, check, leaf_error)");
    return nullptr;
  }
  Py_XSETREF(g_context, Py_NewRef(a[0]));
  Py_XSETREF(g_check, Py_NewRef(a[1]));
  Py_XSETREF(g_leaf_error, Py_NewRef(a[2]));
  Py_RETURN_NONE;
}

// A C++ exception (out of memory from the allocator, say) becomes the Python exception torch raises for it.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(self, a, n);
  END_HANDLE_TH_ERRORS
}
#define CTB_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {CTB_METHOD(setup),         CTB_METHOD(softmax),        CTB_METHOD(vadd),
                          CTB_METHOD(transpose),     CTB_METHOD(layernorm_fwd),  CTB_METHOD(layernorm_bwd),
                          CTB_METHOD(layernorm_dwdb), CTB_METHOD(matmul),        CTB_METHOD(batch_matmul),
                          CTB_METHOD(fmha),          CTB_METHOD(moe_router),     CTB_METHOD(moe_ffn),
                          CTB_METHOD(unary),         CTB_METHOD(binary),         CTB_METHOD(assign),
                          CTB_METHOD(mapreduce),     CTB_METHOD(fft),
                          CTB_METHOD(token_logprobs), CTB_METHOD(token_logprobs_bwd), CTB_METHOD(distill_fwd),
                          CTB_METHOD(distill_bwd),   CTB_METHOD(distill_fwd_bwd), CTB_METHOD(moe_route),
                          CTB_METHOD(moe_route_bwd), CTB_METHOD(rope),           CTB_METHOD(kv_write),
                          CTB_METHOD(kv_read),       CTB_METHOD(fmha_paged),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", "Native call path of cutile_b200.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  for (auto& o : g_ops)
    if (!(o.str = PyUnicode_InternFromString(o.name))) return nullptr;
  PyObject* m = PyModule_Create(&kModule);
  if (!m) return nullptr;
  g_expr = reinterpret_cast<PyTypeObject*>(PyType_FromSpec(&kExprSpec));
  g_tiled = g_expr ? reinterpret_cast<PyTypeObject*>(PyType_FromSpecWithBases(&kTiledSpec, reinterpret_cast<PyObject*>(g_expr)))
                   : nullptr;
  if (!g_tiled || PyModule_AddStringConstant(m, "TORCH_VERSION", CTB_TORCH_VERSION) < 0 ||
      PyModule_AddObjectRef(m, "Expr", reinterpret_cast<PyObject*>(g_expr)) < 0 ||
      PyModule_AddObjectRef(m, "Tiled", reinterpret_cast<PyObject*>(g_tiled)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
