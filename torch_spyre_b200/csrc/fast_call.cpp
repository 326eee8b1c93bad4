// The plain case of the verification operators' Python calls, without Python:
// tensors that are all as the operator wants them, in eager mode with nothing
// to differentiate (rotary: with its gradient).  A function here checks that
// much, allocates the result and calls the C entry on the current stream; in
// every other case it returns None, and the caller takes the Python path, which
// raises or handles what was met.
// (Host time of rotary on 16 tokens: 12 us by the Python path, 4 by this one.)
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdlib>
#include <map>
#include <utility>

namespace {

// C entries, by address (the module is not linked to the library).
struct Entries {
  int (*rotary)(const void *, int32_t, int64_t, int64_t, void *, const float *, int64_t, int64_t, const int32_t *,
                int64_t, int64_t, int64_t, int32_t, int32_t, int32_t *, void *);
  int (*kv_store)(const void *, int64_t, int64_t, void *, const void *, int64_t, int64_t, const void *, int64_t,
                  int64_t, int32_t, void *, void *, int32_t, float *, float *, const int64_t *, const float *, int64_t,
                  int64_t, const int32_t *, int32_t, int64_t, int64_t, int64_t, int64_t, int64_t, int32_t *, void *);
  int (*kv_load)(const void *, int32_t, const float *, const int64_t *, void *, int32_t, int64_t, int64_t, int64_t,
                 int64_t, int32_t *, void *);
  int (*tree_mask)(const int32_t *, const int32_t *, int64_t, int64_t, int64_t, int64_t *, int32_t *, void *);
  int64_t (*tree_workspace_bytes)(int64_t, int64_t, int64_t, int64_t, int64_t);
  int (*tree_attention)(const void *, int32_t, int64_t, int64_t, const void *, const void *, int32_t, const float *,
                        const float *, const int32_t *, int64_t, const int32_t *, const int32_t *, const int64_t *,
                        int64_t, void *, float *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                        int64_t, float, void *, int64_t, int32_t *, void *);
  int (*tree_commit)(void *, void *, int32_t, float *, float *, const int32_t *, int64_t, const int32_t *,
                     const int32_t *, int64_t, const int32_t *, int32_t *, int64_t, int64_t, int64_t, int64_t, int64_t,
                     int64_t, int32_t *, void *);
} entries;
bool bound = false;

// The workspaces that the Python side made, by (device, stream); never freed.
using Key = std::pair<int, void *>;
std::map<Key, at::Tensor> &workspaces() {
  static auto *m = new std::map<Key, at::Tensor>;
  return *m;
}

int code_of(at::ScalarType t) {  // enum b200kv_dtype
  switch (t) {
    case at::kHalf: return 0;
    case at::kBFloat16: return 1;
    case at::kFloat: return 2;
    case at::kChar: return 3;
    case at::kFloat8_e4m3fn: return 4;
    default: return -1;
  }
}
bool is16(int code) { return code == 0 || code == 1; }
bool is8(int code) { return code == 3 || code == 4; }

// The arguments of one call: every tensor is taken from here, so that `ok` tells
// in the end whether all of them were plain CUDA tensors of one device.
struct Call {
  bool ok = bound;
  c10::Device device{c10::kCPU};
  bool has_device = false;

  Call() {
    using c10::DispatchKey;
    const c10::DispatchKeySet included = c10::impl::tls_local_dispatch_key_set().included_;
    ok = ok && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !included.has(DispatchKey::FuncTorchDynamicLayerFrontMode) && !included.has(DispatchKey::Tracer);
  }
  const at::Tensor *tensor(PyObject *o, bool with_grad = false) {
    if (!ok || !THPVariable_CheckExact(o)) {
      ok = false;
      return nullptr;
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    const bool grad = t.requires_grad() && c10::GradMode::is_enabled();
    const bool tangent = t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined();
    if (!t.is_cuda() || t.layout() != c10::kStrided || (grad && !with_grad) || tangent ||
        (has_device && t.device() != device)) {
      ok = false;
      return nullptr;
    }
    device = t.device();
    has_device = true;
    return &t;
  }
  const at::Tensor *optional(PyObject *o) { return o == Py_None ? nullptr : tensor(o); }
  // int32 flag; with B200KV_CHECK set the Python path reads it
  int32_t *flag(PyObject *o) {
    if (o == Py_None) return nullptr;
    const at::Tensor *t = tensor(o);
    const char *check = std::getenv("B200KV_CHECK");
    ok = ok && t->scalar_type() == at::kInt && t->numel() >= 1 && (!check || !*check || (*check == '0' && !check[1]));
    return ok ? t->data_ptr<int32_t>() : nullptr;
  }
  int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  void need(bool c) { ok = ok && c; }
};
bool vector_of(const at::Tensor *t, at::ScalarType type, int64_t n) {
  return t->dim() == 1 && t->scalar_type() == type && t->size(0) == n && t->is_contiguous();
}
void *data(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
void written(const at::Tensor *t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

struct Pool {
  int code = -1;
  int64_t blocks = 0, heads = 0, dim = 0;
};
Pool pool_of(Call &c, const at::Tensor *p, const at::Tensor *scales) {
  Pool r;
  if (!c.ok) return r;
  r.code = code_of(p->scalar_type());
  const int64_t stick = is8(r.code) ? 128 : 64;
  c.need((is8(r.code) || is16(r.code)) && p->dim() == 5 && p->size(3) == 64 && p->size(4) == stick && p->is_contiguous());
  if (!c.ok) return r;
  r.blocks = p->size(0);
  r.heads = p->size(1);
  r.dim = p->size(2) * stick;
  c.need((r.dim == 64 || r.dim == 128) && is8(r.code) == (scales != nullptr));
  if (c.ok && scales)
    c.need(scales->scalar_type() == at::kFloat && scales->dim() == 3 && scales->size(0) == r.blocks &&
           scales->size(1) == r.heads && scales->size(2) == 64 && scales->is_contiguous());
  return r;
}
Pool pools_of(Call &c, const at::Tensor *k, const at::Tensor *v, const at::Tensor *ks, const at::Tensor *vs) {
  const Pool p = pool_of(c, k, ks);
  pool_of(c, v, vs);
  if (c.ok) c.need(k->sizes() == v->sizes() && k->scalar_type() == v->scalar_type());
  return p;
}
bool rows_ok(const at::Tensor *x) { return x->dim() == 3 && x->stride(2) == 1; }
bool table_ok(const at::Tensor *t, const at::Tensor *pos, int64_t tokens, int64_t dim) {
  return t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(2) == 2 && t->is_contiguous() && t->size(1) > 0 &&
         2 * t->size(1) <= dim && vector_of(pos, at::kInt, tokens);
}
void *stream_of(const Call &c) { return c10::cuda::getCurrentCUDAStream(c.device.index()).stream(); }

#define B200KV_ARGS(count)                                     \
  if (n != count) {                                            \
    PyErr_SetString(PyExc_TypeError, "wrong argument count"); \
    return nullptr;                                            \
  }

// x turned, undefined if the entry refuses.
at::Tensor turn(const at::Tensor &x, const at::Tensor &table, const at::Tensor &pos, bool interleaved, bool transpose,
                int32_t *flag) {
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out = at::empty(x.sizes(), x.options());
  const int st = entries.rotary(x.data_ptr(), code_of(x.scalar_type()), x.stride(0), x.stride(1), out.data_ptr(),
                                static_cast<const float *>(table.data_ptr()), table.size(0), 2 * table.size(1),
                                static_cast<const int32_t *>(pos.data_ptr()), x.size(0), x.size(1), x.size(2),
                                interleaved, transpose, flag,
                                c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
  return st == 0 ? out : at::Tensor();
}

// rotary with its gradient: the same map turned the other way.
struct Turn : torch::autograd::Function<Turn> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &table,
                            const at::Tensor &pos, bool interleaved, bool transpose,
                            const std::optional<at::Tensor> &flag) {
    ctx->save_for_backward({table, pos});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["transpose"] = transpose;
    ctx->saved_data["flag"] = flag;
    at::Tensor out = turn(x, table, pos, interleaved, transpose, flag ? flag->data_ptr<int32_t>() : nullptr);
    TORCH_CHECK(out.defined(), "b200kv_rotary failed");
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    at::Tensor g = grads[0];
    if (g.dim() == 3 && g.stride(2) != 1) g = g.contiguous();  // e.g. the expanded gradient of a sum
    at::Tensor none;
    return {Turn::apply(g, saved[0], saved[1], ctx->saved_data["interleaved"].toBool(),
                        !ctx->saved_data["transpose"].toBool(), ctx->saved_data["flag"].toOptional<at::Tensor>()),
            none, none, none, none, none};
  }
};

// rotary(x, table, positions, interleaved, transpose, error_flag)
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(6)
  Call c;
  const at::Tensor *x = c.tensor(a[0], true), *table = c.tensor(a[1]), *pos = c.tensor(a[2]);
  int32_t *flag = c.flag(a[5]);
  if (!c.ok || !rows_ok(x)) Py_RETURN_NONE;
  const int code = code_of(x->scalar_type());
  if (code < 0 || code > 2 || !table_ok(table, pos, x->size(0), x->size(2))) Py_RETURN_NONE;
  const bool interleaved = a[3] == Py_True, transpose = a[4] == Py_True;
  at::Tensor out;
  if (!x->requires_grad() || !c10::GradMode::is_enabled()) {
    out = turn(*x, *table, *pos, interleaved, transpose, flag);
  } else {
    // (what the entry refuses goes to the Python path, which says so)
    if (x->size(2) > 4096 || x->size(1) > 65536 || x->size(0) >= int64_t(1) << 31 || x->numel() == 0 ||
        table->size(0) == 0 || reinterpret_cast<uintptr_t>(table->data_ptr()) % 8 != 0)
      Py_RETURN_NONE;
    std::optional<at::Tensor> kept;
    if (flag) kept = THPVariable_Unpack(a[5]);
    out = Turn::apply(*x, *table, *pos, interleaved, transpose, kept);
  }
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// kv_store(k, v, k_pool, v_pool, slots, k_scales, v_scales, q, table, positions, interleaved, error_flag)
// -> q turned, or True
PyObject *kv_store(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(12)
  Call c;
  const at::Tensor *k = c.tensor(a[0]), *v = c.tensor(a[1]), *kp = c.tensor(a[2]), *vp = c.tensor(a[3]),
                   *slots = c.tensor(a[4]), *ks = c.optional(a[5]), *vs = c.optional(a[6]), *q = c.optional(a[7]),
                   *table = c.optional(a[8]), *pos = c.optional(a[9]);
  int32_t *flag = c.flag(a[11]);
  const Pool p = pools_of(c, kp, vp, ks, vs);
  if (!c.ok || !rows_ok(k) || !rows_ok(v)) Py_RETURN_NONE;
  const int code = code_of(k->scalar_type());
  const int64_t tokens = k->size(0);
  c.need(is16(code) && v->scalar_type() == k->scalar_type() && k->size(1) == p.heads && k->size(2) == p.dim &&
         v->sizes() == k->sizes() && (is8(p.code) || p.code == code) && vector_of(slots, at::kLong, tokens));
  if (q) c.need(table && rows_ok(q) && q->scalar_type() == k->scalar_type() && q->size(0) == tokens && q->size(2) == p.dim);
  if (c.ok && table) c.need(pos && table_ok(table, pos, tokens, p.dim));
  if (!c.ok) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor out;
  if (q) out = at::empty(q->sizes(), q->options());
  const int st = entries.kv_store(
      data(q), q ? q->stride(0) : 0, q ? q->stride(1) : 0, q ? out.data_ptr() : nullptr, k->data_ptr(), k->stride(0),
      k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), code, kp->data_ptr(), vp->data_ptr(), p.code,
      static_cast<float *>(data(ks)), static_cast<float *>(data(vs)), static_cast<const int64_t *>(data(slots)),
      static_cast<const float *>(data(table)), table ? table->size(0) : 0, table ? 2 * table->size(1) : 0,
      static_cast<const int32_t *>(table ? data(pos) : nullptr), a[10] == Py_True, tokens, q ? q->size(1) : 0, p.heads,
      p.dim, p.blocks, flag, stream_of(c));
  if (st != 0) Py_RETURN_NONE;
  for (const at::Tensor *t : {kp, vp, ks, vs}) written(t);
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
}

// kv_load(pool, slots, scales, dtype code, error_flag)
PyObject *kv_load(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(5)
  Call c;
  const at::Tensor *pool = c.tensor(a[0]), *slots = c.tensor(a[1]), *scales = c.optional(a[2]);
  const int64_t code = c.integer(a[3]);
  int32_t *flag = c.flag(a[4]);
  const Pool p = pool_of(c, pool, scales);
  if (!c.ok || code < 0 || code > 2 || slots->dim() != 1 || !vector_of(slots, at::kLong, slots->size(0))) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(c.device);
  const at::ScalarType type = code == 0 ? at::kHalf : (code == 1 ? at::kBFloat16 : at::kFloat);
  at::Tensor out = at::empty({slots->size(0), p.heads, p.dim}, pool->options().dtype(type));
  const int st = entries.kv_load(pool->data_ptr(), p.code, static_cast<const float *>(data(scales)),
                                 static_cast<const int64_t *>(data(slots)), out.data_ptr(), static_cast<int32_t>(code),
                                 slots->size(0), p.heads, p.dim, p.blocks, flag, stream_of(c));
  if (st != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

bool sequences_ok(const at::Tensor *table, const at::Tensor *lens) {
  return table->scalar_type() == at::kInt && table->dim() == 2 && table->stride(1) == 1 &&
         vector_of(lens, at::kInt, table->size(0));
}

// tree_mask(parents, q_indptr, mask_words, error_flag)
PyObject *tree_mask(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(4)
  Call c;
  const at::Tensor *parents = c.tensor(a[0]), *indptr = c.tensor(a[1]);
  const int64_t words = c.integer(a[2]);
  int32_t *flag = c.flag(a[3]);
  if (!c.ok || parents->dim() != 1 || indptr->dim() != 1 || indptr->size(0) < 1 || words < 1) Py_RETURN_NONE;
  if (!vector_of(parents, at::kInt, parents->size(0)) || !vector_of(indptr, at::kInt, indptr->size(0))) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor mask = at::empty({parents->size(0), words}, parents->options().dtype(at::kLong));
  const int st = entries.tree_mask(static_cast<const int32_t *>(data(parents)), static_cast<const int32_t *>(data(indptr)),
                                   indptr->size(0) - 1, parents->size(0), words, static_cast<int64_t *>(mask.data_ptr()),
                                   flag, stream_of(c));
  if (st != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(mask));
}

// tree_attention(q, k_pool, v_pool, block_table, context_lens, q_indptr, mask, scale, max_nodes, k_scales, v_scales,
//                error_flag, want_lse) -> (out, lse or None)
PyObject *tree_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(13)
  Call c;
  const at::Tensor *q = c.tensor(a[0]), *kp = c.tensor(a[1]), *vp = c.tensor(a[2]), *table = c.tensor(a[3]),
                   *lens = c.tensor(a[4]), *indptr = c.tensor(a[5]), *mask = c.optional(a[6]), *ks = c.optional(a[9]),
                   *vs = c.optional(a[10]);
  const double scale = PyFloat_AsDouble(a[7]);
  if (scale == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const int64_t max_nodes = c.integer(a[8]);
  int32_t *flag = c.flag(a[11]);
  const Pool p = pools_of(c, kp, vp, ks, vs);
  if (!c.ok || !rows_ok(q) || !sequences_ok(table, lens)) Py_RETURN_NONE;
  const int code = code_of(q->scalar_type());
  const int64_t N = q->size(0), hq = q->size(1), batch = table->size(0);
  c.need(is16(code) && q->size(2) == p.dim && (is8(p.code) || p.code == code) && vector_of(indptr, at::kInt, batch + 1));
  if (c.ok && mask) c.need(mask->scalar_type() == at::kLong && mask->dim() == 2 && mask->size(0) == N && mask->is_contiguous());
  if (!c.ok || N == 0) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(c.device);
  void *stream = stream_of(c);
  const auto ws = workspaces().find(Key(c.device.index(), stream));
  const int64_t bytes = entries.tree_workspace_bytes(N, batch, hq, p.heads, p.dim);
  if (ws == workspaces().end() || bytes <= 0 || ws->second.numel() < bytes) Py_RETURN_NONE;
  at::Tensor out = at::empty(q->sizes(), q->options()), lse;
  if (a[12] == Py_True) lse = at::empty({N, hq}, q->options().dtype(at::kFloat));
  const int st = entries.tree_attention(
      q->data_ptr(), code, q->stride(0), q->stride(1), kp->data_ptr(), vp->data_ptr(), p.code,
      static_cast<const float *>(data(ks)), static_cast<const float *>(data(vs)),
      static_cast<const int32_t *>(data(table)), table->stride(0), static_cast<const int32_t *>(data(lens)),
      static_cast<const int32_t *>(data(indptr)), static_cast<const int64_t *>(data(mask)), mask ? mask->size(1) : 0,
      out.data_ptr(), lse.defined() ? static_cast<float *>(lse.data_ptr()) : nullptr, N, batch, hq, p.heads, p.dim,
      p.blocks, table->size(1), max_nodes, static_cast<float>(scale), ws->second.data_ptr(), ws->second.numel(), flag,
      stream);
  if (st != 0) Py_RETURN_NONE;
  PyObject *o = THPVariable_Wrap(std::move(out));
  PyObject *l = Py_None;
  if (lse.defined())
    l = THPVariable_Wrap(std::move(lse));
  else
    Py_INCREF(l);
  PyObject *pair = o && l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_XDECREF(o);
  Py_XDECREF(l);
  return pair;
}

// tree_commit(k_pool, v_pool, block_table, context_lens, path, path_lens, k_scales, v_scales, error_flag)
PyObject *tree_commit(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(9)
  Call c;
  const at::Tensor *kp = c.tensor(a[0]), *vp = c.tensor(a[1]), *table = c.tensor(a[2]), *lens = c.tensor(a[3]),
                   *path = c.tensor(a[4]), *plens = c.tensor(a[5]), *ks = c.optional(a[6]), *vs = c.optional(a[7]);
  int32_t *flag = c.flag(a[8]);
  const Pool p = pools_of(c, kp, vp, ks, vs);
  if (!c.ok || !sequences_ok(table, lens)) Py_RETURN_NONE;
  const int64_t batch = table->size(0);
  if (path->scalar_type() != at::kInt || path->dim() != 2 || path->size(0) != batch ||
      (path->size(1) > 1 && path->stride(1) != 1) || !vector_of(plens, at::kInt, batch))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(c.device);
  at::Tensor out = at::empty(lens->sizes(), lens->options());
  const int st = entries.tree_commit(
      kp->data_ptr(), vp->data_ptr(), p.code, static_cast<float *>(data(ks)), static_cast<float *>(data(vs)),
      static_cast<const int32_t *>(data(table)), table->stride(0), static_cast<const int32_t *>(data(lens)),
      static_cast<const int32_t *>(data(path)), batch > 1 ? path->stride(0) : path->size(1),
      static_cast<const int32_t *>(data(plens)), static_cast<int32_t *>(out.data_ptr()), batch, p.heads, p.dim, p.blocks,
      table->size(1), path->size(1), flag, stream_of(c));
  if (st != 0) Py_RETURN_NONE;
  for (const at::Tensor *t : {kp, vp, ks, vs}) written(t);
  return THPVariable_Wrap(std::move(out));
}

// bind(addresses): the C entries in the order of Entries
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(7)
  void **slots = reinterpret_cast<void **>(&entries);
  for (Py_ssize_t i = 0; i < n; ++i) {
    slots[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  bound = true;
  Py_RETURN_NONE;
}

// set_workspace(tensor): for the tensor's device and its current stream
PyObject *set_workspace(PyObject *, PyObject *const *a, Py_ssize_t n) {
  B200KV_ARGS(1)
  if (!THPVariable_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "a tensor is needed");
    return nullptr;
  }
  const at::Tensor &t = THPVariable_Unpack(a[0]);
  workspaces()[Key(t.device().index(), c10::cuda::getCurrentCUDAStream(t.device().index()).stream())] = t;
  Py_RETURN_NONE;
}

// A C++ exception (an allocation that failed, say) leaves as a RuntimeError.
template <PyObject *(*kFn)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
  try {
    return kFn(self, a, n);
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
#define B200KV_METHOD(f) \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&guarded<f>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {B200KV_METHOD(rotary),         B200KV_METHOD(kv_store),    B200KV_METHOD(kv_load),
                         B200KV_METHOD(tree_mask),      B200KV_METHOD(tree_attention), B200KV_METHOD(tree_commit),
                         B200KV_METHOD(bind),           B200KV_METHOD(set_workspace), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
