// Launches of the forward and backward from torch tensors (CPython extension
// pallas_flexattn/_launch.so): outputs and workspace allocated, operands made
// dense and the C ABI called without going through Python objects and ctypes
// conversions for every pointer.  Host code only; the C ABI's entry points are
// handed over by address (bind), so it links against torch alone.
//
// The calls around a KV cache (rotary, append, decode over e4m3 pages, prompts, latent vectors, pages) are checked here
// too: their struct arguments are filled from the tensors' own shapes and strides,
// and they run on the current stream of their tensors' device.
//
// Why: a small training step is bound by the host.  At B2 H4 S300 D64 the
// Python form of these two calls took 13 us (forward) and 18 us (backward; about
// 34 on the autograd engine's thread) of a 136 us step whose kernels take 40.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <vector>

#include "../../include/flexattn.h"

namespace {

using fwd_fn = int (*)(const void*, const void*, const void*, const void*, void*, float*, void*);
using bwd_fn = int (*)(const void*, const void*, const void*, const void*, const void*, const float*, const void*,
                       void*, void*, void*, void*, size_t, void*);
using ws_fn = size_t (*)(const void*);

fwd_fn g_fwd = nullptr;
bwd_fn g_bwd = nullptr;
ws_fn g_bwd_ws = nullptr;

void* address(PyObject* x) { return PyLong_AsVoidPtr(x); }

// Contiguous with a 16-byte aligned base (the kernels use 16-byte loads).
at::Tensor dense16(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 15) ? c.clone() : c;
}

const at::Tensor* tensor(PyObject* x) {
  if (!THPVariable_Check(x)) {
    PyErr_SetString(PyExc_TypeError, "expected a torch tensor");
    return nullptr;
  }
  return &THPVariable_Unpack(x);
}

// bind(fa_fwd, fa_bwd_split, fa_bwd_split_workspace_bytes)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "bind takes 3 addresses");
    return nullptr;
  }
  g_fwd = reinterpret_cast<fwd_fn>(address(a[0]));
  g_bwd = reinterpret_cast<bwd_fn>(address(a[1]));
  g_bwd_ws = reinterpret_cast<ws_fn>(address(a[2]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// fwd(params, q, k, v, stream) -> (status, o, lse).  The caller has checked
// q, k, v against each other and against the params.
PyObject* py_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !g_fwd) {
    PyErr_SetString(PyExc_TypeError, "fwd(params, q, k, v, stream) after bind");
    return nullptr;
  }
  const void* params = address(a[0]);
  void* stream = address(a[4]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t[3];
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = tensor(a[1 + i]))) return nullptr;
  const at::Tensor q = dense16(*t[0]), k = dense16(*t[1]), v = dense16(*t[2]);
  at::Tensor o = at::empty_like(q);
  at::Tensor lse = at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat));
  const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
  void* op = o.mutable_data_ptr();
  float* lp = lse.mutable_data_ptr<float>();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_fwd(params, qp, kp, vp, op, lp, stream);
  Py_END_ALLOW_THREADS
  return Py_BuildValue("iNN", rc, THPVariable_Wrap(o), THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// bwd(params, q, k, v, o, lse, do, stream) -> (status, dq, dk, dv)
PyObject* py_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !g_bwd) {
    PyErr_SetString(PyExc_TypeError, "bwd(params, q, k, v, o, lse, do, stream) after bind");
    return nullptr;
  }
  const void* params = address(a[0]);
  void* stream = address(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = tensor(a[1 + i]))) return nullptr;
  const at::Tensor q = dense16(*t[0]), k = dense16(*t[1]), v = dense16(*t[2]), o = dense16(*t[3]);
  const at::Tensor lse = t[4]->scalar_type() == at::kFloat ? t[4]->contiguous() : t[4]->to(at::kFloat).contiguous();
  const at::Tensor dout = dense16(t[5]->scalar_type() == q.scalar_type() ? *t[5] : t[5]->to(q.scalar_type()));
  if (o.sizes() != q.sizes() || dout.sizes() != q.sizes() || lse.sizes() != q.sizes().slice(0, 3) ||
      o.scalar_type() != q.scalar_type()) {
    PyErr_SetString(PyExc_ValueError, "o / do / lse shapes do not match q");
    return nullptr;
  }
  if (o.device() != q.device() || dout.device() != q.device() || lse.device() != q.device()) {
    PyErr_SetString(PyExc_ValueError, "o / do / lse are not on q's device");
    return nullptr;
  }
  const size_t need = g_bwd_ws(params), bytes = need < 256 ? 256 : need;
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr(), *op = o.const_data_ptr(),
             *dp = dout.const_data_ptr();
  const float* lp = lse.const_data_ptr<float>();
  void *gq = dq.mutable_data_ptr(), *gk = dk.mutable_data_ptr(), *gv = dv.mutable_data_ptr(), *wp = ws.mutable_data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_bwd(params, qp, kp, vp, op, lp, dp, gq, gk, gv, wp, bytes, stream);
  Py_END_ALLOW_THREADS
  return Py_BuildValue("iNNN", rc, THPVariable_Wrap(dq), THPVariable_Wrap(dk), THPVariable_Wrap(dv));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------ around a KV cache ----
decltype(&fa_apply_rotary) g_rotary = nullptr;
decltype(&fa_kv_append) g_append = nullptr;
decltype(&fa_fwd_kvcache_fp8) g_decode = nullptr;
decltype(&fa_fwd_kvcache_fp8_workspace_bytes) g_decode_ws = nullptr;
decltype(&fa_int64_to_int32) g_saturate = nullptr;
decltype(&fa_strerror) g_strerror = nullptr;

// bind_cache(fa_apply_rotary, fa_kv_append, fa_fwd_kvcache_fp8, fa_fwd_kvcache_fp8_workspace_bytes,
//            fa_int64_to_int32, fa_strerror)
PyObject* py_bind_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "bind_cache takes 6 addresses");
    return nullptr;
  }
  g_rotary = reinterpret_cast<decltype(g_rotary)>(address(a[0]));
  g_append = reinterpret_cast<decltype(g_append)>(address(a[1]));
  g_decode = reinterpret_cast<decltype(g_decode)>(address(a[2]));
  g_decode_ws = reinterpret_cast<decltype(g_decode_ws)>(address(a[3]));
  g_saturate = reinterpret_cast<decltype(g_saturate)>(address(a[4]));
  g_strerror = reinterpret_cast<decltype(g_strerror)>(address(a[5]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

#define REFUSE(type, text)          \
  do {                              \
    PyErr_SetString(type, text);    \
    return nullptr;                 \
  } while (0)

// A tensor argument, or a null pointer for None; false with an exception set otherwise.
bool optional(PyObject* x, const at::Tensor** t) {
  *t = nullptr;
  if (x == Py_None) return true;
  return (*t = tensor(x)) != nullptr;
}

// (B, H, T, D) with rows that the kernels' 16-byte accesses can take as they
// are, else a dense copy.
bool rows_ok(const at::Tensor& t) {
  const int64_t m = 16 / t.element_size() - 1;
  if (t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) & m)) return false;
  return true;
}
fa_strided strided(const at::Tensor& t) {
  fa_strided s{};
  s.data = t.const_data_ptr();
  // (strides of dimensions of size one are never used: they may be anything)
  s.stride_b = t.size(0) > 1 ? t.stride(0) : 0;
  s.stride_h = t.size(1) > 1 ? t.stride(1) : 0;
  s.stride_t = t.size(2) > 1 ? t.stride(2) : 0;
  s.heads = static_cast<int32_t>(t.size(1));
  return s;
}
constexpr int64_t kMaxSize = 0x7fffffff;
bool sizes_fit(const at::Tensor& t) {
  for (int64_t d : t.sizes())
    if (d > kMaxSize) return false;
  return true;
}

const char* const kFreqText = "inv_freq must be a dense float64 vector with at most head_dim / 2 entries";
bool freq_ok(const at::Tensor& f, int64_t D) {
  return f.dim() == 1 && f.scalar_type() == at::kDouble && f.is_contiguous() && f.size(0) >= 1 && 2 * f.size(0) <= D;
}

void* stream_of(const at::Device& dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

// Lengths or page ids, int32 or int64, as dense int32 on dev (the current device).  What 32 bits do not hold becomes
// their first or last number: a page or a length as impossible as it.
at::Tensor row_ints(const at::Tensor& t, const at::Device& dev) {
  if (t.scalar_type() == at::kInt) return t.device() == dev && t.is_contiguous() ? t : t.to(dev).contiguous();
  const at::Tensor x = t.to(dev).contiguous();
  at::Tensor y = at::empty(x.sizes(), x.options().dtype(at::kInt));
  const int rc = x.numel() ? g_saturate(x.const_data_ptr<int64_t>(), y.mutable_data_ptr<int32_t>(), x.numel(), stream_of(dev)) : FA_OK;
  TORCH_CHECK(rc == FA_OK, "flexattn C ABI error ", rc, ": ", g_strerror(rc));
  return y;
}

struct Turn {  // how a rotary call turns, besides its tensors
  bool interleaved, inverse;
  double scale;
  int64_t offset;
};

// Whether a forward-mode derivative (a dual tensor's tangent) comes with t: nothing here computes one, and a
// dual tensor need not require grad.
bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
const char* const kTangentText = "apply_rotary has no forward-mode derivative";

// fa_apply_rotary on checked tensors; k and pos may be undefined.
std::vector<at::Tensor> turn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& f, const at::Tensor& pos,
                             const Turn& t) {
  const c10::DeviceGuard guard(q.device());
  std::vector<at::Tensor> out;
  at::Tensor src[2], p;
  const int64_t B = q.size(0), T = q.size(2), D = q.size(3);
  fa_rotary_call c{};
  c.abi_version = FA_ABI_VERSION;
  c.dtype = q.scalar_type() == at::kFloat ? FA_DTYPE_F32 : FA_DTYPE_BF16;
  c.B = static_cast<int32_t>(B);
  c.T = static_cast<int32_t>(T);
  c.D = static_cast<int32_t>(D);
  c.inverse = t.inverse;
  c.rotary.inv_freq = f.const_data_ptr<double>();
  c.rotary.pairs = static_cast<int32_t>(f.size(0));
  c.rotary.interleaved = t.interleaved;
  c.rotary.scale = static_cast<float>(t.scale);
  for (const at::Tensor* x : {&q, &k}) {
    if (!x->defined()) continue;
    out.push_back(at::empty(x->sizes(), x->options()));
    if (x->numel() == 0) continue;
    at::Tensor& s = src[c.count];
    s = x->stride(3) == 1 || D == 1 ? *x : x->contiguous();
    c.in[c.count] = strided(s);
    c.out[c.count++] = out.back().mutable_data_ptr();
  }
  if (pos.defined()) {
    p = pos.size(-1) <= 1 || pos.stride(-1) == 1 ? pos : pos.contiguous();
    c.positions = p.const_data_ptr();
    c.positions_64 = p.scalar_type() == at::kLong;
    c.positions_stride = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
  }
  c.offset = t.offset;
  if (c.count) {
    const int rc = g_rotary(&c, stream_of(q.device()));
    TORCH_CHECK(rc == FA_OK, "flexattn C ABI error ", rc, ": ", g_strerror(rc));
  }
  return out;
}

// The rotation as an autograd node: as a Python function, which crosses into the
// interpreter twice (once from the engine's thread), forward and gradient took 68 us at B2 H4 S300 D64, so 60.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const std::optional<at::Tensor>& k, const at::Tensor& f,
                                                const std::optional<at::Tensor>& pos, bool interleaved, bool inverse,
                                                double scale, int64_t offset) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({f, pos ? *pos : at::Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["offset"] = offset;
    return turn(q, k ? *k : at::Tensor(), f, pos ? *pos : at::Tensor(), {interleaved, inverse, scale, offset});
  }
  static std::optional<at::Tensor> given(const at::Tensor& t) {
    return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt;
  }
  // The rotation's transpose; a node again where the gradient is differentiated.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Turn t{ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool(),
                 ctx->saved_data["scale"].toDouble(), ctx->saved_data["offset"].toInt()};
    at::Tensor gq = ctx->needs_input_grad(0) ? g[0] : at::Tensor();
    at::Tensor gk = g.size() > 1 && ctx->needs_input_grad(1) ? g[1] : at::Tensor();
    torch::autograd::variable_list out(8);
    if (!gq.defined() && !gk.defined()) return out;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(gq) && !has_tangent(gk), kTangentText);
    const bool first = gq.defined();
    const at::Tensor a = first ? gq : gk, b = first ? gk : at::Tensor();
    const auto r = at::GradMode::is_enabled()
                       ? apply(a, given(b), saved[0], given(saved[1]), t.interleaved, t.inverse, t.scale, t.offset)
                       : turn(a, b, saved[0], saved[1], t);
    out[first ? 0 : 1] = r[0];
    if (r.size() > 1) out[1] = r[1];
    return out;
  }
};

// rotary(q, k | None, inv_freq, interleaved, scale, positions | None, offset) -> q' or (q', k'); differentiable
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_rotary) REFUSE(PyExc_TypeError, "rotary takes 7 arguments, after bind_cache");
  const at::Tensor *q = tensor(a[0]), *k, *pos;
  if (!q || !optional(a[1], &k)) return nullptr;
  const at::Tensor* f = tensor(a[2]);
  if (!f || !optional(a[5], &pos)) return nullptr;
  const int interleaved = PyObject_IsTrue(a[3]);
  const double scale = PyFloat_AsDouble(a[4]);
  const long long offset = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (q->dim() != 4 || (k && k->dim() != 4)) REFUSE(PyExc_ValueError, "query and key must be (B, H, T, D)");
  if (q->scalar_type() != at::kBFloat16 && q->scalar_type() != at::kFloat)
    REFUSE(PyExc_TypeError, "apply_rotary takes bfloat16 or float32 tensors");
  if (k && k->scalar_type() != q->scalar_type()) REFUSE(PyExc_TypeError, "query and key must share a dtype");
  const int64_t B = q->size(0), T = q->size(2), D = q->size(3);
  if (k && (k->size(0) != B || k->size(2) != T || k->size(3) != D))
    REFUSE(PyExc_ValueError, "batch, length and head dim of query and key must match");
  if (!freq_ok(*f, D)) REFUSE(PyExc_ValueError, kFreqText);
  if (D > 1024 || !sizes_fit(*q) || (k && !sizes_fit(*k))) REFUSE(PyExc_ValueError, "head dim at most 1024, other sizes below 2^31");
  if (pos) {
    if (pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong)
      REFUSE(PyExc_TypeError, "positions must be int32 or int64");
    const bool row = pos->dim() == 1 && pos->size(0) == T;
    if (!row && !(pos->dim() == 2 && pos->size(1) == T && (pos->size(0) == B || pos->size(0) == 1)))
      REFUSE(PyExc_ValueError, "positions must be (T,), (1, T) or (B, T)");
  }
  if (has_tangent(*q) || (k && has_tangent(*k)) || has_tangent(*f)) REFUSE(PyExc_NotImplementedError, kTangentText);
  if (f->requires_grad() && at::GradMode::is_enabled())
    REFUSE(PyExc_NotImplementedError, "apply_rotary has no gradient of inv_freq: detach it");
  const at::Device dev = q->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "query and key must be GPU tensors");
  if ((k && k->device() != dev) || f->device() != dev || (pos && pos->device() != dev))
    REFUSE(PyExc_ValueError, "query, key, inv_freq and positions must be on one device");
  const at::Tensor none;
  const bool grad = at::GradMode::is_enabled() && (q->requires_grad() || (k && k->requires_grad()));
  const Turn t{interleaved != 0, false, scale, offset};
  const auto out = grad ? RotaryFunction::apply(*q, RotaryFunction::given(k ? *k : none), *f,
                                                RotaryFunction::given(pos ? *pos : none), t.interleaved, t.inverse, t.scale,
                                                t.offset)
                        : turn(*q, k ? *k : none, *f, pos ? *pos : none, t);
  if (!k) return THPVariable_Wrap(out[0]);
  return Py_BuildValue("NN", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
  END_HANDLE_TH_ERRORS
}

// The checks that append and decode share: the cache's tensors and tables.
// `v8`: e4m3 with scales; sets an exception and returns false where refused.
bool cache_ok(const at::Tensor& k, const at::Tensor& v, const at::Tensor* ks, const at::Tensor* vs, const at::Tensor* table,
              int64_t B, int64_t D) {
  PyObject* value = PyExc_ValueError;
  const char* bad = nullptr;
  const auto type = ks ? at::kFloat8_e4m3fn : at::kBFloat16;
  if (k.scalar_type() != type || v.scalar_type() != type) {
    value = PyExc_TypeError;
    bad = ks ? "the cache's key and value must be float8_e4m3fn" : "the cache's key and value must be bfloat16";
  } else if (k.dim() != 4 || k.sizes() != v.sizes()) {
    bad = "the cache's key and value must both be (num_pages, Hkv, page_size, D)";
  } else if (k.size(0) < 1 || k.size(1) < 1 || k.size(2) < FA_KV_RUN || k.size(2) % FA_KV_RUN) {
    bad = "page_size must be a multiple of 32, with at least one page and head";
  } else if (k.size(3) != D || (D != 32 && D != 64 && D != 128)) {
    bad = "the head dim must be 32, 64 or 128, the cache's and the tokens' the same";
  } else if (!k.is_contiguous() || !v.is_contiguous()) {
    bad = "the cache's tensors must be contiguous";
  } else if (!sizes_fit(k)) {
    bad = "the cache's sizes must be below 2^31";
  } else if (ks) {
    const at::IntArrayRef s = ks->sizes();
    if (ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat) {
      value = PyExc_TypeError;
      bad = "the cache's scales must be float32";
    } else if (s.size() != 3 || s[0] != k.size(0) || s[1] != k.size(1) || s[2] != k.size(2) / FA_KV_RUN ||
               vs->sizes() != s || !ks->is_contiguous() || !vs->is_contiguous()) {
      bad = "the cache's scales must be dense (num_pages, Hkv, page_size / 32)";
    }
  }
  if (!bad) {
    if (!table) {
      if (k.size(0) < B) bad = "without a page_table the cache has a page for every batch row";
    } else if (table->dim() != 2 || table->size(0) != B || table->size(1) < 1) {
      bad = "page_table must be (B, max_pages)";
    } else if (table->scalar_type() != at::kInt && table->scalar_type() != at::kLong) {
      value = PyExc_TypeError;
      bad = "page_table must be int32 or int64";
    }
  }
  if (bad) PyErr_SetString(value, bad);
  return !bad;
}
bool lens_ok(const at::Tensor* t, int64_t B, const char* shape_text) {
  if (!t) return true;
  if (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) {
    PyErr_SetString(PyExc_TypeError, "lengths must be int32 or int64");
    return false;
  }
  if (t->dim() != 1 || t->size(0) != B) {
    PyErr_SetString(PyExc_ValueError, shape_text);
    return false;
  }
  return true;
}

// append(k cache, v cache, k scale | None, v scale | None, key, value, kv_lens, table | None, new_lens | None,
//        inv_freq | None, interleaved, scale, query | None) -> (status, query' | None)
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || !g_append) REFUSE(PyExc_TypeError, "append takes 13 arguments, after bind_cache");
  const at::Tensor *kc = tensor(a[0]), *vc, *ks, *vs, *k, *v, *lens, *table, *fresh, *f, *q;
  if (!kc || !(vc = tensor(a[1])) || !optional(a[2], &ks) || !optional(a[3], &vs) || !(k = tensor(a[4])) ||
      !(v = tensor(a[5])) || !(lens = tensor(a[6])) || !optional(a[7], &table) || !optional(a[8], &fresh) ||
      !optional(a[9], &f) || !optional(a[12], &q))
    return nullptr;
  const int interleaved = PyObject_IsTrue(a[10]);
  const double scale = PyFloat_AsDouble(a[11]);
  if (PyErr_Occurred()) return nullptr;
  if (!ks != !vs) REFUSE(PyExc_TypeError, "an 8-bit cache has key and value scales");
  if (k->dim() != 4 || k->sizes() != v->sizes() || (q && q->dim() != 4))
    REFUSE(PyExc_ValueError, "key and value must both be (B, Hkv, T, D), query (B, Hq, T, D)");
  if (k->scalar_type() != at::kBFloat16 || v->scalar_type() != at::kBFloat16 || (q && q->scalar_type() != at::kBFloat16))
    REFUSE(PyExc_TypeError, "append_kv_cache takes bfloat16 query, key and value");
  const int64_t B = k->size(0), T = k->size(2), D = k->size(3);
  if (q && (q->size(0) != B || q->size(2) != T || q->size(3) != D))
    REFUSE(PyExc_ValueError, "batch, length and head dim of query and key must match");
  if (q && !f) REFUSE(PyExc_ValueError, "query is rotated with the keys: it needs rotary");
  if (!cache_ok(*kc, *vc, ks, vs, table, B, D)) return nullptr;
  if (k->size(1) != kc->size(1)) REFUSE(PyExc_ValueError, "head counts of key and cache do not match");
  if (!lens_ok(lens, B, "kv_lens must have one entry per batch row") ||
      !lens_ok(fresh, B, "new_lens must have one entry per batch row"))
    return nullptr;
  if (f && !freq_ok(*f, D)) REFUSE(PyExc_ValueError, kFreqText);
  if (f && f->size(0) % 8) REFUSE(PyExc_ValueError, "append_kv_cache takes a rotary_dim that is a multiple of 16");
  if (!sizes_fit(*k) || (q && !sizes_fit(*q))) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = kc->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "the cache must be on the GPU");
  if (vc->device() != dev || (ks && (ks->device() != dev || vs->device() != dev)) || k->device() != dev ||
      v->device() != dev || (q && q->device() != dev) || (f && f->device() != dev))
    REFUSE(PyExc_ValueError, "cache, tokens and inv_freq must be on one device");
  const c10::DeviceGuard guard(dev);
  at::Tensor out;
  if (q) out = at::empty(q->sizes(), q->options());
  int rc = FA_OK;
  if (k->numel() || (q && q->numel())) {
    const at::Tensor kk = rows_ok(*k) ? *k : dense16(*k), vv = rows_ok(*v) ? *v : dense16(*v);
    const at::Tensor ll = row_ints(*lens, dev);
    at::Tensor tt, nn, qq;
    fa_kv_append_call c{};
    c.abi_version = FA_ABI_VERSION;
    c.cache_dtype = ks ? FA_DTYPE_FP8_E4M3 : FA_DTYPE_BF16;
    c.B = static_cast<int32_t>(B);
    c.T = static_cast<int32_t>(T);
    c.D = static_cast<int32_t>(D);
    c.num_pages = static_cast<int32_t>(kc->size(0));
    c.page_size = static_cast<int32_t>(kc->size(2));
    c.max_pages = 1;
    c.key = strided(kk);
    c.value = strided(vv);
    if (q && q->numel()) {
      qq = rows_ok(*q) ? *q : dense16(*q);
      c.query = strided(qq);
      c.query_out = out.mutable_data_ptr();
    }
    c.k_cache = kc->mutable_data_ptr();
    c.v_cache = vc->mutable_data_ptr();
    if (ks) {
      c.k_scale = ks->mutable_data_ptr<float>();
      c.v_scale = vs->mutable_data_ptr<float>();
    }
    if (table) {
      tt = row_ints(*table, dev);
      c.page_table = tt.const_data_ptr<int32_t>();
      c.max_pages = static_cast<int32_t>(tt.size(1));
    }
    c.kv_lens = ll.const_data_ptr<int32_t>();
    if (fresh) {
      nn = row_ints(*fresh, dev);
      c.new_lens = nn.const_data_ptr<int32_t>();
    }
    if (f) {
      c.rotary.inv_freq = f->const_data_ptr<double>();
      c.rotary.pairs = static_cast<int32_t>(f->size(0));
      c.rotary.interleaved = interleaved;
      c.rotary.scale = static_cast<float>(scale);
    }
    rc = g_append(&c, stream_of(dev));
    // written through raw pointers: autograd learns of it here (inference tensors have no version)
    for (const at::Tensor* t : {kc, vc, ks, vs})
      if (rc == FA_OK && t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  if (!q) return Py_BuildValue("iO", rc, Py_None);
  return Py_BuildValue("iN", rc, THPVariable_Wrap(out));
  END_HANDLE_TH_ERRORS
}

// decode(q, k, v, k scale, v scale, kv_lens | None, table | None, q_lens | None, left, right, slopes | None,
//        softcap, scale, gqa, kv_len | None) -> (status, o, lse)
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15 || !g_decode) REFUSE(PyExc_TypeError, "decode takes 15 arguments, after bind_cache");
  const at::Tensor *q = tensor(a[0]), *k, *v, *ks, *vs, *lens, *table, *ql, *slopes;
  if (!q || !(k = tensor(a[1])) || !(v = tensor(a[2])) || !(ks = tensor(a[3])) || !(vs = tensor(a[4])) ||
      !optional(a[5], &lens) || !optional(a[6], &table) || !optional(a[7], &ql) || !optional(a[10], &slopes))
    return nullptr;
  const int64_t left = std::min<int64_t>(PyLong_AsLong(a[8]), kMaxSize), right = std::min<int64_t>(PyLong_AsLong(a[9]), kMaxSize);
  const double softcap = PyFloat_AsDouble(a[11]), scale = PyFloat_AsDouble(a[12]);
  const int gqa = PyObject_IsTrue(a[13]);
  const int64_t kv_len = a[14] == Py_None ? 0 : PyLong_AsLong(a[14]);
  if (PyErr_Occurred()) return nullptr;
  if (q->dim() != 4) REFUSE(PyExc_ValueError, "query must be (B, Hq, Sq, D)");
  if (q->scalar_type() != at::kBFloat16) REFUSE(PyExc_TypeError, "flex_decode_fp8 takes bfloat16 queries");
  const int64_t B = q->size(0), Hq = q->size(1), Sq = q->size(2), D = q->size(3);
  if (!cache_ok(*k, *v, ks, vs, table, B, D)) return nullptr;
  const int64_t Hkv = k->size(1);
  if (Hq != Hkv && !gqa) REFUSE(PyExc_ValueError, "query and cache head counts differ: pass enable_gqa=True for grouped-query attention");
  if (Hq % Hkv) REFUSE(PyExc_ValueError, "number of q heads must be a multiple of the number of kv heads");
  if (!lens_ok(lens, B, "kv_lens must have one entry per batch row") ||
      !lens_ok(ql, B, "query_lens must have one entry per batch row"))
    return nullptr;
  if (slopes && (slopes->scalar_type() != at::kFloat || slopes->dim() != 1 || slopes->size(0) != Hq))
    REFUSE(PyExc_ValueError, "ALiBi needs one slope per q head");
  if (!(scale >= 0.0) || !(softcap >= 0.0)) REFUSE(PyExc_ValueError, "scale must be positive");
  // (0: the default scale, no soft-cap: nothing else may become it)
  auto fits = [](double x) { return x == 0.0 || (x >= FLT_MIN && x <= FLT_MAX); };
  if (!fits(scale) || !fits(softcap)) REFUSE(PyExc_ValueError, "scale and soft-cap must be normal float32 numbers");
  const int64_t pages = table ? table->size(1) : 1, all = pages * k->size(2);
  if (a[14] != Py_None && (kv_len < 1 || kv_len > all)) REFUSE(PyExc_ValueError, "kv_len must be in [1, max_pages * page_size]");
  const int64_t cap = kv_len ? kv_len : all;
  if (!sizes_fit(*q) || pages > kMaxSize || cap > kMaxSize) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = q->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "query and cache must be on the GPU");
  if (k->device() != dev || v->device() != dev || ks->device() != dev || vs->device() != dev ||
      (slopes && slopes->device() != dev))
    REFUSE(PyExc_ValueError, "query and cache must be on one device");
  const c10::DeviceGuard guard(dev);
  const at::Tensor qq = rows_ok(*q) ? *q : dense16(*q);
  at::Tensor o = at::empty(qq.sizes(), qq.options());
  at::Tensor lse = at::empty(qq.sizes().slice(0, 3), qq.options().dtype(at::kFloat));
  int rc = FA_OK;
  if (qq.numel()) {
    at::Tensor ll, tt, qn;
    fa_params p{};
    p.abi_version = FA_ABI_VERSION;
    p.dtype = FA_DTYPE_FP8_E4M3;
    p.B = static_cast<int32_t>(B);
    p.Hq = static_cast<int32_t>(Hq);
    p.Hkv = static_cast<int32_t>(Hkv);
    p.Sq = static_cast<int32_t>(Sq);
    p.Skv = static_cast<int32_t>(cap);
    p.D = static_cast<int32_t>(D);
    p.scale = static_cast<float>(scale);
    p.window_left = static_cast<int32_t>(left);
    p.window_right = static_cast<int32_t>(right);
    p.alibi_slopes = slopes ? slopes->const_data_ptr<float>() : nullptr;
    p.softcap = static_cast<float>(softcap);
    fa_fp8_cache c{};
    c.k = k->const_data_ptr();
    c.v = v->const_data_ptr();
    c.k_scale = ks->const_data_ptr<float>();
    c.v_scale = vs->const_data_ptr<float>();
    c.page_size = static_cast<int32_t>(k->size(2));
    c.num_pages = static_cast<int32_t>(k->size(0));
    c.max_pages = static_cast<int32_t>(pages);
    if (table) c.page_table = (tt = row_ints(*table, dev)).const_data_ptr<int32_t>();
    if (lens) c.kv_lens = (ll = row_ints(*lens, dev)).const_data_ptr<int32_t>();
    if (ql) c.q_lens = (qn = row_ints(*ql, dev)).const_data_ptr<int32_t>();
    const size_t bytes = g_decode_ws(&p, &c);
    at::Tensor ws;
    if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, qq.options().dtype(at::kByte));
    const fa_strided qs = strided(qq);
    void *op = o.mutable_data_ptr(), *wp = bytes ? ws.mutable_data_ptr() : nullptr;
    float* lp = lse.mutable_data_ptr<float>();
    rc = g_decode(&p, &c, &qs, op, lp, wp, bytes, stream_of(dev));
  }
  return Py_BuildValue("iNN", rc, THPVariable_Wrap(o), THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------- prompts, latent vectors and pages ----
decltype(&fa_prefill) g_prefill = nullptr;
decltype(&fa_prefill_workspace_bytes) g_prefill_ws = nullptr;
decltype(&fa_latent_append) g_latent_append = nullptr;
decltype(&fa_latent_decode) g_latent = nullptr;
decltype(&fa_latent_decode_workspace_bytes) g_latent_ws = nullptr;
decltype(&fa_copy_pages) g_copy_pages = nullptr;
decltype(&fa_fork_rows) g_fork = nullptr;
decltype(&fa_fork_rows_workspace_bytes) g_fork_ws = nullptr;
decltype(&fa_compact_pages) g_compact = nullptr;
decltype(&fa_compact_pages_workspace_bytes) g_compact_ws = nullptr;

// bind_serve(fa_prefill, fa_prefill_workspace_bytes, fa_latent_append, fa_latent_decode,
//            fa_latent_decode_workspace_bytes, fa_copy_pages, fa_fork_rows, fa_fork_rows_workspace_bytes,
//            fa_compact_pages, fa_compact_pages_workspace_bytes)
PyObject* py_bind_serve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "bind_serve takes 10 addresses");
    return nullptr;
  }
  g_prefill = reinterpret_cast<decltype(g_prefill)>(address(a[0]));
  g_prefill_ws = reinterpret_cast<decltype(g_prefill_ws)>(address(a[1]));
  g_latent_append = reinterpret_cast<decltype(g_latent_append)>(address(a[2]));
  g_latent = reinterpret_cast<decltype(g_latent)>(address(a[3]));
  g_latent_ws = reinterpret_cast<decltype(g_latent_ws)>(address(a[4]));
  g_copy_pages = reinterpret_cast<decltype(g_copy_pages)>(address(a[5]));
  g_fork = reinterpret_cast<decltype(g_fork)>(address(a[6]));
  g_fork_ws = reinterpret_cast<decltype(g_fork_ws)>(address(a[7]));
  g_compact = reinterpret_cast<decltype(g_compact)>(address(a[8]));
  g_compact_ws = reinterpret_cast<decltype(g_compact_ws)>(address(a[9]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// written through raw pointers: autograd learns of it here (inference tensors have no version)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int64_t window(PyObject* x) { return std::max<int64_t>(std::min<int64_t>(PyLong_AsLong(x), kMaxSize), -1); }

// prefill(q, k, v, k scale | None, v scale | None, kv_lens | None, table | None, q_lens | None, q_starts | None, left, right,
//         slopes | None, softcap, scale, gqa, kv_len | None) -> (status, o, lse)
PyObject* py_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 16 || !g_prefill) REFUSE(PyExc_TypeError, "prefill takes 16 arguments, after bind_serve");
  const at::Tensor *q = tensor(a[0]), *k, *v, *ks, *vs, *lens, *table, *ql, *starts, *slopes;
  if (!q || !(k = tensor(a[1])) || !(v = tensor(a[2])) || !optional(a[3], &ks) || !optional(a[4], &vs) ||
      !optional(a[5], &lens) || !optional(a[6], &table) || !optional(a[7], &ql) || !optional(a[8], &starts) ||
      !optional(a[11], &slopes))
    return nullptr;
  const int64_t left = window(a[9]), right = window(a[10]);
  const double softcap = PyFloat_AsDouble(a[12]), scale = PyFloat_AsDouble(a[13]);
  const int gqa = PyObject_IsTrue(a[14]);
  const int64_t kv_len = a[15] == Py_None ? 0 : PyLong_AsLong(a[15]);
  if (PyErr_Occurred()) return nullptr;
  if (!ks != !vs) REFUSE(PyExc_TypeError, "an 8-bit cache has key and value scales");
  if (q->dim() != 4) REFUSE(PyExc_ValueError, "query must be (B, Hq, T, D), packed (1, Hq, tokens, D)");
  if (q->scalar_type() != at::kBFloat16) REFUSE(PyExc_TypeError, "flex_prefill takes bfloat16 queries");
  if (starts) {
    if (ql) REFUSE(PyExc_ValueError, "pass query_lens or query_starts, not both");
    if (starts->scalar_type() != at::kInt && starts->scalar_type() != at::kLong)
      REFUSE(PyExc_TypeError, "query_starts must be int32 or int64");
    if (q->size(0) != 1 || starts->dim() != 1 || starts->size(0) < 2 || starts->size(0) > kMaxSize)
      REFUSE(PyExc_ValueError, "packed queries are (1, Hq, tokens, D), with query_starts (B + 1,) of at least one row");
  }
  const int64_t B = starts ? starts->size(0) - 1 : q->size(0), Hq = q->size(1), T = q->size(2), D = q->size(3);
  if (!cache_ok(*k, *v, ks, vs, table, B, D)) return nullptr;
  const int64_t Hkv = k->size(1);
  if (Hq != Hkv && !gqa) REFUSE(PyExc_ValueError, "query and cache head counts differ: pass enable_gqa=True for grouped-query attention");
  if (Hq % Hkv) REFUSE(PyExc_ValueError, "number of q heads must be a multiple of the number of kv heads");
  if (!lens_ok(lens, B, "kv_lens must have one entry per batch row") ||
      !lens_ok(ql, B, "query_lens must have one entry per batch row"))
    return nullptr;
  if (slopes && (slopes->scalar_type() != at::kFloat || slopes->dim() != 1 || slopes->size(0) != Hq || !slopes->is_contiguous()))
    REFUSE(PyExc_ValueError, "ALiBi needs one slope per q head");
  if (!(scale >= 0.0) || !(softcap >= 0.0)) REFUSE(PyExc_ValueError, "scale must be positive");
  auto fits = [](double x) { return x == 0.0 || (x >= FLT_MIN && x <= FLT_MAX); };  // (0: the default, none)
  if (!fits(scale) || !fits(softcap)) REFUSE(PyExc_ValueError, "scale and soft-cap must be normal float32 numbers");
  const int64_t pages = table ? table->size(1) : 1, all = pages * k->size(2);
  if (a[15] != Py_None && (kv_len < 1 || kv_len > all)) REFUSE(PyExc_ValueError, "kv_len must be in [1, max_pages * page_size]");
  const int64_t cap = kv_len ? kv_len : all;
  if (!sizes_fit(*q) || pages > kMaxSize || cap > kMaxSize) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = q->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "query and cache must be on the GPU");
  if (k->device() != dev || v->device() != dev || (ks && (ks->device() != dev || vs->device() != dev)) ||
      (slopes && slopes->device() != dev))
    REFUSE(PyExc_ValueError, "query and cache must be on one device");
  const c10::DeviceGuard guard(dev);
  const at::Tensor qq = rows_ok(*q) ? *q : dense16(*q);
  // laid out as the query is: what a projection wrote as (tokens, heads, D) comes back so for the next one
  at::Tensor o = qq.is_non_overlapping_and_dense() ? at::empty_strided(qq.sizes(), qq.strides(), qq.options())
                                                   : at::empty(qq.sizes(), qq.options());
  at::Tensor lse = at::empty(qq.sizes().slice(0, 3), qq.options().dtype(at::kFloat));
  int rc = FA_OK;
  if (qq.numel()) {
    at::Tensor ll, tt, qn, ss;
    fa_prefill_call c{};
    c.abi_version = FA_ABI_VERSION;
    c.cache_dtype = ks ? FA_DTYPE_FP8_E4M3 : FA_DTYPE_BF16;
    c.B = static_cast<int32_t>(B);
    c.Hkv = static_cast<int32_t>(Hkv);
    c.T = static_cast<int32_t>(T);
    c.D = static_cast<int32_t>(D);
    c.page_size = static_cast<int32_t>(k->size(2));
    c.num_pages = static_cast<int32_t>(k->size(0));
    c.max_pages = static_cast<int32_t>(pages);
    c.kv_len = static_cast<int32_t>(cap);
    c.window_left = static_cast<int32_t>(left);
    c.window_right = static_cast<int32_t>(right);
    c.scale = static_cast<float>(scale);
    c.softcap = static_cast<float>(softcap);
    c.alibi_slopes = slopes ? slopes->const_data_ptr<float>() : nullptr;
    c.query = strided(qq);
    c.out = strided(o);
    c.out.data = o.mutable_data_ptr();
    c.lse = lse.mutable_data_ptr<float>();
    c.k_cache = k->const_data_ptr();
    c.v_cache = v->const_data_ptr();
    if (ks) {
      c.k_scale = ks->const_data_ptr<float>();
      c.v_scale = vs->const_data_ptr<float>();
    }
    if (table) c.page_table = (tt = row_ints(*table, dev)).const_data_ptr<int32_t>();
    if (lens) c.kv_lens = (ll = row_ints(*lens, dev)).const_data_ptr<int32_t>();
    if (ql) c.q_lens = (qn = row_ints(*ql, dev)).const_data_ptr<int32_t>();
    if (starts) c.q_starts = (ss = row_ints(*starts, dev)).const_data_ptr<int32_t>();
    const size_t bytes = g_prefill_ws(&c);
    at::Tensor ws;
    if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, qq.options().dtype(at::kByte));
    rc = g_prefill(&c, bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(dev));
  }
  return Py_BuildValue("iNN", rc, THPVariable_Wrap(o), THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// A cache of latent vectors and the table of its rows.
bool latent_ok(const at::Tensor& c, int64_t L, const at::Tensor* table, int64_t B) {
  PyObject* value = PyExc_ValueError;
  const char* bad = nullptr;
  const int64_t R = c.dim() == 3 ? c.size(2) - L : 0;
  if (c.scalar_type() != at::kBFloat16) {
    value = PyExc_TypeError;
    bad = "the cache must be bfloat16";
  } else if (c.dim() != 3 || c.size(0) < 1 || c.size(1) < FA_KV_RUN || c.size(1) % FA_KV_RUN) {
    bad = "the cache must be (num_pages, page_size, latent_dim + rope_dim), page_size a multiple of 32";
  } else if ((L != 128 && L != 256 && L != 512) || (R != 32 && R != 64)) {
    bad = "latent_dim must be 128, 256 or 512, rope_dim 32 or 64";
  } else if (!c.is_contiguous()) {
    bad = "the cache must be contiguous";
  } else if (!sizes_fit(c)) {
    bad = "the cache's sizes must be below 2^31";
  } else if (!table) {
    if (c.size(0) < B) bad = "without a page_table the cache has a page for every batch row";
  } else if (table->dim() != 2 || table->size(0) != B || table->size(1) < 1) {
    bad = "page_table must be (B, max_pages)";
  } else if (table->scalar_type() != at::kInt && table->scalar_type() != at::kLong) {
    value = PyExc_TypeError;
    bad = "page_table must be int32 or int64";
  }
  if (bad) PyErr_SetString(value, bad);
  return !bad;
}

// latent_append(cache, latent_dim, latent, key rope, kv_lens, table | None, new_lens | None, inv_freq | None, interleaved,
//               scale, query rope | None) -> (status, query rope' | None)
PyObject* py_latent_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !g_latent_append) REFUSE(PyExc_TypeError, "latent_append takes 11 arguments, after bind_serve");
  const at::Tensor *kc = tensor(a[0]), *x, *k, *lens, *table, *fresh, *f, *q;
  const int64_t L = PyLong_AsLong(a[1]);
  if (!kc || !(x = tensor(a[2])) || !(k = tensor(a[3])) || !(lens = tensor(a[4])) || !optional(a[5], &table) ||
      !optional(a[6], &fresh) || !optional(a[7], &f) || !optional(a[10], &q))
    return nullptr;
  const int interleaved = PyObject_IsTrue(a[8]);
  const double scale = PyFloat_AsDouble(a[9]);
  if (PyErr_Occurred()) return nullptr;
  if (x->dim() != 3 || k->dim() != 3 || (q && q->dim() != 4))
    REFUSE(PyExc_ValueError, "latent and key_rope must be (B, T, dim), query_rope (B, H, T, rope_dim)");
  if (x->scalar_type() != at::kBFloat16 || k->scalar_type() != at::kBFloat16 || (q && q->scalar_type() != at::kBFloat16))
    REFUSE(PyExc_TypeError, "append_latent_cache takes bfloat16 latent, key_rope and query_rope");
  const int64_t B = x->size(0), T = x->size(1);
  if (!latent_ok(*kc, L, table, B)) return nullptr;
  const int64_t R = kc->size(2) - L;
  if (x->size(2) != L || k->size(0) != B || k->size(1) != T || k->size(2) != R ||
      (q && (q->size(0) != B || q->size(2) != T || q->size(3) != R)))
    REFUSE(PyExc_ValueError, "batch, length and dims of latent, key_rope, query_rope and cache must match");
  if (q && !f) REFUSE(PyExc_ValueError, "query_rope is rotated with the keys: it needs rotary");
  if (!lens_ok(lens, B, "kv_lens must have one entry per batch row") ||
      !lens_ok(fresh, B, "new_lens must have one entry per batch row"))
    return nullptr;
  if (f && !freq_ok(*f, R)) REFUSE(PyExc_ValueError, "inv_freq must be a dense float64 vector with at most rope_dim / 2 entries");
  if (f && f->size(0) % 8) REFUSE(PyExc_ValueError, "append_latent_cache takes a rotary_dim that is a multiple of 16");
  if (!sizes_fit(*x) || (q && !sizes_fit(*q))) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = kc->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "the cache must be on the GPU");
  if (x->device() != dev || k->device() != dev || (q && q->device() != dev) || (f && f->device() != dev))
    REFUSE(PyExc_ValueError, "cache, tokens and inv_freq must be on one device");
  const c10::DeviceGuard guard(dev);
  at::Tensor out;
  if (q) out = at::empty(q->sizes(), q->options());
  int rc = FA_OK;
  if (x->numel()) {
    auto rows = [](const at::Tensor& t) {
      const at::Tensor u = t.unsqueeze(1);
      return rows_ok(u) ? u : dense16(u);
    };
    const at::Tensor xx = rows(*x), kk = rows(*k), ll = row_ints(*lens, dev);
    at::Tensor tt, nn, qq;
    fa_latent_append_call c{};
    c.abi_version = FA_ABI_VERSION;
    c.B = static_cast<int32_t>(B);
    c.T = static_cast<int32_t>(T);
    c.latent_dim = static_cast<int32_t>(L);
    c.rope_dim = static_cast<int32_t>(R);
    c.num_pages = static_cast<int32_t>(kc->size(0));
    c.page_size = static_cast<int32_t>(kc->size(1));
    c.max_pages = 1;
    c.latent = strided(xx);
    c.rope = strided(kk);
    if (q && q->numel()) {
      qq = rows_ok(*q) ? *q : dense16(*q);
      c.query = strided(qq);
      c.query_out = out.mutable_data_ptr();
    }
    c.cache = kc->mutable_data_ptr();
    if (table) {
      tt = row_ints(*table, dev);
      c.page_table = tt.const_data_ptr<int32_t>();
      c.max_pages = static_cast<int32_t>(tt.size(1));
    }
    c.kv_lens = ll.const_data_ptr<int32_t>();
    if (fresh) c.new_lens = (nn = row_ints(*fresh, dev)).const_data_ptr<int32_t>();
    if (f) {
      c.rotary.inv_freq = f->const_data_ptr<double>();
      c.rotary.pairs = static_cast<int32_t>(f->size(0));
      c.rotary.interleaved = interleaved;
      c.rotary.scale = static_cast<float>(scale);
    }
    rc = g_latent_append(&c, stream_of(dev));
    if (rc == FA_OK) written(*kc);
  }
  if (!q) return Py_BuildValue("iO", rc, Py_None);
  return Py_BuildValue("iN", rc, THPVariable_Wrap(out));
  END_HANDLE_TH_ERRORS
}

// latent_decode(query, query rope, cache, latent_dim, scale, kv_lens | None, table | None, q_lens | None, left, right,
//               kv_len | None) -> (status, o, lse)
PyObject* py_latent_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !g_latent) REFUSE(PyExc_TypeError, "latent_decode takes 11 arguments, after bind_serve");
  const at::Tensor *q = tensor(a[0]), *qr, *kc, *lens, *table, *ql;
  if (!q || !(qr = tensor(a[1])) || !(kc = tensor(a[2])) || !optional(a[5], &lens) || !optional(a[6], &table) ||
      !optional(a[7], &ql))
    return nullptr;
  const int64_t L = PyLong_AsLong(a[3]);
  const double scale = PyFloat_AsDouble(a[4]);
  const int64_t left = window(a[8]), right = window(a[9]);
  const int64_t kv_len = a[10] == Py_None ? 0 : PyLong_AsLong(a[10]);
  if (PyErr_Occurred()) return nullptr;
  if (q->dim() != 4 || qr->dim() != 4) REFUSE(PyExc_ValueError, "query must be (B, H, T, latent_dim), query_rope (B, H, T, rope_dim)");
  if (q->scalar_type() != at::kBFloat16 || qr->scalar_type() != at::kBFloat16)
    REFUSE(PyExc_TypeError, "flex_decode_latent takes bfloat16 query and query_rope");
  const int64_t B = q->size(0), H = q->size(1), T = q->size(2);
  if (!latent_ok(*kc, L, table, B)) return nullptr;
  if (q->size(3) != L || qr->size(0) != B || qr->size(1) != H || qr->size(2) != T || qr->size(3) != kc->size(2) - L)
    REFUSE(PyExc_ValueError, "sizes of query, query_rope and cache do not match");
  if (!lens_ok(lens, B, "kv_lens must have one entry per batch row") ||
      !lens_ok(ql, B, "query_lens must have one entry per batch row"))
    return nullptr;
  if (!(scale >= FLT_MIN && scale <= FLT_MAX)) REFUSE(PyExc_ValueError, "scale must be a positive normal float32 number");
  const int64_t pages = table ? table->size(1) : 1, all = pages * kc->size(1);
  if (a[10] != Py_None && (kv_len < 1 || kv_len > all)) REFUSE(PyExc_ValueError, "kv_len must be in [1, max_pages * page_size]");
  const int64_t cap = kv_len ? kv_len : all;
  if (!sizes_fit(*q) || pages > kMaxSize || cap > kMaxSize) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = q->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "query and cache must be on the GPU");
  if (qr->device() != dev || kc->device() != dev) REFUSE(PyExc_ValueError, "query and cache must be on one device");
  const c10::DeviceGuard guard(dev);
  at::Tensor o = at::empty(q->sizes(), q->options());
  at::Tensor lse = at::empty(q->sizes().slice(0, 3), q->options().dtype(at::kFloat));
  int rc = FA_OK;
  if (q->numel()) {
    const at::Tensor qq = rows_ok(*q) ? *q : dense16(*q), rr = rows_ok(*qr) ? *qr : dense16(*qr);
    at::Tensor ll, tt, qn;
    fa_latent_call c{};
    c.abi_version = FA_ABI_VERSION;
    c.B = static_cast<int32_t>(B);
    c.T = static_cast<int32_t>(T);
    c.latent_dim = static_cast<int32_t>(L);
    c.rope_dim = static_cast<int32_t>(kc->size(2) - L);
    c.page_size = static_cast<int32_t>(kc->size(1));
    c.num_pages = static_cast<int32_t>(kc->size(0));
    c.max_pages = static_cast<int32_t>(pages);
    c.kv_len = static_cast<int32_t>(cap);
    c.window_left = static_cast<int32_t>(left);
    c.window_right = static_cast<int32_t>(right);
    c.scale = static_cast<float>(scale);
    c.query = strided(qq);
    c.query_rope = strided(rr);
    c.o = o.mutable_data_ptr();
    c.lse = lse.mutable_data_ptr<float>();
    c.cache = kc->const_data_ptr();
    if (table) c.page_table = (tt = row_ints(*table, dev)).const_data_ptr<int32_t>();
    if (lens) c.kv_lens = (ll = row_ints(*lens, dev)).const_data_ptr<int32_t>();
    if (ql) c.q_lens = (qn = row_ints(*ql, dev)).const_data_ptr<int32_t>();
    const size_t bytes = g_latent_ws(&c);
    at::Tensor ws;
    if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, q->options().dtype(at::kByte));
    rc = g_latent(&c, bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(dev));
  }
  return Py_BuildValue("iNN", rc, THPVariable_Wrap(o), THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// The tensors of a call on pages: those of one cache or of a list of them, dense, of as many pages each, on one device.
// (Here and not in Python: the 32 tensors of eight layers took 9 us there.)
struct Paged {
  std::vector<const at::Tensor*> t;
  std::vector<fa_paged_tensor> p;
  int64_t page_size = 0;

  bool refuse(PyObject* type, const char* text) {
    PyErr_SetString(type, text);
    return false;
  }
  bool add(const at::Tensor& x, int64_t dims, int at) {  // at: the dimension of the page size (0: none)
    if (x.dim() != dims) return refuse(PyExc_ValueError, "key and value are (num_pages, Hkv, page_size, D), latent vectors (num_pages, page_size, dim)");
    if (x.numel() == 0 || !x.is_contiguous()) return refuse(PyExc_ValueError, "a cache's tensors must be dense and not empty");
    if (!sizes_fit(x)) return refuse(PyExc_ValueError, "sizes must be below 2^31");
    if (!t.empty() && x.size(0) != t.front()->size(0)) return refuse(PyExc_ValueError, "the caches must have as many pages each");
    if (!t.empty() && x.device() != t.front()->device()) return refuse(PyExc_ValueError, "the caches must be on one device");
    if (at) {
      if (page_size && x.size(at) != page_size) return refuse(PyExc_ValueError, "the caches must have one page size");
      page_size = x.size(at);
    }
    t.push_back(&x);
    p.push_back({const_cast<void*>(x.const_data_ptr()), x.numel() / x.size(0) * x.element_size()});
    return true;
  }
  static bool sequence(PyObject* x) { return PyTuple_Check(x) || PyList_Check(x); }
  // (key, value), (key, value, key scale, value scale) or (latent data, its length)
  bool cache(PyObject* c) {
    const char* const text = "a cache is an Fp8KVCache, a LatentKVCache or a (key, value) pair of tensors";
    if (!sequence(c)) return refuse(PyExc_TypeError, text);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(c);
    PyObject** x = PySequence_Fast_ITEMS(c);
    if (n == 2 && THPVariable_Check(x[0]) && PyLong_Check(x[1])) return add(THPVariable_Unpack(x[0]), 3, 1);
    if (n != 2 && n != 4) return refuse(PyExc_TypeError, text);
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_Check(x[i])) return refuse(PyExc_TypeError, text);
      if (!add(THPVariable_Unpack(x[i]), i < 2 ? 4 : 3, i < 2 ? 2 : 0)) return false;
    }
    return true;
  }
  bool read(PyObject* caches) {
    if (!sequence(caches) || PySequence_Fast_GET_SIZE(caches) < 1)
      return refuse(PyExc_TypeError, "caches must be a cache or a list of caches");
    PyObject** x = PySequence_Fast_ITEMS(caches);
    if (THPVariable_Check(x[0])) return cache(caches);
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(caches); ++i)
      if (!cache(x[i])) return false;
    return true;
  }
};

// copy_pages(caches, src, dst) -> status
PyObject* py_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !g_copy_pages) REFUSE(PyExc_TypeError, "copy_pages takes 3 arguments, after bind_serve");
  Paged c;
  if (!c.read(a[0])) return nullptr;
  const at::Tensor *src = tensor(a[1]), *dst;
  if (!src || !(dst = tensor(a[2]))) return nullptr;
  for (const at::Tensor* x : {src, dst}) {
    if (x->scalar_type() != at::kInt && x->scalar_type() != at::kLong) REFUSE(PyExc_TypeError, "page ids must be int32 or int64");
    if (x->dim() != 1 || x->size(0) != src->size(0) || x->size(0) > kMaxSize)
      REFUSE(PyExc_ValueError, "src and dst must be vectors of one length");
  }
  const at::Device dev = c.t[0]->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "the caches must be on the GPU");
  int rc = FA_OK;
  if (src->size(0)) {
    const c10::DeviceGuard guard(dev);
    const at::Tensor s = row_ints(*src, dev), d = row_ints(*dst, dev);
    rc = g_copy_pages(c.p.data(), static_cast<int32_t>(c.p.size()), static_cast<int32_t>(c.t[0]->size(0)),
                      s.const_data_ptr<int32_t>(), d.const_data_ptr<int32_t>(), static_cast<int32_t>(s.size(0)), stream_of(dev));
    if (rc == FA_OK)
      for (const at::Tensor* x : c.t) written(*x);
  }
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// page_plan(fork, caches, table, kv_lens, parents | None, room | None, room_all, keep | None)
//   -> (status, table', lens' | None, count)
PyObject* py_page_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !g_fork) REFUSE(PyExc_TypeError, "page_plan takes 8 arguments, after bind_serve");
  const bool fork = PyObject_IsTrue(a[0]);
  Paged k;
  if (!k.read(a[1])) return nullptr;
  const std::vector<const at::Tensor*>& t = k.t;
  const int64_t page_size = k.page_size, room_all = PyLong_AsLong(a[6]);
  const at::Tensor *table = tensor(a[2]), *lens, *parents, *room, *keep;
  if (!table || !(lens = tensor(a[3])) || !optional(a[4], &parents) || !optional(a[5], &room) || !optional(a[7], &keep)) return nullptr;
  if (PyErr_Occurred()) return nullptr;
  const int64_t pages = t[0]->size(0);
  if (table->scalar_type() != at::kInt && table->scalar_type() != at::kLong)
    REFUSE(PyExc_TypeError, "page_table must be int32 or int64");
  if (table->dim() != 2 || table->size(0) < 1 || table->size(1) < 1) REFUSE(PyExc_ValueError, "page_table must be (B, max_pages)");
  const int64_t B = table->size(0), M = table->size(1);
  if (!lens_ok(lens, B, "kv_lens must have one entry per row of the page table")) return nullptr;
  if (parents && ((parents->scalar_type() != at::kInt && parents->scalar_type() != at::kLong)))
    REFUSE(PyExc_TypeError, "parents must be int32 or int64");
  if (parents && (parents->dim() != 1 || parents->size(0) < 1)) REFUSE(PyExc_ValueError, "parents must be a vector of at least one row");
  const int64_t N = parents ? parents->size(0) : B;
  if (!lens_ok(room, N, "room must be a number or have one entry per row")) return nullptr;
  if (room_all < 0 || room_all > kMaxSize) REFUSE(PyExc_ValueError, "room must not be negative, and below 2^31");
  if (keep && keep->scalar_type() != at::kBool) REFUSE(PyExc_TypeError, "keep must be a bool tensor");
  if (keep && (keep->dim() != 1 || keep->size(0) != pages)) REFUSE(PyExc_ValueError, "keep must have one entry per page");
  if (!sizes_fit(*table) || N > kMaxSize) REFUSE(PyExc_ValueError, "sizes must be below 2^31");
  const at::Device dev = t[0]->device();
  if (!dev.is_cuda()) REFUSE(PyExc_ValueError, "the caches must be on the GPU");
  if (keep && keep->device() != dev) REFUSE(PyExc_ValueError, "keep must be on the caches' device");
  const c10::DeviceGuard guard(dev);
  const at::Tensor tt = row_ints(*table, dev), ll = row_ints(*lens, dev);
  at::Tensor pp, rr, kk;
  fa_page_plan_call c{};
  c.abi_version = FA_ABI_VERSION;
  c.B = static_cast<int32_t>(B);
  c.N = static_cast<int32_t>(N);
  c.max_pages = static_cast<int32_t>(M);
  c.page_size = static_cast<int32_t>(page_size);
  c.num_pages = static_cast<int32_t>(pages);
  c.room_all = static_cast<int32_t>(room_all);
  c.page_table = tt.const_data_ptr<int32_t>();
  c.kv_lens = ll.const_data_ptr<int32_t>();
  if (parents) c.parents = (pp = row_ints(*parents, dev)).const_data_ptr<int32_t>();
  if (room) c.room = (rr = row_ints(*room, dev)).const_data_ptr<int32_t>();
  if (keep) c.keep = static_cast<const uint8_t*>((kk = keep->contiguous()).const_data_ptr());
  const auto ints = tt.options();
  at::Tensor out = at::empty({N, M}, ints), count = at::empty({}, ints), olens;
  c.out_table = out.mutable_data_ptr<int32_t>();
  c.out_count = count.mutable_data_ptr<int32_t>();
  if (fork) c.out_lens = (olens = at::empty({N}, ints)).mutable_data_ptr<int32_t>();
  c.tensors = k.p.data();
  c.tensor_count = static_cast<int32_t>(k.p.size());
  const size_t bytes = (fork ? g_fork_ws : g_compact_ws)(&c);
  at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(bytes, 16))}, ints.dtype(at::kByte));
  const int rc = (fork ? g_fork : g_compact)(&c, ws.mutable_data_ptr(), bytes, stream_of(dev));
  if (rc == FA_OK)
    for (const at::Tensor* x : t) written(*x);
  if (!fork) return Py_BuildValue("iNON", rc, THPVariable_Wrap(out), Py_None, THPVariable_Wrap(count));
  return Py_BuildValue("iNNN", rc, THPVariable_Wrap(out), THPVariable_Wrap(olens), THPVariable_Wrap(count));
  END_HANDLE_TH_ERRORS
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f));
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_bind)), METH_FASTCALL, nullptr},
    {"fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_fwd)), METH_FASTCALL, nullptr},
    {"bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_bwd)), METH_FASTCALL, nullptr},
    {"bind_cache", fast(py_bind_cache), METH_FASTCALL, nullptr},
    {"rotary", fast(py_rotary), METH_FASTCALL, nullptr},
    {"append", fast(py_append), METH_FASTCALL, nullptr},
    {"decode", fast(py_decode), METH_FASTCALL, nullptr},
    {"bind_serve", fast(py_bind_serve), METH_FASTCALL, nullptr},
    {"prefill", fast(py_prefill), METH_FASTCALL, nullptr},
    {"latent_append", fast(py_latent_append), METH_FASTCALL, nullptr},
    {"latent_decode", fast(py_latent_decode), METH_FASTCALL, nullptr},
    {"copy_pages", fast(py_copy_pages), METH_FASTCALL, nullptr},
    {"page_plan", fast(py_page_plan), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch(void) { return PyModule_Create(&module); }
