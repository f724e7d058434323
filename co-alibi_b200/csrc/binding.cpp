// Python binding of the serving operators: argument checks, allocation and the C-ABI
// call in one step.  A decoding step calls them once per layer on a few tokens, where the
// same work in Python (some thirty tensor attributes, packing the argument struct) took 14
// to 26 microseconds a call beside kernels of 2 to 6.  co_alibi_attn/serving.py documents
// the functions and their arguments; these take all of them by position.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "coalibi.h"

namespace {

using at::Tensor;

struct Refused {
  PyObject* type;
  std::string text;
};

std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(int n) { return std::to_string(n); }

template <typename... T>
[[noreturn]] void refuse(PyObject* type, const char* what, const T&... parts) {
  throw Refused{type, (std::string("co_alibi_attn: ") + what + ": " + ... + text(parts))};
}

std::string shape_of(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}
std::string shape_of(const Tensor& t) { return shape_of(t.sizes()); }

const Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, what, name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}

// The C-ABI code of a 16-bit type, or -1.
int dtype16(const Tensor& t) {
  const auto d = t.scalar_type();
  return d == at::kHalf ? COALIBI_F16 : d == at::kBFloat16 ? COALIBI_BF16 : -1;
}
int dtype_any(const Tensor& t) { return t.scalar_type() == at::kFloat ? COALIBI_F32 : dtype16(t); }

void on(const char* what, const char* name, const Tensor& t, c10::Device device) {
  if (t.device() != device) refuse(PyExc_ValueError, what, name, " is on ", t.device().str(), ", not ", device.str());
}

// The operators have no backward: a result that silently dropped its graph would train wrongly.
void no_grad(const char* what, const char* name, const Tensor& t) {
  if (c10::GradMode::is_enabled() && t.requires_grad())
    refuse(PyExc_RuntimeError, what, name, " requires grad, but there is no backward: call this under torch.no_grad()");
}

// As after torch's own in-place operations, a backward over a saved t fails instead of reading the
// new values.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The first three strides of [., ., ., D], 0 for a dimension of one entry.
void strides(const Tensor& t, long long* s) {
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// Whether every row of t [., ., ., D] is contiguous and 16-byte aligned.
bool rows16(const Tensor& t) {
  long long s[3];
  strides(t, s);
  return (t.stride(3) == 1 || t.size(3) == 1) && ((s[0] | s[1] | s[2]) & 7) == 0 &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

Tensor aligned_rows(const Tensor& t) { return rows16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

void check_cache(const char* what, const Tensor& k, const Tensor& v, const Tensor& table, int64_t B, int64_t D,
                 at::ScalarType dtype, c10::Device device) {
  if (k.dim() != 4 || v.sizes() != k.sizes())
    refuse(PyExc_ValueError, what, "k_pages and v_pages must both be [n_pages, Hkv, page_size, D], got ", shape_of(k),
           " and ", shape_of(v));
  if (k.scalar_type() != dtype || v.scalar_type() != dtype)
    refuse(PyExc_TypeError, what, "the cache holds ", c10::toString(k.scalar_type()), " and ",
           c10::toString(v.scalar_type()), ", the inputs ", c10::toString(dtype));
  if (k.size(3) != D) refuse(PyExc_ValueError, what, "the cache has head_dim ", k.size(3), ", the inputs ", D);
  if (k.size(2) % 16 != 0 || k.numel() == 0)
    refuse(PyExc_ValueError, what, "page_size must be a positive multiple of 16 and the pool not empty, got ",
           shape_of(k));
  if (k.size(0) > 0x7fffffff) refuse(PyExc_ValueError, what, "too many pages");
  for (const Tensor* t : {&k, &v}) {
    if (!rows16(*t)) refuse(PyExc_ValueError, what, "k_pages and v_pages must have contiguous, 16-byte aligned rows");
    for (int i = 0; i < 3; ++i)
      if (t->size(i) > 1 && t->stride(i) == 0)
        refuse(PyExc_ValueError, what, "k_pages and v_pages must not be expanded tensors");
  }
  if (table.scalar_type() != at::kInt) refuse(PyExc_TypeError, what, "page_table must be int32");
  if (table.dim() != 2 || table.size(0) != B || table.size(1) == 0 || (table.size(1) > 1 && table.stride(1) != 1))
    refuse(PyExc_ValueError, what, "page_table must be [", B, ", max_pages] with contiguous rows, got ",
           shape_of(table));
  if (table.size(1) * k.size(2) > 0x7fffff00)
    refuse(PyExc_ValueError, what, "a page table row must hold fewer than 2**31 tokens");
  on(what, "k_pages", k, device);
  on(what, "v_pages", v, device);
  on(what, "page_table", table, device);
}

// An index tensor of the given shape (one or two dimensions), contiguous.
Tensor indices(PyObject* o, const char* what, const char* name, at::IntArrayRef shape, at::ScalarType dtype,
               c10::Device device) {
  const Tensor& t = tensor(o, what, name);
  if (t.scalar_type() != dtype)
    refuse(PyExc_TypeError, what, name, " must be ", c10::toString(dtype), ", got ", c10::toString(t.scalar_type()));
  if (t.sizes() != shape) refuse(PyExc_ValueError, what, name, " must have shape ", shape_of(shape), ", got ", shape_of(t));
  on(what, name, t, device);
  return t.contiguous();
}

void* status_ptr(PyObject* o, const char* what) { return tensor(o, what, "status").data_ptr(); }

void check(int code, const char* fn) {
  if (code == COALIBI_OK) return;
  std::string s = std::string("co_alibi_attn: ") + fn + " failed: " + coalibi_strerror(code) + " (code " +
                  std::to_string(code) + ")";
  if (*coalibi_last_error()) s += std::string(": ") + coalibi_last_error();
  throw Refused{PyExc_RuntimeError, s};
}

void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// (k, v, k_pages, v_pages, page_table, start, count, q, rotary, interleaved, positions, status)
PyObject* append_paged_kv(PyObject* const* a) {
  const char* what = "append_paged_kv";
  const Tensor &k0 = tensor(a[0], what, "k"), &v0 = tensor(a[1], what, "v");
  const Tensor &kp = tensor(a[2], what, "k_pages"), &vp = tensor(a[3], what, "v_pages");
  const Tensor& table = tensor(a[4], what, "page_table");
  if (k0.dim() != 4 || v0.sizes() != k0.sizes())
    refuse(PyExc_ValueError, what, "k and v must both be [B, Hkv, S, D], got ", shape_of(k0), " and ", shape_of(v0));
  const int64_t B = k0.size(0), Hkv = k0.size(1), S = k0.size(2), D = k0.size(3);
  const auto dtype = k0.scalar_type();
  const auto device = k0.device();
  const bool with_q = a[7] != Py_None;
  CoalibiPagedAppendArgs p{};
  p.dtype = dtype16(k0);
  if (p.dtype < 0 || v0.scalar_type() != dtype || (with_q && tensor(a[7], what, "q").scalar_type() != dtype))
    refuse(PyExc_TypeError, what, "k, v and q must all be float16 or bfloat16");
  if (D != 64 && D != 128) refuse(PyExc_ValueError, what, "head_dim must be 64 or 128, got ", D);
  check_cache(what, kp, vp, table, B, D, dtype, device);
  if (kp.size(1) != Hkv) refuse(PyExc_ValueError, what, "the cache has ", kp.size(1), " kv heads, k ", Hkv);
  on(what, "v", v0, device);
  no_grad(what, "k", k0), no_grad(what, "v", v0), no_grad(what, "k_pages", kp), no_grad(what, "v_pages", vp);
  Tensor q, q_out, start, count, positions, cos, sin;
  if (with_q) {
    q = THPVariable_Unpack(a[7]);
    if (q.dim() != 4 || q.size(0) != B || q.size(2) != S || q.size(3) != D)
      refuse(PyExc_ValueError, what, "q must be [", B, ", Hq, ", S, ", ", D, "], got ", shape_of(q));
    on(what, "q", q, device);
    no_grad(what, "q", q);
    q = aligned_rows(q.detach());
    q_out = at::empty_like(q);
    p.Hq = (int)q.size(1);
    p.q = q.data_ptr();
    p.q_out = q_out.data_ptr();
    strides(q, p.q_stride);
    strides(q_out, p.q_out_stride);
  }
  start = indices(a[5], what, "start", {B}, at::kInt, device);
  p.start = start.data_ptr<int>();
  if (a[6] != Py_None) {
    count = indices(a[6], what, "count", {B}, at::kInt, device);
    p.count = count.data_ptr<int>();
  }
  if (a[10] != Py_None) {
    positions = indices(a[10], what, "positions", {B, S}, at::kInt, device);
    p.positions = positions.data_ptr<int>();
  }
  if (a[8] != Py_None) {
    if (!PyTuple_Check(a[8]) || PyTuple_GET_SIZE(a[8]) != 2)
      refuse(PyExc_TypeError, what, "rotary must be a tuple (cos, sin)");
    cos = tensor(PyTuple_GET_ITEM(a[8], 0), what, "cos");
    sin = tensor(PyTuple_GET_ITEM(a[8], 1), what, "sin");
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat)
      refuse(PyExc_TypeError, what, "the rotary tables must be float32");
    if (cos.dim() != 2 || sin.sizes() != cos.sizes() || cos.size(0) == 0 || cos.size(0) > 0x7fffffff ||
        cos.size(1) % 8 != 0 || cos.size(1) == 0 || 2 * cos.size(1) > D)
      refuse(PyExc_ValueError, what, "the rotary tables must be [n_pos, R / 2] with R a multiple of 16 up to ", D,
             ", got ", shape_of(cos), " and ", shape_of(sin));
    on(what, "cos", cos, device);
    on(what, "sin", sin, device);
    for (Tensor* t : {&cos, &sin})
      if (!t->is_contiguous() || (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15))
        *t = t->clone(at::MemoryFormat::Contiguous);
    p.cos = cos.data_ptr<float>();
    p.sin = sin.data_ptr<float>();
    p.n_pos = (int)cos.size(0);
    p.rot = 2 * (int)cos.size(1);
  }
  if (k0.numel() > 0) {
    const Tensor k = aligned_rows(k0), v = aligned_rows(v0);
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_pages = kp.data_ptr();
    p.v_pages = vp.data_ptr();
    p.page_table = table.data_ptr<int>();
    p.status = static_cast<int*>(status_ptr(a[11], what));
    strides(k, p.k_stride);
    strides(v, p.v_stride);
    strides(kp, p.k_page_stride);
    strides(vp, p.v_page_stride);
    p.table_stride = table.stride(0);
    p.B = (int)B, p.Hkv = (int)Hkv, p.S = (int)S, p.D = (int)D;
    p.page_size = (int)kp.size(2), p.max_pages = (int)table.size(1), p.n_pages = (int)kp.size(0);
    const int truth = PyObject_IsTrue(a[9]);
    if (truth < 0) return nullptr;
    p.interleaved = truth;
    if (with_q && p.Hq == 0) p.q = nullptr, p.q_out = nullptr;
    check(coalibi_paged_append(&p, stream_of(device)), "coalibi_paged_append");
    written(kp), written(vp);
  }
  if (!with_q) Py_RETURN_NONE;
  return THPVariable_Wrap(q_out);
}

// (q, k_pages, v_pages, page_table, ctx_lens, tree_mask, sm_scale, slopes, status)
PyObject* paged_tree_attention(PyObject* const* a) {
  const char* what = "paged_tree_attention";
  const Tensor& q0 = tensor(a[0], what, "q");
  const Tensor &kp = tensor(a[1], what, "k_pages"), &vp = tensor(a[2], what, "v_pages");
  const Tensor &table = tensor(a[3], what, "page_table"), &slopes0 = tensor(a[7], what, "slopes");
  if (q0.dim() != 4) refuse(PyExc_ValueError, what, "q must be [B, Hq, Sq, D], got ", shape_of(q0));
  const int64_t B = q0.size(0), Hq = q0.size(1), Sq = q0.size(2), D = q0.size(3);
  const auto device = q0.device();
  CoalibiPagedAttentionArgs p{};
  p.dtype = dtype16(q0);
  if (p.dtype < 0) refuse(PyExc_TypeError, what, "q must be float16 or bfloat16, got ", c10::toString(q0.scalar_type()));
  if (D != 64 && D != 128) refuse(PyExc_ValueError, what, "head_dim must be 64 or 128, got ", D);
  if (Sq > COALIBI_TREE_MAX_SQ)
    refuse(PyExc_ValueError, what, "at most ", COALIBI_TREE_MAX_SQ, " rows per request, got ", Sq);
  check_cache(what, kp, vp, table, B, D, q0.scalar_type(), device);
  const int64_t Hkv = kp.size(1);
  if (Hq % Hkv != 0) refuse(PyExc_ValueError, what, "num_heads ", Hq, " must be a multiple of num_kv_heads ", Hkv);
  const Tensor ctx = indices(a[4], what, "ctx_lens", {B}, at::kInt, device);
  Tensor mask;
  if (a[5] != Py_None) {
    const int64_t dims = tensor(a[5], what, "tree_mask").dim();
    mask = dims == 1 ? indices(a[5], what, "tree_mask", {Sq}, at::kLong, device)
                     : indices(a[5], what, "tree_mask", {B, Sq}, at::kLong, device);
    p.tree_mask = reinterpret_cast<const long long*>(mask.data_ptr<int64_t>());
    p.mask_stride = dims == 1 ? 0 : Sq;
  }
  p.slopes_dtype = dtype_any(slopes0);
  if (p.slopes_dtype < 0)
    refuse(PyExc_TypeError, what, "slopes must be float16, bfloat16 or float32, got ",
           c10::toString(slopes0.scalar_type()));
  if (slopes0.dim() != 1 || slopes0.size(0) != Hq)
    refuse(PyExc_ValueError, what, "slopes must have shape [", Hq, "], got ", shape_of(slopes0));
  on(what, "slopes", slopes0, device);
  no_grad(what, "q", q0), no_grad(what, "k_pages", kp), no_grad(what, "v_pages", vp);
  no_grad(what, "slopes", slopes0);
  p.sm_scale = (float)(1.0 / std::sqrt((double)D));
  if (a[6] != Py_None) {
    const double s = PyFloat_AsDouble(a[6]);
    if (s == -1.0 && PyErr_Occurred()) return nullptr;
    p.sm_scale = (float)s;
  }
  const Tensor q = aligned_rows(q0.detach()), slopes = slopes0.contiguous();
  Tensor o = at::empty_like(q);
  if (q.numel() > 0) {
    const size_t bytes = coalibi_paged_attention_workspace_bytes((int)B, (int)Hq, (int)Hkv, (int)Sq, (int)D);
    const Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    p.q = q.data_ptr();
    p.o = o.data_ptr();
    p.k_pages = kp.data_ptr();
    p.v_pages = vp.data_ptr();
    p.slopes = slopes.data_ptr();
    p.page_table = table.data_ptr<int>();
    p.ctx_lens = ctx.data_ptr<int>();
    p.status = static_cast<int*>(status_ptr(a[8], what));
    strides(q, p.q_stride);
    strides(o, p.o_stride);
    strides(kp, p.k_page_stride);
    strides(vp, p.v_page_stride);
    p.table_stride = table.stride(0);
    p.B = (int)B, p.Hq = (int)Hq, p.Hkv = (int)Hkv, p.Sq = (int)Sq, p.D = (int)D;
    p.page_size = (int)kp.size(2), p.max_pages = (int)table.size(1), p.n_pages = (int)kp.size(0);
    check(coalibi_paged_attention(&p, ws.data_ptr(), bytes, stream_of(device)), "coalibi_paged_attention");
  }
  return THPVariable_Wrap(o);
}

// A sampling parameter: a number, or a tensor [B] (kept alive in `keep`).
template <typename T>
const T* per_row(PyObject* o, const char* name, int64_t B, at::ScalarType dtype, c10::Device device, Tensor& keep,
                 T* all) {
  const char* what = "sample_tokens";
  if (THPVariable_Check(o)) {
    keep = indices(o, what, name, {B}, dtype, device);
    return keep.data_ptr<T>();
  }
  if (std::is_same<T, int>::value) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
    *all = (T)(v > 0x7fffffff ? 0x7fffffff : v < 0 ? 0 : v);
  } else {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
    *all = (T)v;
  }
  return nullptr;
}

// (logits, noise, temperature, top_k, top_p, min_p)
PyObject* sample_tokens(PyObject* const* a) {
  const char* what = "sample_tokens";
  const Tensor &logits0 = tensor(a[0], what, "logits"), &noise0 = tensor(a[1], what, "noise");
  if (logits0.dim() != 2 || noise0.sizes() != logits0.sizes())
    refuse(PyExc_ValueError, what, "logits and noise must both be [B, V], got ", shape_of(logits0), " and ",
           shape_of(noise0));
  CoalibiSampleArgs p{};
  p.dtype = dtype_any(logits0);
  if (p.dtype < 0 || noise0.scalar_type() != at::kFloat)
    refuse(PyExc_TypeError, what, "logits must be float16, bfloat16 or float32 and noise float32, got ",
           c10::toString(logits0.scalar_type()), " and ", c10::toString(noise0.scalar_type()));
  const int64_t B = logits0.size(0), V = logits0.size(1);
  const auto device = logits0.device();
  on(what, "noise", noise0, device);
  if (V == 0 || V > COALIBI_SAMPLE_MAX_VOCAB)
    refuse(PyExc_ValueError, what, "the vocabulary must have 1 to 2**21 tokens, got ", V);
  const Tensor logits = logits0.stride(1) == 1 || V == 1 ? logits0.detach() : logits0.detach().contiguous();
  const Tensor noise = noise0.stride(1) == 1 || V == 1 ? noise0.detach() : noise0.detach().contiguous();
  Tensor tokens = at::empty({B}, logits.options().dtype(at::kLong));
  Tensor logprobs = at::empty({B}, logits.options().dtype(at::kFloat));
  Tensor keep[4];
  p.temperature = per_row<float>(a[2], "temperature", B, at::kFloat, device, keep[0], &p.temperature_all);
  p.top_k = per_row<int>(a[3], "top_k", B, at::kInt, device, keep[1], &p.top_k_all);
  p.top_p = per_row<float>(a[4], "top_p", B, at::kFloat, device, keep[2], &p.top_p_all);
  p.min_p = per_row<float>(a[5], "min_p", B, at::kFloat, device, keep[3], &p.min_p_all);
  if (B > 0) {
    p.logits = logits.data_ptr();
    p.noise = noise.data_ptr<float>();
    p.tokens = reinterpret_cast<long long*>(tokens.data_ptr<int64_t>());
    p.logprobs = logprobs.data_ptr<float>();
    p.logits_stride = B > 1 ? logits.stride(0) : 0;
    p.noise_stride = B > 1 ? noise.stride(0) : 0;
    p.B = (int)B, p.V = (int)V;
    check(coalibi_sample(&p, stream_of(device)), "coalibi_sample");
  }
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(tokens));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(logprobs));
  return pair;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& r) {
    if (r.type != nullptr) PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "co_alibi_attn: unknown C++ exception");
  }
  return nullptr;
}

#define METHOD(name, n) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(append_paged_kv, 12), METHOD(paged_tree_attention, 9), METHOD(sample_tokens, 6),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
