// Python binding of the serving operators: argument checks, allocation and the C-ABI
// call in one step.  A decoding step calls them once per layer on a few tokens, where the
// same work in Python (some thirty tensor attributes, packing the argument struct) took 14
// to 26 microseconds a call beside kernels of 2 to 6.  co_alibi_attn/serving.py documents
// the functions and their arguments; these take all of them by position.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <stdexcept>
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

// A result that silently dropped a forward-mode tangent would have a derivative of 0.
void no_tangent(const char* what, const char* name, const Tensor& t) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined())
    refuse(PyExc_RuntimeError, what, name, " carries a forward-mode tangent, but there is no forward-mode derivative");
}

// The operators have no backward: a result that silently dropped its graph would train wrongly.
void no_grad(const char* what, const char* name, const Tensor& t) {
  no_tangent(what, name, t);
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
  return (t.stride(3) == 1 || t.size(3) == 1) && ((s[0] | s[1] | s[2]) & (16 / t.element_size() - 1)) == 0 &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

// (a call of torch costs a microsecond or more: none where nothing is to be done)
Tensor aligned_rows(const Tensor& t) { return rows16(t) ? t : t.detach().clone(at::MemoryFormat::Contiguous); }
Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, c10::Device device) {
  return at::detail::empty_cuda(sizes, dtype, device, std::nullopt);  // (at::empty without its two dispatches)
}
Tensor empty_as(const Tensor& t) { return t.is_contiguous() ? empty(t.sizes(), t.scalar_type(), t.device()) : at::empty_like(t); }

// The scales of a cache in 8 bits.
struct Scales {
  Tensor k, v;
  CoalibiCacheScales c{};
  bool given = false;
};

Scales scales_of(PyObject* o, const char* what) {
  Scales s;
  if (o == Py_None) return s;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) refuse(PyExc_TypeError, what, "scales must be a tuple (k_scales, v_scales)");
  s.k = tensor(PyTuple_GET_ITEM(o, 0), what, "k_scales");
  s.v = tensor(PyTuple_GET_ITEM(o, 1), what, "v_scales");
  s.given = true;
  return s;
}

void check_scales(const char* what, Scales& s, const Tensor& pages, c10::Device device) {
  const int64_t blocks = pages.size(2) / COALIBI_QUANT_BLOCK;
  const char* names[2] = {"k_scales", "v_scales"};
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = i ? s.v : s.k;
    if (t.scalar_type() != at::kFloat) refuse(PyExc_TypeError, what, names[i], " must be float32, got ", c10::toString(t.scalar_type()));
    if (t.dim() != 3 || t.size(0) != pages.size(0) || t.size(1) != pages.size(1) || t.size(2) != blocks)
      refuse(PyExc_ValueError, what, names[i], " must be [", pages.size(0), ", ", pages.size(1), ", ", blocks, "], got ", shape_of(t));
    if (blocks > 1 && t.stride(2) != 1) refuse(PyExc_ValueError, what, names[i], " must have contiguous rows");
    on(what, names[i], t, device);
    for (int d = 0; d < 2; ++d) {
      if (t.size(d) > 1 && t.stride(d) == 0) refuse(PyExc_ValueError, what, names[i], " must not be an expanded tensor");
      (i ? s.c.v_stride : s.c.k_stride)[d] = t.size(d) > 1 ? t.stride(d) : 0;
    }
  }
  s.c.k = s.k.data_ptr<float>();
  s.c.v = s.v.data_ptr<float>();
}

// dtype: of the values that go in or come out; the pools' own, unless they hold codes.
void check_cache(const char* what, const Tensor& k, const Tensor& v, const Tensor& table, int64_t B, int64_t D,
                 at::ScalarType dtype, c10::Device device, Scales& scales) {
  const bool codes = k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn;
  if (codes != scales.given)
    refuse(PyExc_TypeError, what, codes ? "a cache of float8_e4m3fn needs scales" : "scales are for a cache of float8_e4m3fn, got ",
           codes ? "" : c10::toString(k.scalar_type()));
  if (k.dim() != 4 || v.sizes() != k.sizes())
    refuse(PyExc_ValueError, what, "k_pages and v_pages must both be [n_pages, Hkv, page_size, D], got ", shape_of(k),
           " and ", shape_of(v));
  if (!codes && (k.scalar_type() != dtype || v.scalar_type() != dtype))
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
  if (codes) check_scales(what, scales, k, device);
}

// An index tensor of the given shape (one or two dimensions), contiguous.
Tensor indices(const Tensor& t, const char* what, const char* name, at::IntArrayRef shape, at::ScalarType dtype,
               c10::Device device) {
  if (t.scalar_type() != dtype)
    refuse(PyExc_TypeError, what, name, " must be ", c10::toString(dtype), ", got ", c10::toString(t.scalar_type()));
  if (t.sizes() != shape) refuse(PyExc_ValueError, what, name, " must have shape ", shape_of(shape), ", got ", shape_of(t));
  on(what, name, t, device);
  return t.contiguous();
}
Tensor indices(PyObject* o, const char* what, const char* name, at::IntArrayRef shape, at::ScalarType dtype,
               c10::Device device) {
  return indices(tensor(o, what, name), what, name, shape, dtype, device);
}

void rotary_of(PyObject* o, const char* what, Tensor& cos, Tensor& sin) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2)
    refuse(PyExc_TypeError, what, "rotary must be a tuple (cos, sin)");
  cos = tensor(PyTuple_GET_ITEM(o, 0), what, "cos");
  sin = tensor(PyTuple_GET_ITEM(o, 1), what, "sin");
}

// The rotary tables, made contiguous and aligned.
void check_rotary(const char* what, int64_t D, c10::Device device, Tensor& cos, Tensor& sin) {
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

// (k, v, k_pages, v_pages, page_table, start, count, q, rotary, interleaved, positions, status, scales)
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
  Scales scales = scales_of(a[12], what);
  check_cache(what, kp, vp, table, B, D, dtype, device, scales);
  if (scales.given) no_grad(what, "k_scales", scales.k), no_grad(what, "v_scales", scales.v);
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
    q = aligned_rows(q);
    q_out = empty_as(q);
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
    rotary_of(a[8], what, cos, sin);
    check_rotary(what, D, device, cos, sin);
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
    if (scales.given) {
      check(coalibi_paged_append8(&p, &scales.c, stream_of(device)), "coalibi_paged_append8");
      written(scales.k), written(scales.v);
    } else {
      check(coalibi_paged_append(&p, stream_of(device)), "coalibi_paged_append");
    }
    written(kp), written(vp);
  }
  if (!with_q) Py_RETURN_NONE;
  return THPVariable_Wrap(q_out);
}

// (q, k_pages, v_pages, page_table, ctx_lens, tree_mask, sm_scale, slopes, status, scales)
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
  Scales scales = scales_of(a[9], what);
  check_cache(what, kp, vp, table, B, D, q0.scalar_type(), device, scales);
  if (scales.given) no_grad(what, "k_scales", scales.k), no_grad(what, "v_scales", scales.v);
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
  const Tensor q = aligned_rows(q0), slopes = slopes0.contiguous();
  Tensor o = empty_as(q);
  if (q.numel() > 0) {
    const size_t bytes = (scales.given ? coalibi_paged_attention8_workspace_bytes : coalibi_paged_attention_workspace_bytes)(
        (int)B, (int)Hq, (int)Hkv, (int)Sq, (int)D);
    const Tensor ws = empty({(int64_t)bytes}, at::kByte, device);
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
    if (scales.given)
      check(coalibi_paged_attention8(&p, &scales.c, ws.data_ptr(), bytes, stream_of(device)), "coalibi_paged_attention8");
    else
      check(coalibi_paged_attention(&p, ws.data_ptr(), bytes, stream_of(device)), "coalibi_paged_attention");
  }
  return THPVariable_Wrap(o);
}

// (k_pages, v_pages, page_table, positions, scales, bf16, status)
PyObject* read_paged_kv(PyObject* const* a) {
  const char* what = "read_paged_kv";
  const Tensor &kp = tensor(a[0], what, "k_pages"), &vp = tensor(a[1], what, "v_pages");
  const Tensor &table = tensor(a[2], what, "page_table"), &positions0 = tensor(a[3], what, "positions");
  if (positions0.dim() != 2) refuse(PyExc_ValueError, what, "positions must be [B, S], got ", shape_of(positions0));
  const int64_t B = positions0.size(0), S = positions0.size(1);
  const auto device = kp.device();
  const bool bf16 = PyObject_IsTrue(a[5]);
  const auto dtype = bf16 ? at::kBFloat16 : at::kHalf;
  Scales scales = scales_of(a[4], what);
  if (!scales.given) refuse(PyExc_TypeError, what, "scales must be a tuple (k_scales, v_scales)");
  if (kp.dim() == 4 && kp.size(3) != 64 && kp.size(3) != 128) refuse(PyExc_ValueError, what, "head_dim must be 64 or 128, got ", kp.size(3));
  check_cache(what, kp, vp, table, B, kp.dim() == 4 ? kp.size(3) : 0, dtype, device, scales);
  no_grad(what, "k_scales", scales.k), no_grad(what, "v_scales", scales.v);
  no_grad(what, "k_pages", kp), no_grad(what, "v_pages", vp);
  const int64_t Hkv = kp.size(1), D = kp.size(3);
  if (S > 0x7fffffff) refuse(PyExc_ValueError, what, "too many tokens");
  const Tensor positions = indices(a[3], what, "positions", {B, S}, at::kInt, device);
  Tensor k = empty({B, Hkv, S, D}, dtype, device), v = empty_as(k);
  if (k.numel() > 0) {
    CoalibiPagedReadArgs p{};
    p.k_pages = kp.data_ptr();
    p.v_pages = vp.data_ptr();
    p.page_table = table.data_ptr<int>();
    p.positions = positions.data_ptr<int>();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.status = static_cast<int*>(status_ptr(a[6], what));
    strides(kp, p.k_page_stride);
    strides(vp, p.v_page_stride);
    p.table_stride = table.stride(0);
    p.B = (int)B, p.Hkv = (int)Hkv, p.S = (int)S, p.D = (int)D;
    p.page_size = (int)kp.size(2), p.max_pages = (int)table.size(1), p.n_pages = (int)kp.size(0);
    p.dtype = bf16 ? COALIBI_BF16 : COALIBI_F16;
    check(coalibi_paged_read8(&p, &scales.c, stream_of(device)), "coalibi_paged_read8");
  }
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
  return pair;
}

// The arguments of the heads' forward; its backward takes them too.
struct HeadsIn {
  Tensor qkv, weight[2], cos, sin, start, positions, status;  // undefined: not given
  int64_t Hq, Hkv;
  double eps;
  bool interleaved;
};

// What a call of the C entries needs, and the tensors it points at.
struct Heads {
  CoalibiHeadsArgs p{};
  Tensor qkv, weight[2], cos, sin, start, positions;
  int64_t B, S, Hq, Hkv, D;
};

Heads check_heads(const HeadsIn& a) {
  const char* what = "norm_rotate_qkv";
  Heads h;
  const Tensor& x = a.qkv;
  h.Hq = a.Hq, h.Hkv = a.Hkv;
  if (x.dim() != 4) refuse(PyExc_ValueError, what, "qkv must be [B, S, num_heads + 2 num_kv_heads, D], got ", shape_of(x));
  h.B = x.size(0), h.S = x.size(1), h.D = x.size(3);
  if (h.Hq <= 0 || h.Hkv <= 0 || h.Hq > 65535 || h.Hkv > 65535 || x.size(2) != h.Hq + 2 * h.Hkv)
    refuse(PyExc_ValueError, what, "qkv must hold num_heads + 2 num_kv_heads heads, got ", shape_of(x), " with ", h.Hq, " and ", h.Hkv);
  CoalibiHeadsArgs& p = h.p;
  p.dtype = p.weight_dtype = dtype16(x);
  if (p.dtype < 0) refuse(PyExc_TypeError, what, "qkv must be float16 or bfloat16, got ", c10::toString(x.scalar_type()));
  if (h.D != 64 && h.D != 128) refuse(PyExc_ValueError, what, "head_dim must be 64 or 128, got ", h.D);
  if (h.B > 0x7fffffff || h.S > 0x7fffffff || h.B * h.S > 0x7fffffff) refuse(PyExc_ValueError, what, "too many tokens");
  const auto device = x.device();
  if (!device.is_cuda()) refuse(PyExc_ValueError, what, "qkv is on ", device.str());
  h.qkv = aligned_rows(x);
  strides(h.qkv, p.qkv_stride);
  const char* names[2] = {"q_weight", "k_weight"};
  at::ScalarType type = x.scalar_type();
  bool seen = false;
  for (int i = 0; i < 2; ++i) {
    const Tensor& w = a.weight[i];
    if (!w.defined()) continue;
    if ((w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat) || (seen && w.scalar_type() != type))
      refuse(PyExc_TypeError, what, "the weights must both be ", c10::toString(x.scalar_type()), " or float32, got ", c10::toString(w.scalar_type()));
    if (w.dim() != 1 || w.size(0) != h.D) refuse(PyExc_ValueError, what, names[i], " must have shape [", h.D, "], got ", shape_of(w));
    on(what, names[i], w, device);
    h.weight[i] = w.is_contiguous() && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 3) == 0 ? w : w.detach().clone(at::MemoryFormat::Contiguous);
    type = w.scalar_type();
    seen = true;
  }
  if (seen && type == at::kFloat) p.weight_dtype = COALIBI_F32;
  p.q_weight = h.weight[0].defined() ? h.weight[0].data_ptr() : nullptr;
  p.k_weight = h.weight[1].defined() ? h.weight[1].data_ptr() : nullptr;
  if (!(a.eps >= 0)) refuse(PyExc_ValueError, what, "eps must not be negative");
  p.eps = (float)a.eps;
  if (a.cos.defined()) {
    h.cos = a.cos, h.sin = a.sin;
    check_rotary(what, h.D, device, h.cos, h.sin);
    p.cos = h.cos.data_ptr<float>();
    p.sin = h.sin.data_ptr<float>();
    p.n_pos = (int)h.cos.size(0);
    p.rot = 2 * (int)h.cos.size(1);
  }
  if (a.start.defined()) {
    h.start = indices(a.start, what, "start", {h.B}, at::kInt, device);
    p.start = h.start.data_ptr<int>();
  }
  if (a.positions.defined()) {
    h.positions = indices(a.positions, what, "positions", {h.B, h.S}, at::kInt, device);
    p.positions = h.positions.data_ptr<int>();
  }
  p.interleaved = a.interleaved;
  p.status = static_cast<int*>(a.status.data_ptr());
  p.qkv = h.qkv.data_ptr();
  p.B = (int)h.B, p.S = (int)h.S, p.Hq = (int)h.Hq, p.Hkv = (int)h.Hkv, p.D = (int)h.D;
  return h;
}

using torch::autograd::variable_list;

variable_list heads_forward(const HeadsIn& a) {
  Heads h = check_heads(a);
  CoalibiHeadsArgs& p = h.p;
  const auto device = h.qkv.device();
  const auto dtype = h.qkv.scalar_type();
  Tensor q = empty({h.B, h.Hq, h.S, h.D}, dtype, device), k = empty({h.B, h.Hkv, h.S, h.D}, dtype, device);
  Tensor v = empty_as(k);
  if (h.qkv.numel() > 0) {
    p.q = q.data_ptr();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    strides(q, p.q_stride), strides(k, p.k_stride), strides(v, p.v_stride);
    check(coalibi_heads_fwd(&p, stream_of(device)), "coalibi_heads_fwd");
  }
  return {q, k, v};
}

// (dqkv, the weights' gradients where there are weights)
variable_list heads_backward(const HeadsIn& a, const variable_list& grads) {
  const char* what = "norm_rotate_qkv's backward";
  Heads h = check_heads(a);
  CoalibiHeadsArgs& p = h.p;
  const auto device = h.qkv.device();
  Tensor d[3];
  const char* names[3] = {"the gradient of q", "the gradient of k", "the gradient of v"};
  for (int i = 0; i < 3; ++i) {
    const Tensor& t = grads[i];
    const int64_t H = i ? h.Hkv : h.Hq;
    if (t.sizes() != at::IntArrayRef{h.B, H, h.S, h.D} || t.scalar_type() != h.qkv.scalar_type())
      refuse(PyExc_ValueError, what, names[i], " has shape ", shape_of(t), " and type ", c10::toString(t.scalar_type()));
    on(what, names[i], t, device);
    d[i] = aligned_rows(t);
  }
  Tensor dqkv = empty({h.B, h.S, h.Hq + 2 * h.Hkv, h.D}, h.qkv.scalar_type(), device), dw[2];
  for (int i = 0; i < 2; ++i)
    if (h.weight[i].defined())
      dw[i] = h.qkv.numel() > 0 ? empty({h.D}, h.weight[i].scalar_type(), device) : at::zeros_like(h.weight[i].detach());
  if (h.qkv.numel() > 0) {
    const size_t bytes = coalibi_heads_bwd_workspace_bytes((int)h.Hq, (int)h.Hkv, (int)h.D);
    const Tensor ws = empty({(int64_t)bytes}, at::kByte, device);
    p.q = d[0].data_ptr();
    p.k = d[1].data_ptr();
    p.v = d[2].data_ptr();
    strides(d[0], p.q_stride), strides(d[1], p.k_stride), strides(d[2], p.v_stride);
    p.dqkv = dqkv.data_ptr();
    p.dq_weight = dw[0].defined() ? dw[0].data_ptr() : nullptr;
    p.dk_weight = dw[1].defined() ? dw[1].data_ptr() : nullptr;
    check(coalibi_heads_bwd(&p, ws.data_ptr(), bytes, stream_of(device)), "coalibi_heads_bwd");
  }
  return {dqkv, dw[0], dw[1]};
}

// The heads in a graph.  The backward runs in the engine's thread without the interpreter's lock, so nothing of it
// is a Python object (through torch.autograd.Function forward and backward of 650 tokens took the host 160 us, 130 so; a
// single product and its gradient take 50).
struct HeadsGrad : torch::autograd::Function<HeadsGrad> {
  using Context = torch::autograd::AutogradContext;
  using Weight = std::optional<Tensor>;

  static variable_list forward(Context* ctx, const Tensor& qkv, const Weight& q_weight, const Weight& k_weight, const HeadsIn* a) {
    variable_list out = heads_forward(*a);
    ctx->save_for_backward({qkv, a->weight[0], a->weight[1], a->cos, a->sin, a->start, a->positions});
    ctx->saved_data["status"] = a->status;  // (not saved as a variable: it is written to)
    ctx->saved_data["heads"] = std::vector<int64_t>{a->Hq, a->Hkv, a->interleaved};
    ctx->saved_data["eps"] = a->eps;
    return out;
  }

  static variable_list backward(Context* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const auto heads = ctx->saved_data["heads"].toIntVector();
    const HeadsIn a{s[0], {s[1], s[2]}, s[3], s[4], s[5], s[6], ctx->saved_data["status"].toTensor(),
                    heads[0], heads[1], ctx->saved_data["eps"].toDouble(), heads[2] != 0};
    variable_list d;
    try {
      d = heads_backward(a, grads);
    } catch (const Refused& r) {
      throw std::runtime_error(r.text);
    }
    if (c10::GradMode::is_enabled()) {  // no second derivative: an error where one is asked for
      for (Tensor& t : d)
        if (t.defined()) t.set_requires_grad(true);
      d = (*std::make_shared<torch::autograd::DelayedError>("co_alibi_attn: norm_rotate_qkv has no second derivative", 3))(std::move(d));
    }
    return {d[0], d[1], d[2], Tensor()};
  }
};

int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}

// (qkv, num_heads, num_kv_heads, q_weight, k_weight, eps, rotary, start, positions, interleaved, status) -> (q, k, v)
PyObject* norm_rotate_qkv(PyObject* const* a) {
  const char* what = "norm_rotate_qkv";
  HeadsIn in;
  const auto given = [what](PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, what, name); };
  in.qkv = tensor(a[0], what, "qkv");
  in.Hq = whole(a[1]), in.Hkv = whole(a[2]);
  in.weight[0] = given(a[3], "q_weight"), in.weight[1] = given(a[4], "k_weight");
  in.eps = PyFloat_AsDouble(a[5]);
  if (in.eps == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  no_tangent(what, "qkv", in.qkv);
  for (int i = 0; i < 2; ++i)
    if (in.weight[i].defined()) no_tangent(what, i ? "k_weight" : "q_weight", in.weight[i]);
  if (a[6] != Py_None) {
    rotary_of(a[6], what, in.cos, in.sin);
    no_grad(what, "cos", in.cos), no_grad(what, "sin", in.sin);
  }
  in.start = given(a[7], "start"), in.positions = given(a[8], "positions");
  const int truth = PyObject_IsTrue(a[9]);
  if (truth < 0) throw Refused{nullptr, ""};
  in.interleaved = truth;
  in.status = tensor(a[10], what, "status");
  bool graph = false;
  for (const Tensor& t : {in.qkv, in.weight[0], in.weight[1]}) graph |= t.defined() && t.requires_grad();
  const auto weight = [&in](int i) { return in.weight[i].defined() ? HeadsGrad::Weight(in.weight[i]) : HeadsGrad::Weight(); };
  const variable_list out = graph && c10::GradMode::is_enabled() ? HeadsGrad::apply(in.qkv, weight(0), weight(1), &in) : heads_forward(in);
  PyObject* t = PyTuple_New(3);
  if (t == nullptr) return nullptr;
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(out[i]));
  return t;
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
  Tensor tokens = empty({B}, at::kLong, device);
  Tensor logprobs = empty({B}, at::kFloat, device);
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
  } catch (python_error& e) {  // of a hook on saved tensors
    e.restore();
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
PyMethodDef methods[] = {METHOD(append_paged_kv, 13), METHOD(paged_tree_attention, 10), METHOD(sample_tokens, 6),
                         METHOD(read_paged_kv, 7), METHOD(norm_rotate_qkv, 11),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
