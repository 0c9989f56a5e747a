// The eager calls' host side in C++: what `paged_kernels.paged_decode`,
// `paged_kernels.paged_prefill` and `rope.rope_kv_write` (over an int8 pool
// too) and `engine.ops.linear_int8` do in Python before they reach the C ABI (reading the
// operands, the checks, the output and workspace, the call).
//
// A decode layer over a few short contexts runs ~8 us on the GPU, and its two
// calls took 31 us of Python and ctypes (about half checks and attribute
// reads, half converting ~60 arguments); through here they take 15.
//
// Each function serves exactly what the Python code would pass on unchanged:
// plain torch tensors on one ROCm device, in the layouts and dtypes the C ABI
// takes. For anything else (another device or dtype, a layout that needs a
// copy, a shape that does not match, a tensor subclass) it does nothing and
// returns None, and the Python code, which converts or raises, runs as
// before. A failed call returns its status for the Python code to raise.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <Python.h>

#include <cmath>
#include <cstdint>

#include "../../include/liteinfer_amd.h"

namespace {

using PlanFn = decltype(&li_paged_decode_plan);
using DecodeFn = decltype(&li_paged_decode_write);
using PrefillPlanFn = decltype(&li_paged_prefill_plan);
using PrefillFn = decltype(&li_paged_prefill_ex);
using RopeFn = decltype(&li_rope_kv_write);
using RopeF8Fn = decltype(&li_rope_kv_write_fp8);
PlanFn g_plan = nullptr;
DecodeFn g_decode = nullptr;
PrefillPlanFn g_prefill_plan = nullptr;
PrefillFn g_prefill = nullptr;
RopeFn g_rope = nullptr;
RopeF8Fn g_rope_f8 = nullptr;
decltype(&li_paged_decode_int8) g_decode_int8 = nullptr;
decltype(&li_paged_prefill_int8_plan) g_prefill_int8_plan = nullptr;
decltype(&li_paged_prefill_int8) g_prefill_int8 = nullptr;
decltype(&li_rope_kv_write_int8) g_rope_int8 = nullptr;
decltype(&li_linear_int8_plan) g_linear_int8_plan = nullptr;
decltype(&li_linear_int8) g_linear_int8 = nullptr;

// The interpreter lock is given up for the allocation and the launch, as
// torch's own calls and ctypes do.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// A plain tensor (no subclass, so no __torch_function__ of its own) that
// holds device memory of its own, or nullptr.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
  const auto keys = t.key_set();
  if (keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::FuncTorchBatched) ||
      keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Functionalize) ||
      t.is_neg() || t.is_conj())
    return nullptr;
  return &t;
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LI_F32;
    case at::kHalf: return LI_F16;
    case at::kBFloat16: return LI_BF16;
    case at::kFloat8_e4m3fn: return LI_FP8_E4M3;
    default: return -1;
  }
}

bool pools_ok(const at::Tensor& k, const at::Tensor& v) {
  return k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.stride(2) == 1 &&
         k.scalar_type() == v.scalar_type();
}

// The pool's element code beside 16- or 32-bit rows of type `rows` (scales
// checked for an fp8 pool), or -1.
int pool_code(at::ScalarType rows, const at::Tensor& pool, double k_scale, double v_scale) {
  const int code = code_of(rows);
  if (code < 0 || code == LI_FP8_E4M3) return -1;
  if (pool.scalar_type() == rows) return code;
  if (pool.scalar_type() != at::kFloat8_e4m3fn || code == LI_F32) return -1;
  if (!(k_scale > 0) || !(v_scale > 0) || !std::isfinite(k_scale) || !std::isfinite(v_scale)) return -1;
  return LI_FP8_E4M3;
}

// 1: a number into *out; 0: not one this serves.
bool number(PyObject* o, double* out) {
  if (PyFloat_CheckExact(o)) *out = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *out = PyLong_AsDouble(o);
  else return false;
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool integer(PyObject* o, int64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && !PyErr_Occurred();
}

// decode(query, key_pool, value_pool, slot_table, context_lens, scaling, groups, block_kv, num_splits (0: None),
//        flags, k_scale, v_scale, new_key or None, new_value or None, stream) -> out, status, or None
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15 || !g_decode) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *kp = plain(a[1]), *vp = plain(a[2]), *st = plain(a[3]), *cl = plain(a[4]);
  double scaling, k_scale, v_scale;
  int64_t groups, block_kv, splits, flags, stream;
  if (!q || !kp || !vp || !st || !cl || !number(a[5], &scaling) || !integer(a[6], &groups) || !integer(a[7], &block_kv) ||
      !integer(a[8], &splits) || !integer(a[9], &flags) || !number(a[10], &k_scale) || !number(a[11], &v_scale) ||
      !integer(a[14], &stream))
    Py_RETURN_NONE;
  const auto device = q->device();
  if (kp->device() != device || vp->device() != device || st->device() != device || cl->device() != device) Py_RETURN_NONE;
  if (!pools_ok(*kp, *vp) || kp->size(0) >= (int64_t(1) << 31)) Py_RETURN_NONE;
  const int kv = pool_code(q->scalar_type(), *kp, k_scale, v_scale);
  if (kv < 0 || q->dim() != 3 || q->stride(2) != 1 || st->dim() != 2 || st->scalar_type() != at::kLong ||
      st->stride(1) != 1 || cl->dim() != 1 || cl->scalar_type() != at::kInt || cl->stride(0) != 1)
    Py_RETURN_NONE;
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2), kv_heads = kp->size(1), width = st->size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (groups < 1 || heads % groups || heads / groups != kv_heads || dim != kp->size(2) || st->size(0) != batch ||
      cl->size(0) != batch || batch < 1 || batch > kInt || heads > kInt || width > kInt || splits < 0 || splits > kInt ||
      block_kv < 0 || block_kv > kInt || flags < 0 || flags > kInt)
    Py_RETURN_NONE;
  const at::Tensor *nk = nullptr, *nv = nullptr;
  if (a[12] != Py_None || a[13] != Py_None) {
    nk = plain(a[12]), nv = plain(a[13]);
    if (!nk || !nv) Py_RETURN_NONE;
    for (const at::Tensor* t : {nk, nv})
      if (t->dim() != 3 || t->size(0) != batch || t->size(1) != kv_heads || t->size(2) != dim || t->stride(2) != 1 ||
          t->scalar_type() != q->scalar_type() || t->device() != device)
        Py_RETURN_NONE;
    if (nk->strides() != nv->strides()) Py_RETURN_NONE;
  }
  size_t need = 0;
  if (g_plan((int)batch, (int)heads, (int)kv_heads, (int)dim, (int)width, (int)splits, 0, (int)block_kv, nullptr, nullptr,
             &need) != LI_OK)
    Py_RETURN_NONE;
  try {
    at::Tensor out, workspace;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      out = at::empty_like(*q);
      if (need) workspace = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
      status = g_decode(q->data_ptr(), q->stride(0), q->stride(1), kp->data_ptr(), vp->data_ptr(), kp->stride(0),
                        kp->stride(1), st->const_data_ptr<int64_t>(), st->stride(0), (int)width,
                        cl->const_data_ptr<int32_t>(), nk ? nk->data_ptr() : nullptr, nv ? nv->data_ptr() : nullptr,
                        nk ? nk->stride(0) : 0, nk ? nk->stride(1) : 0, kp->size(0), nullptr, out.data_ptr(),
                        out.stride(0), out.stride(1), (int)batch, (int)heads, (int)kv_heads, (int)dim, (float)scaling,
                        (int)splits, (int)block_kv, need ? workspace.data_ptr() : nullptr, need,
                        code_of(q->scalar_type()), kv, (float)k_scale, (float)v_scale, (int)flags,
                        reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    // (An allocation that failed: the Python code tries it again and raises torch's own error.)
    Py_RETURN_NONE;
  }
}

// prefill(query, key_pool, value_pool, slot_table, context_lens, query_start_loc, max_query_len, scaling, groups,
//         block_kv, block_q, flags, k_scale, v_scale, out or None, stream) -> out, status, or None
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16 || !g_prefill) Py_RETURN_NONE;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &st = *t[3], &cl = *t[4], &qsl = *t[5];
  double scaling, k_scale, v_scale;
  int64_t longest, groups, block_kv, block_q, flags, stream;
  if (!integer(a[6], &longest) || !number(a[7], &scaling) || !integer(a[8], &groups) || !integer(a[9], &block_kv) ||
      !integer(a[10], &block_q) || !integer(a[11], &flags) || !number(a[12], &k_scale) || !number(a[13], &v_scale) ||
      !integer(a[15], &stream) || !pools_ok(kp, vp) || kp.size(0) >= (int64_t(1) << 31))
    Py_RETURN_NONE;
  const int kv = pool_code(q.scalar_type(), kp, k_scale, v_scale);
  if (kv < 0 || q.dim() != 3 || q.stride(2) != 1 || st.dim() != 2 || st.scalar_type() != at::kLong || st.stride(1) != 1 ||
      cl.dim() != 1 || cl.scalar_type() != at::kInt || cl.stride(0) != 1 || qsl.dim() != 1 ||
      qsl.scalar_type() != at::kInt || qsl.stride(0) != 1)
    Py_RETURN_NONE;
  const int64_t batch = cl.size(0), heads = q.size(1), dim = q.size(2), kv_heads = kp.size(1), width = st.size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (groups < 1 || heads % groups || heads / groups != kv_heads || dim != kp.size(2) || st.size(0) != batch ||
      qsl.size(0) != batch + 1 || batch < 1 || batch > kInt || heads > kInt || width > kInt || longest < 0 ||
      longest > kInt || block_kv < 0 || block_kv > kInt || block_q < 0 || block_q > kInt || flags < 0 || flags > kInt)
    Py_RETURN_NONE;
  const at::Tensor* given = nullptr;
  if (a[14] != Py_None) {
    given = plain(a[14]);
    if (!given || given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() ||
        given->device() != q.device() || given->stride(2) != 1)
      Py_RETURN_NONE;
  }
  size_t need = 0;
  if (g_prefill_plan((int)batch, (int)heads, (int)kv_heads, (int)dim, (int)width, 0, &need) != LI_OK) Py_RETURN_NONE;
  try {
    at::Tensor out, workspace;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      if (!given) out = at::empty_like(q);
      const at::Tensor& o = given ? *given : out;
      if (need) workspace = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      status = g_prefill(q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(), kp.stride(0), kp.stride(1),
                         st.const_data_ptr<int64_t>(), st.stride(0), (int)width, cl.const_data_ptr<int32_t>(),
                         qsl.const_data_ptr<int32_t>(), (int)batch, (int)longest, o.data_ptr(), o.stride(0), o.stride(1),
                         (int)heads, (int)kv_heads, (int)dim, (float)scaling, (int)block_q, (int)block_kv,
                         need ? workspace.data_ptr() : nullptr, need, code_of(q.scalar_type()), kv, (float)k_scale,
                         (float)v_scale, (int)flags, reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    if (given) return (Py_INCREF(a[14]), a[14]);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// rope(q, k, v, cos, sin, slots, key_pool, value_pool, k_scale, v_scale, bad_slots or None, stream)
//   -> rotated q, status, or None
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12 || !g_rope) Py_RETURN_NONE;
  const at::Tensor* t[8];
  for (int i = 0; i < 8; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cos = *t[3], &sin = *t[4], &slots = *t[5], &kp = *t[6], &vp = *t[7];
  double k_scale, v_scale;
  int64_t stream;
  if (!number(a[8], &k_scale) || !number(a[9], &v_scale) || !integer(a[11], &stream) || !pools_ok(kp, vp)) Py_RETURN_NONE;
  const auto dtype = q.scalar_type();
  const int kv = pool_code(dtype, kp, k_scale, v_scale);
  if (kv < 0 || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || cos.dim() != 3 || sin.dim() != 3) Py_RETURN_NONE;
  for (int i = 1; i < 5; ++i)
    if (t[i]->scalar_type() != dtype) Py_RETURN_NONE;
  const int64_t batch = q.size(0), heads = q.size(1), tokens = q.size(2), dim = q.size(3), kv_heads = k.size(1);
  if (k.sizes() != v.sizes() || k.size(0) != batch || k.size(2) != tokens || k.size(3) != dim || kv_heads != kp.size(1) ||
      dim != kp.size(2) || dim % 2 || cos.sizes() != sin.sizes() || cos.strides() != sin.strides() ||
      cos.size(1) != tokens || cos.size(2) != dim || (cos.size(0) != 1 && cos.size(0) != batch))
    Py_RETURN_NONE;
  if (slots.scalar_type() != at::kLong || !slots.is_contiguous() || slots.numel() != batch * tokens || slots.numel() < 1)
    Py_RETURN_NONE;
  int32_t* bad = nullptr;
  if (a[10] != Py_None) {
    const at::Tensor* b = plain(a[10]);
    if (!b || b->scalar_type() != at::kInt || b->numel() < 1 || b->device() != q.device()) Py_RETURN_NONE;
    bad = b->data_ptr<int32_t>();
  }
  const int64_t cs[3] = {cos.size(0) == 1 ? 0 : cos.stride(0), cos.stride(1), cos.stride(2)};
  try {
    at::Tensor out;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      out = at::empty({batch, tokens, heads, dim}, q.options()).transpose(1, 2);
      const int64_t os[4] = {out.stride(0), out.stride(1), out.stride(2), out.stride(3)};
      void* s = reinterpret_cast<void*>(stream);
      const int64_t* sl = slots.const_data_ptr<int64_t>();
      if (kv == LI_FP8_E4M3)
        status = g_rope_f8(q.data_ptr(), q.strides().data(), k.data_ptr(), k.strides().data(), v.data_ptr(),
                           v.strides().data(), cos.data_ptr(), sin.data_ptr(), cs, batch, tokens, sl, out.data_ptr(), os,
                           kp.data_ptr(), vp.data_ptr(), kp.size(0), kp.stride(0), kp.stride(1), (int)heads,
                           (int)kv_heads, (int)dim, code_of(dtype), (float)k_scale, (float)v_scale, bad, s);
      else
        status = g_rope(q.data_ptr(), q.strides().data(), k.data_ptr(), k.strides().data(), v.data_ptr(),
                        v.strides().data(), cos.data_ptr(), sin.data_ptr(), cs, batch, tokens, sl, out.data_ptr(), os,
                        kp.data_ptr(), vp.data_ptr(), kp.size(0), kp.stride(0), kp.stride(1), (int)heads, (int)kv_heads,
                        (int)dim, code_of(dtype), bad, s);
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// The slots of a block of an int8 pool with these scales, or 0: not what this serves.
int64_t block_of(const at::Tensor& kp, const at::Tensor& ks, const at::Tensor& vs) {
  if (kp.scalar_type() != at::kChar || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || ks.dim() != 2 ||
      ks.sizes() != vs.sizes() || ks.strides() != vs.strides() || ks.size(1) != kp.size(1) || ks.stride(1) != 1 ||
      ks.stride(0) < kp.size(1) || ks.size(0) < 1 || kp.size(0) % ks.size(0) || ks.device() != kp.device() ||
      vs.device() != kp.device())
    return 0;
  return kp.size(0) / ks.size(0);
}

bool rows_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// decode_int8(query, key_pool, value_pool, slot_table, context_lens, key_scales, value_scales, scaling, groups,
//             block_kv, num_splits (0: None), flags, stream) -> out, status, or None
PyObject* decode_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13 || !g_decode_int8) Py_RETURN_NONE;
  const at::Tensor* t[7];
  for (int i = 0; i < 7; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &st = *t[3], &cl = *t[4], &ks = *t[5], &vs = *t[6];
  double scaling;
  int64_t groups, block_kv, splits, flags, stream;
  if (!number(a[7], &scaling) || !integer(a[8], &groups) || !integer(a[9], &block_kv) || !integer(a[10], &splits) ||
      !integer(a[11], &flags) || !integer(a[12], &stream) || !pools_ok(kp, vp) || kp.size(0) >= (int64_t(1) << 31))
    Py_RETURN_NONE;
  const int64_t block = block_of(kp, ks, vs);
  if (!block || !rows_type(q.scalar_type()) || q.dim() != 3 || q.stride(2) != 1 || st.dim() != 2 ||
      st.scalar_type() != at::kLong || st.stride(1) != 1 || cl.dim() != 1 || cl.scalar_type() != at::kInt ||
      cl.stride(0) != 1)
    Py_RETURN_NONE;
  const int64_t batch = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = kp.size(1), width = st.size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (groups < 1 || heads % groups || heads / groups != kv_heads || dim != kp.size(2) || st.size(0) != batch ||
      cl.size(0) != batch || batch < 1 || batch > kInt || heads > kInt || width > kInt || splits < 0 || splits > kInt ||
      block_kv < 0 || block_kv > kInt || flags < 0 || flags > kInt || block > kInt)
    Py_RETURN_NONE;
  size_t need = 0;
  if (g_plan((int)batch, (int)heads, (int)kv_heads, (int)dim, (int)width, (int)splits, 0, (int)block_kv, nullptr, nullptr,
             &need) != LI_OK)
    Py_RETURN_NONE;
  try {
    at::Tensor out, workspace;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      out = at::empty_like(q);
      if (need) workspace = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      status = g_decode_int8(q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(),
                             ks.const_data_ptr<float>(), vs.const_data_ptr<float>(), (int)block, ks.stride(0), kp.stride(0),
                             kp.stride(1), st.const_data_ptr<int64_t>(), st.stride(0), (int)width,
                             cl.const_data_ptr<int32_t>(), out.data_ptr(), out.stride(0), out.stride(1), (int)batch,
                             (int)heads, (int)kv_heads, (int)dim, (float)scaling, (int)splits, (int)block_kv,
                             need ? workspace.data_ptr() : nullptr, need, code_of(q.scalar_type()), (int)flags,
                             reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// prefill_int8(query, key_pool, value_pool, slot_table, context_lens, query_start_loc, key_scales, value_scales,
//              max_query_len, context_tokens, scaling, groups, block_kv, block_q, flags, out or None, stream)
//   -> out, status, or None
PyObject* prefill_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 17 || !g_prefill_int8) Py_RETURN_NONE;
  const at::Tensor* t[8];
  for (int i = 0; i < 8; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &st = *t[3], &cl = *t[4], &qsl = *t[5], &ks = *t[6], &vs = *t[7];
  double scaling;
  int64_t longest, tokens, groups, block_kv, block_q, flags, stream;
  if (!integer(a[8], &longest) || !integer(a[9], &tokens) || !number(a[10], &scaling) || !integer(a[11], &groups) ||
      !integer(a[12], &block_kv) || !integer(a[13], &block_q) || !integer(a[14], &flags) || !integer(a[16], &stream) ||
      !pools_ok(kp, vp) || kp.size(0) >= (int64_t(1) << 31))
    Py_RETURN_NONE;
  const int64_t block = block_of(kp, ks, vs);
  if (!block || !rows_type(q.scalar_type()) || q.dim() != 3 || q.stride(2) != 1 || st.dim() != 2 ||
      st.scalar_type() != at::kLong || st.stride(1) != 1 || cl.dim() != 1 || cl.scalar_type() != at::kInt ||
      cl.stride(0) != 1 || qsl.dim() != 1 || qsl.scalar_type() != at::kInt || qsl.stride(0) != 1)
    Py_RETURN_NONE;
  const int64_t batch = cl.size(0), heads = q.size(1), dim = q.size(2), kv_heads = kp.size(1), width = st.size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (groups < 1 || heads % groups || heads / groups != kv_heads || dim != kp.size(2) || st.size(0) != batch ||
      qsl.size(0) != batch + 1 || batch < 1 || batch > kInt || heads > kInt || width > kInt || longest < 0 ||
      longest > kInt || tokens < 0 || block_kv < 0 || block_kv > kInt || block_q < 0 || block_q > kInt || flags < 0 ||
      flags > kInt || block > kInt)
    Py_RETURN_NONE;
  const at::Tensor* given = nullptr;
  if (a[15] != Py_None) {
    given = plain(a[15]);
    if (!given || given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() ||
        given->device() != q.device() || given->stride(2) != 1)
      Py_RETURN_NONE;
  }
  size_t need = 0;
  if (g_prefill_int8_plan((int)batch, (int)heads, (int)kv_heads, (int)dim, (int)width, (int)longest, tokens,
                          code_of(q.scalar_type()), &need) != LI_OK)
    Py_RETURN_NONE;
  try {
    at::Tensor out, workspace;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      if (!given) out = at::empty_like(q);
      const at::Tensor& o = given ? *given : out;
      if (need) workspace = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      status = g_prefill_int8(q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(),
                              ks.const_data_ptr<float>(), vs.const_data_ptr<float>(), (int)block, ks.stride(0),
                              kp.stride(0), kp.stride(1), st.const_data_ptr<int64_t>(), st.stride(0), (int)width,
                              cl.const_data_ptr<int32_t>(), qsl.const_data_ptr<int32_t>(), (int)batch, (int)longest, tokens,
                              o.data_ptr(), o.stride(0), o.stride(1), (int)heads, (int)kv_heads, (int)dim, (float)scaling,
                              (int)block_q, (int)block_kv, need ? workspace.data_ptr() : nullptr, need,
                              code_of(q.scalar_type()), (int)flags, reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    if (given) return (Py_INCREF(a[15]), a[15]);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// rope_int8(q, k, v, cos, sin, slots, key_pool, value_pool, key_scales, value_scales, bad_slots or None, stream)
//   -> rotated q, status, or None
PyObject* rope_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12 || !g_rope_int8) Py_RETURN_NONE;
  const at::Tensor* t[10];
  for (int i = 0; i < 10; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cos = *t[3], &sin = *t[4], &slots = *t[5], &kp = *t[6], &vp = *t[7],
                   &ks = *t[8], &vs = *t[9];
  int64_t stream;
  if (!integer(a[11], &stream) || !pools_ok(kp, vp)) Py_RETURN_NONE;
  const auto dtype = q.scalar_type();
  const int64_t block = block_of(kp, ks, vs);
  if (!block || !rows_type(dtype) || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || cos.dim() != 3 || sin.dim() != 3)
    Py_RETURN_NONE;
  for (int i = 1; i < 5; ++i)
    if (t[i]->scalar_type() != dtype) Py_RETURN_NONE;
  const int64_t batch = q.size(0), heads = q.size(1), tokens = q.size(2), dim = q.size(3), kv_heads = k.size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (k.sizes() != v.sizes() || k.size(0) != batch || k.size(2) != tokens || k.size(3) != dim || kv_heads != kp.size(1) ||
      dim != kp.size(2) || dim % 2 || cos.sizes() != sin.sizes() || cos.strides() != sin.strides() ||
      cos.size(1) != tokens || cos.size(2) != dim || (cos.size(0) != 1 && cos.size(0) != batch) || block > kInt ||
      heads > kInt || dim > kInt)
    Py_RETURN_NONE;
  if (slots.scalar_type() != at::kLong || !slots.is_contiguous() || slots.numel() != batch * tokens || slots.numel() < 1)
    Py_RETURN_NONE;
  int32_t* bad = nullptr;
  if (a[10] != Py_None) {
    const at::Tensor* b = plain(a[10]);
    if (!b || b->scalar_type() != at::kInt || b->numel() < 1 || b->device() != q.device()) Py_RETURN_NONE;
    bad = b->data_ptr<int32_t>();
  }
  const int64_t cs[3] = {cos.size(0) == 1 ? 0 : cos.stride(0), cos.stride(1), cos.stride(2)};
  try {
    at::Tensor out;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      out = at::empty({batch, tokens, heads, dim}, q.options()).transpose(1, 2);
      const int64_t os[4] = {out.stride(0), out.stride(1), out.stride(2), out.stride(3)};
      status = g_rope_int8(q.data_ptr(), q.strides().data(), k.data_ptr(), k.strides().data(), v.data_ptr(),
                           v.strides().data(), cos.data_ptr(), sin.data_ptr(), cs, batch, tokens,
                           slots.const_data_ptr<int64_t>(), out.data_ptr(), os, kp.data_ptr(), vp.data_ptr(),
                           ks.data_ptr<float>(), vs.data_ptr<float>(), kp.size(0), (int)block, kp.stride(0), kp.stride(1),
                           ks.stride(0), (int)heads, (int)kv_heads, (int)dim, code_of(dtype), bad,
                           reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// linear_int8(x, codes, scales, stream) -> out, status, or None
PyObject* linear_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 || !g_linear_int8) Py_RETURN_NONE;
  const at::Tensor* t[3];
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = plain(a[i])) || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  const at::Tensor &x = *t[0], &w = *t[1], &scales = *t[2];
  int64_t stream;
  if (!integer(a[3], &stream) || !rows_type(x.scalar_type()) || x.requires_grad() || x.dim() < 1 ||
      w.scalar_type() != at::kChar || w.dim() != 2 || w.stride(1) != 1 || scales.scalar_type() != at::kFloat ||
      scales.dim() != 1)
    Py_RETURN_NONE;
  const int64_t rows_n = w.size(0), k = w.size(1);
  constexpr int64_t kInt = 0x7fffffff;
  if (rows_n < 2 || k < 2 || rows_n > kInt || k > kInt || x.size(-1) != k || scales.size(0) != rows_n || scales.stride(0) != 1)
    Py_RETURN_NONE;
  // Rows of x evenly strided: contiguous, or two axes with the last one so.
  int64_t rows = x.numel() / k, x_s = k;
  if (x.dim() == 2 && x.stride(1) == 1) x_s = x.stride(0);
  else if (!x.is_contiguous()) Py_RETURN_NONE;
  const int64_t padded = (k + 15) / 16 * 16, stride = w.stride(0);
  if (rows < 1 || rows > kInt || x_s < 0 || stride % 16 || stride < padded ||
      reinterpret_cast<uintptr_t>(w.const_data_ptr()) % 16 ||
      w.storage_offset() + (rows_n - 1) * stride + padded > (int64_t)w.storage().nbytes())
    Py_RETURN_NONE;
  size_t need = 0;
  if (g_linear_int8_plan((int)rows, (int)rows_n, (int)k, &need) != LI_OK) Py_RETURN_NONE;
  try {
    at::Tensor out, workspace;
    int status;
    {
      Unlocked unlocked;
      at::AutoDispatchBelowADInplaceOrView below;
      c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
      shape.back() = rows_n;
      out = at::empty(shape, x.options());
      workspace = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
      status = g_linear_int8(x.data_ptr(), x_s, w.const_data_ptr(), stride, scales.const_data_ptr<float>(), out.data_ptr(),
                             rows_n, (int)rows, (int)rows_n, (int)k, workspace.data_ptr(), need, code_of(x.scalar_type()),
                             reinterpret_cast<void*>(stream));
    }
    if (status != LI_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(out));
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// bind_int8(decode, prefill plan, prefill, rope, linear plan, linear): the loaded library's entry points of the int8 calls.
PyObject* bind_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t p[6];
  for (int i = 0; i < 6; ++i)
    if (n != 6 || !integer(a[i], &p[i])) {
      PyErr_SetString(PyExc_TypeError, "bind_int8 takes six addresses");
      return nullptr;
    }
  g_decode_int8 = reinterpret_cast<decltype(g_decode_int8)>(p[0]);
  g_prefill_int8_plan = reinterpret_cast<decltype(g_prefill_int8_plan)>(p[1]);
  g_prefill_int8 = reinterpret_cast<decltype(g_prefill_int8)>(p[2]);
  g_rope_int8 = reinterpret_cast<decltype(g_rope_int8)>(p[3]);
  g_linear_int8_plan = reinterpret_cast<decltype(g_linear_int8_plan)>(p[4]);
  g_linear_int8 = reinterpret_cast<decltype(g_linear_int8)>(p[5]);
  Py_RETURN_NONE;
}

// bind(decode plan, decode_write, prefill plan, prefill, rope, rope_fp8): the loaded library's entry points, as addresses.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t p[6];
  for (int i = 0; i < 6; ++i)
    if (n != 6 || !integer(a[i], &p[i])) {
      PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
      return nullptr;
    }
  g_plan = reinterpret_cast<PlanFn>(p[0]);
  g_decode = reinterpret_cast<DecodeFn>(p[1]);
  g_prefill_plan = reinterpret_cast<PrefillPlanFn>(p[2]);
  g_prefill = reinterpret_cast<PrefillFn>(p[3]);
  g_rope = reinterpret_cast<RopeFn>(p[4]);
  g_rope_f8 = reinterpret_cast<RopeF8Fn>(p[5]);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"decode_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode_int8)), METH_FASTCALL, nullptr},
    {"prefill_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill_int8)), METH_FASTCALL, nullptr},
    {"rope_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_int8)), METH_FASTCALL, nullptr},
    {"linear_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_int8)), METH_FASTCALL, nullptr},
    {"bind_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_int8)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__fast_calls() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "build_id", LI_BUILD_ID) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
