// The Python side of the calls that a serving step makes once per layer (prism_amd/packed.py, rotate_qk): argument
// checks, result tensors and the call into libprism_kv.so, in one crossing.
//
// A step of a few decode tokens is host-bound: its kernels run 2 to 10 us.  The same checks in Python and the call
// through ctypes (25 to 30 arguments) took 16 to 22 us a call; here they take about 3, and the launch.  The entry
// points are the ones of include/prism_kv.h, found in the library that the package has loaded (attach).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <limits>
#include <string>

#include "../../include/prism_kv.h"

namespace {

// ---- the attached library ----
#define ENTRIES(X) X(pkv_rotate_qk) X(pkv_packed_rope_append) X(pkv_packed_attn) X(pkv_packed_workspace_bytes) \
  X(pkv_key_weights) X(pkv_key_weights_workspace_bytes) X(pkv_sample) X(pkv_sample_workspace_bytes) X(pkv_last_error)
#define DECLARE(name) decltype(&::name) lib_##name = nullptr;
ENTRIES(DECLARE)
PyObject* g_error = nullptr;  // PrismKVError

struct Failed {};  // the Python error is set

[[noreturn]] void refuse(const std::string& what) {
  PyErr_SetString(PyExc_RuntimeError, what.c_str());
  throw Failed{};
}
void check(int rc, const char* fn) {
  if (rc == PKV_OK) return;
  PyErr_Format(g_error, "%s failed (code %d): %s", fn, rc, lib_pkv_last_error());
  throw Failed{};
}

// ---- arguments ----
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor, not %s", name, Py_TYPE(o)->tp_name);
    throw Failed{};
  }
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed{};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Failed{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed{};
  return v != 0;
}
void* address(PyObject* o) { return reinterpret_cast<void*>(uintptr_t(integer(o))); }

std::string shape_of(const at::Tensor& t) { return c10::str(t.scalar_type(), " ", t.sizes()); }
void on_gpu(const at::Tensor& t, const char* name) {
  if (!t.is_cuda())
    refuse(c10::str(name, " must be a ROCm device tensor (got ", t.device(), "); prism_amd has no CPU path"));
}
void on_device(const at::Tensor& t, const char* name, c10::Device d) {
  if (t.device() != d) refuse(c10::str(name, " must be on ", d, ", not ", t.device()));
}

// The word that a kernel sets its error bits in.
int32_t* status_word(PyObject* o, c10::Device d) {
  const at::Tensor& t = tensor(o, "status");
  if (t.scalar_type() != at::kInt || t.numel() < 1 || t.device() != d)
    refuse(c10::str("status must be an int32 word on ", d, ", got ", shape_of(t), " on ", t.device()));
  return t.data_ptr<int32_t>();
}

// The tables' rotary_dim.
int rotary_dim(const at::Tensor& cos, const at::Tensor& sin, int64_t head_dim, c10::Device d) {
  const at::Tensor* tables[] = {&cos, &sin};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *tables[i];
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || !t.is_contiguous() || t.device() != d)
      refuse(c10::str(i ? "sin" : "cos", " must be a contiguous float32 [n_pos, rotary_dim / 2] table on ", d,
                      " (rotary_tables), got ", shape_of(t)));
  }
  if (cos.sizes() != sin.sizes() || cos.size(0) == 0 || cos.size(1) == 0)
    refuse(c10::str("cos ", cos.sizes(), " and sin ", sin.sizes(), " must have one shape, not empty"));
  if (cos.size(0) > std::numeric_limits<int32_t>::max()) refuse("cos and sin have more than 2^31 - 1 rows");
  if (2 * cos.size(1) > head_dim)
    refuse(c10::str("tables for a rotary_dim of ", 2 * cos.size(1), " do not fit head_dim ", head_dim));
  return int(2 * cos.size(1));
}

const void* norm_weight(PyObject* o, const char* name, int64_t head_dim, at::ScalarType dtype, c10::Device d) {
  if (!given(o)) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != dtype || t.dim() != 1 || t.size(0) != head_dim || !t.is_contiguous() || t.device() != d)
    refuse(c10::str(name, " must be a contiguous ", dtype, " [", head_dim, "] vector on ", d, ", got ", shape_of(t)));
  return t.data_ptr();
}

struct Rows {
  int64_t token, head;  // strides
};
// [..., heads, head_dim] as [tokens, heads, head_dim], without a copy.
Rows token_rows(const at::Tensor& t, const char* name, int64_t tokens) {
  const int64_t dims = t.dim(), hd = t.size(dims - 1);
  if (t.stride(dims - 1) != 1 && hd > 1) refuse(c10::str(name, " must be contiguous in head_dim"));
  if (tokens <= 1) return {0, t.stride(dims - 2)};
  int64_t stride = 0, covered = 1;  // tokens counted so far, from the innermost dimension
  for (int64_t i = dims - 3; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (covered == 1)
      stride = t.stride(i);
    else if (t.stride(i) != stride * covered)
      refuse(c10::str(name, " must flatten to a token axis without a copy"));
    covered *= t.size(i);
  }
  return {stride, t.stride(dims - 2)};
}

// ---- rotate_qk ----
PyObject* rotate_qk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) return PyErr_Format(PyExc_TypeError, "rotate_qk takes 13 arguments");
  try {
    const at::Tensor& q = tensor(a[0], "q");
    on_gpu(q, "q");
    const auto dtype = q.scalar_type();
    const int code = dtype == at::kBFloat16 ? PKV_BF16 : dtype == at::kHalf ? PKV_FP16 : dtype == at::kFloat ? PKV_FP32 : -1;
    if (code < 0) refuse(c10::str("q must be bfloat16, float16 or float32, got ", dtype));
    int32_t* const status = status_word(a[11], q.device());
    const int64_t dims = q.dim();
    if (dims < 3) refuse(c10::str("q must be [..., n_heads, head_dim] with a token axis, got ", q.sizes()));
    const c10::Device dev = q.device();
    const int64_t hd = q.size(dims - 1), nh = q.size(dims - 2);
    int64_t tokens = 1;
    for (int64_t i = 0; i < dims - 2; ++i) tokens *= q.size(i);
    const at::Tensor &pos = tensor(a[2], "positions"), &cos = tensor(a[3], "cos"), &sin = tensor(a[4], "sin");
    const int rd = rotary_dim(cos, sin, hd, dev);
    const void* qw = norm_weight(a[6], "q_norm_w", hd, dtype, dev);
    if (pos.scalar_type() != at::kInt || pos.device() != dev || pos.numel() != tokens || !pos.is_contiguous())
      refuse(c10::str("positions must be contiguous int32, one for each of the ", tokens, " tokens, on ", dev));
    const bool has_k = given(a[1]);
    if (!has_k && (given(a[7]) || given(a[10]))) refuse("k_norm_w and k_out need a k");
    const void* kw = norm_weight(a[7], "k_norm_w", hd, dtype, dev);
    at::Tensor q_out, k_out;
    auto result = [&](PyObject* o, const char* name, const at::Tensor& like) {
      if (!given(o)) return at::empty(like.sizes(), like.options().requires_grad(false));
      const at::Tensor& t = tensor(o, name);
      if (t.scalar_type() != dtype || t.device() != dev || t.sizes() != like.sizes())
        refuse(c10::str(name, " must be ", dtype, " ", like.sizes(), " on ", dev, ", got ", shape_of(t)));
      return t;
    };
    const void* k_ptr = nullptr;
    void* ko_ptr = nullptr;
    Rows kr = {0, 0}, ko = {0, 0};
    int64_t nk = 0;
    if (has_k) {
      const at::Tensor& k = tensor(a[1], "k");
      bool same = k.scalar_type() == dtype && k.device() == dev && k.dim() == dims;
      for (int64_t i = 0; same && i < dims; ++i) same = i == dims - 2 || k.size(i) == q.size(i);
      if (!same) refuse(c10::str("k ", shape_of(k), " must match q ", shape_of(q), " but for the heads"));
      nk = k.size(dims - 2);
      k_out = result(a[10], "k_out", k);
      kr = token_rows(k, "k", tokens);
      ko = token_rows(k_out, "k_out", tokens);
      k_ptr = k.data_ptr();
      ko_ptr = k_out.data_ptr();
    }
    q_out = result(a[9], "q_out", q);
    const Rows qr = token_rows(q, "q", tokens), qo = token_rows(q_out, "q_out", tokens);
    if (hd > 1024 || nh + nk > 65536)
      refuse(c10::str(nh, " + ", nk, " heads of ", hd, ": at most 65536 heads of at most 1024 elements"));
    if (tokens > 0 && nh + nk > 0)
      check(lib_pkv_rotate_qk(q.data_ptr(), qr.token, qr.head, k_ptr, kr.token, kr.head, pos.data_ptr<int32_t>(),
                              cos.data_ptr<float>(), sin.data_ptr<float>(), int32_t(cos.size(0)), qw, kw,
                              float(real(a[8])), q_out.data_ptr(), qo.token, qo.head, ko_ptr, ko.token, ko.head, tokens,
                              int32_t(nh), int32_t(nk), int32_t(hd), rd, truth(a[5]) ? 1 : 0, code,
                              status, address(a[12])),
            "pkv_rotate_qk");
    PyObject* kobj = has_k ? THPVariable_Wrap(k_out) : (Py_INCREF(Py_None), Py_None);
    return Py_BuildValue("(NN)", THPVariable_Wrap(q_out), kobj);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---- the batch ----
struct Batch {
  int64_t tokens, batch, n_heads, n_kv, head_dim, page_size, num_pages, max_blocks;
  const int32_t *positions, *slots, *block_table;
  c10::Device device;
};
constexpr const char* kBatchName = "prism_amd.PackedBatch";
void drop_batch(PyObject* capsule) { delete static_cast<Batch*>(PyCapsule_GetPointer(capsule, kBatchName)); }

// new_batch(a tensor of the batch's device, the sizes, the addresses of positions, slots and block_table)
PyObject* new_batch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) return PyErr_Format(PyExc_TypeError, "new_batch takes 12 arguments");
  try {
    int64_t v[8];
    for (int i = 0; i < 8; ++i) v[i] = integer(a[1 + i]);
    Batch* b = new Batch{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], static_cast<int32_t*>(address(a[9])),
                         static_cast<int32_t*>(address(a[10])), static_cast<int32_t*>(address(a[11])),
                         tensor(a[0], "buffer").device()};
    return PyCapsule_New(b, kBatchName, drop_batch);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
const Batch& batch_of(PyObject* o) {
  auto* b = static_cast<Batch*>(PyCapsule_GetPointer(o, kBatchName));
  if (!b) throw Failed{};
  return *b;
}

// The caches' page stride.
int64_t check_cache(const at::Tensor& k, const at::Tensor& v, const Batch& b) {
  const at::Tensor* both[] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *both[i];
    const char* name = i ? "v_cache" : "k_cache";
    on_gpu(t, name);
    if (t.scalar_type() != at::kBFloat16) refuse(c10::str(name, " must be bfloat16, got ", t.scalar_type()));
    if (t.dim() != 4) refuse(c10::str(name, " must be [num_pages, page_size, n_kv, head_dim]"));
    on_device(t, name, b.device);
  }
  if (k.sizes() != v.sizes() || k.strides() != v.strides())
    refuse("k_cache and v_cache must have the same shape and strides");
  if (k.size(1) != b.page_size || k.size(2) != b.n_kv || k.size(3) != b.head_dim || k.size(0) < b.num_pages)
    refuse(c10::str("cache of ", k.sizes(), " does not fit a batch laid out for [", b.num_pages, ", ", b.page_size, ", ",
                    b.n_kv, ", ", b.head_dim, "]"));
  if (k.stride(1) != b.n_kv * b.head_dim || k.stride(2) != b.head_dim || k.stride(3) != 1)
    refuse("k_cache/v_cache must be contiguous within a page");
  return k.stride(0);
}

Rows check_rows(const at::Tensor& t, const char* name, const Batch& b) {
  on_gpu(t, name);
  if (t.scalar_type() != at::kBFloat16) refuse(c10::str(name, " must be bfloat16, got ", t.scalar_type()));
  if (t.dim() != 3 || t.size(0) < b.tokens || t.size(1) != b.n_heads || t.size(2) != b.head_dim)
    refuse(c10::str(name, " has shape ", t.sizes(), ", expected [>= ", b.tokens, ", ", b.n_heads, ", ", b.head_dim, "]"));
  if (t.stride(2) != 1) refuse(c10::str(name, " must be contiguous in head_dim"));
  on_device(t, name, b.device);
  return {t.stride(0), t.stride(1)};
}

// A result of `rows` rows, zero behind the batch's tokens.
at::Tensor new_rows(at::IntArrayRef sizes, at::ScalarType dtype, const Batch& b) {
  at::Tensor t = at::empty(sizes, at::TensorOptions().dtype(dtype).device(b.device));
  if (sizes[0] > b.tokens) t.narrow(0, b.tokens, sizes[0] - b.tokens).zero_();
  return t;
}

PyObject* packed_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14) return PyErr_Format(PyExc_TypeError, "packed_rope_append takes 14 arguments");
  try {
    const at::Tensor &qkv = tensor(a[0], "qkv"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache");
    const Batch& b = batch_of(a[3]);
    on_gpu(qkv, "qkv");
    int32_t* const status = status_word(a[12], b.device);
    const int64_t page_stride = check_cache(kc, vc, b);
    const int64_t width = (b.n_heads + 2 * b.n_kv) * b.head_dim;
    if (qkv.scalar_type() != at::kBFloat16 || qkv.dim() != 2 || qkv.size(0) < b.tokens || qkv.size(1) != width ||
        qkv.stride(1) != 1)
      refuse(c10::str("qkv must be bfloat16 [>= ", b.tokens, ", ", width, "], contiguous in its last dimension, got ",
                      shape_of(qkv)));
    on_device(qkv, "qkv", b.device);
    const at::Tensor &cos = tensor(a[4], "cos"), &sin = tensor(a[5], "sin");
    const int rd = rotary_dim(cos, sin, b.head_dim, b.device);
    const void* qw = norm_weight(a[7], "q_norm_w", b.head_dim, at::kBFloat16, b.device);
    const void* kw = norm_weight(a[8], "k_norm_w", b.head_dim, at::kBFloat16, b.device);
    const int32_t* positions = b.positions;
    if (given(a[10])) {
      const at::Tensor& p = tensor(a[10], "positions");
      if (p.scalar_type() != at::kInt || p.dim() != 1 || p.size(0) < b.tokens || p.device() != b.device ||
          (b.tokens > 1 && p.stride(0) != 1))
        refuse(c10::str("positions must be contiguous int32 [>= ", b.tokens, "] on ", b.device));
      positions = p.data_ptr<int32_t>();
    }
    at::Tensor q_out;
    Rows qo;
    if (given(a[11])) {
      q_out = tensor(a[11], "q_out");
      qo = check_rows(q_out, "q_out", b);
    } else {
      q_out = new_rows({qkv.size(0), b.n_heads, b.head_dim}, at::kBFloat16, b);
      qo = {b.n_heads * b.head_dim, b.head_dim};
    }
    if (b.tokens > 0)
      check(lib_pkv_packed_rope_append(
                qkv.data_ptr(), qkv.stride(0), positions, b.slots, cos.data_ptr<float>(), sin.data_ptr<float>(),
                int32_t(cos.size(0)), qw, kw, float(real(a[9])), q_out.data_ptr(), qo.token, qo.head, kc.data_ptr(),
                vc.data_ptr(), page_stride, b.tokens, int32_t(b.n_heads), int32_t(b.n_kv), int32_t(b.head_dim), rd,
                truth(a[6]) ? 1 : 0, int32_t(b.page_size), int32_t(b.num_pages),
                status, address(a[13])),
            "pkv_packed_rope_append");
    return THPVariable_Wrap(q_out);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// packed_attention(q, k_cache, v_cache, batch, plan (window, items, n_items, merges, n_merges, partials, merge_rows),
// sinks, softmax_scale or None, return_lse, out, status, stream)
PyObject* packed_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return PyErr_Format(PyExc_TypeError, "packed_attention takes 11 arguments");
  try {
    const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache");
    const Batch& b = batch_of(a[3]);
    const Rows qr = check_rows(q, "q", b);
    int32_t* const status = status_word(a[9], b.device);
    const int64_t page_stride = check_cache(kc, vc, b);
    if (!PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 7) refuse("a plan has 7 entries");
    int64_t plan[7];
    for (int i = 0; i < 7; ++i) plan[i] = integer(PyTuple_GET_ITEM(a[4], i));
    const float* sinks = nullptr;
    if (given(a[5])) {
      const at::Tensor& t = tensor(a[5], "sinks");
      if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != b.n_heads || !t.is_contiguous() ||
          t.device() != b.device)
        refuse(c10::str("sinks must be a contiguous float32 [", b.n_heads, "] vector on ", b.device, ", got ", shape_of(t)));
      sinks = t.data_ptr<float>();
    }
    const double scale = given(a[6]) ? real(a[6]) : 1.0 / std::sqrt(double(b.head_dim));
    const bool want_lse = truth(a[7]);
    at::Tensor out, lse, ws;
    Rows o;
    if (given(a[8])) {
      out = tensor(a[8], "out");
      o = check_rows(out, "out", b);
    } else {
      out = new_rows(q.sizes(), at::kBFloat16, b);
      o = {b.n_heads * b.head_dim, b.head_dim};
    }
    if (want_lse) lse = new_rows({q.size(0), b.n_heads}, at::kFloat, b);
    if (b.tokens > 0) {
      // the partials of this call alone, from torch's allocator: of the current stream, or of the graph it captures
      const size_t bytes = lib_pkv_packed_workspace_bytes(int32_t(plan[5]), int32_t(b.n_kv), int32_t(b.head_dim));
      if (bytes) ws = at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(b.device));
      check(lib_pkv_packed_attn(
                q.data_ptr(), qr.token, qr.head, kc.data_ptr(), vc.data_ptr(), page_stride, b.block_table, b.max_blocks,
                out.data_ptr(), o.token, o.head, want_lse ? lse.data_ptr<float>() : nullptr, sinks,
                reinterpret_cast<const int32_t*>(plan[1]), int32_t(plan[2]), reinterpret_cast<const int32_t*>(plan[3]),
                int32_t(plan[4]), int32_t(plan[5]), int32_t(plan[6]), bytes ? ws.data_ptr() : nullptr, bytes,
                int32_t(b.tokens), int32_t(b.batch), int32_t(b.n_heads), int32_t(b.n_kv), int32_t(b.head_dim),
                int32_t(b.page_size), int32_t(b.num_pages), int32_t(b.max_blocks), int32_t(plan[0]), float(scale),
                status, address(a[10])),
            "pkv_packed_attn");
    }
    if (!want_lse) return THPVariable_Wrap(out);
    return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// packed_key_weights(q, k_cache, lse, key_weights, batch, plan (window, items, the lists' three counts, partials),
// softmax_scale or None, status, stream)
PyObject* packed_key_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return PyErr_Format(PyExc_TypeError, "packed_key_weights takes 9 arguments");
  try {
    const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &lse = tensor(a[2], "lse"),
                     &w = tensor(a[3], "key_weights");
    const Batch& b = batch_of(a[4]);
    const Rows qr = check_rows(q, "q", b);
    int32_t* const status = status_word(a[7], b.device);
    const int64_t page_stride = check_cache(kc, kc, b);
    on_gpu(lse, "lse");
    if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) < b.tokens || lse.size(1) != b.n_heads ||
        (b.n_heads > 1 && lse.stride(1) != 1) || (b.tokens > 1 && lse.stride(0) < b.n_heads))
      refuse(c10::str("lse must be float32 [>= ", b.tokens, ", ", b.n_heads, "], contiguous in its last dimension, got ",
                      shape_of(lse)));
    on_device(lse, "lse", b.device);
    on_gpu(w, "key_weights");
    if (w.scalar_type() != at::kFloat || w.dim() != 3 || w.size(0) < b.num_pages || w.size(1) != b.n_kv ||
        w.size(2) != b.page_size || w.stride(2) != 1 || (b.n_kv > 1 && w.stride(1) != b.page_size) ||
        (w.size(0) > 1 && w.stride(0) < b.n_kv * b.page_size))
      refuse(c10::str("key_weights must be float32 [>= ", b.num_pages, ", ", b.n_kv, ", ", b.page_size,
                      "], contiguous within a page, got ", shape_of(w)));
    on_device(w, "key_weights", b.device);
    if (!PyTuple_Check(a[5]) || PyTuple_GET_SIZE(a[5]) != 6) refuse("a plan of key weights has 6 entries");
    int64_t plan[6];
    for (int i = 0; i < 6; ++i) plan[i] = integer(PyTuple_GET_ITEM(a[5], i));
    const double scale = given(a[6]) ? real(a[6]) : 1.0 / std::sqrt(double(b.head_dim));
    if (b.tokens > 0) {
      // the partial sums of this call alone, from torch's allocator: of the current stream, or of the graph it captures
      at::Tensor ws;
      const size_t bytes = lib_pkv_key_weights_workspace_bytes(int32_t(plan[5]), int32_t(b.n_kv));
      if (bytes) ws = at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(b.device));
      check(lib_pkv_key_weights(
                q.data_ptr(), qr.token, qr.head, kc.data_ptr(), page_stride, lse.data_ptr<float>(),
                b.tokens > 1 ? lse.stride(0) : b.n_heads, w.data_ptr<float>(),
                w.size(0) > 1 ? w.stride(0) : b.n_kv * b.page_size, b.block_table, b.max_blocks,
                reinterpret_cast<const int32_t*>(plan[1]), int32_t(plan[2]), int32_t(plan[3]), int32_t(plan[4]),
                int32_t(plan[5]), bytes ? ws.data_ptr() : nullptr, bytes, int32_t(b.tokens), int32_t(b.batch),
                int32_t(b.n_heads), int32_t(b.n_kv), int32_t(b.head_dim), int32_t(b.page_size), int32_t(b.num_pages),
                int32_t(b.max_blocks), int32_t(plan[0]), float(scale), status, address(a[8])),
            "pkv_key_weights");
    }
    return THPVariable_Wrap(w);
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// A setting: a number for every row, or a tensor with one a row.
struct Setting {
  const void* rows = nullptr;
  double all = 0;
};
Setting setting(PyObject* o, const char* name, double none, bool whole, int64_t rows, c10::Device d) {
  if (!given(o)) return {nullptr, none};
  if (!THPVariable_Check(o)) {
    if (whole) {
      const int64_t v = integer(o);
      return {nullptr, double(v < 0 ? 0 : v > 0x7fffffff ? 0x7fffffff : v)};
    }
    const double v = real(o);
    if (std::isnan(v)) refuse(c10::str(name, " is not a number"));
    return {nullptr, v};
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  const auto type = whole ? at::kInt : at::kFloat;
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != rows || !t.is_contiguous() || t.device() != d)
    refuse(c10::str(name, " must be a number, or contiguous ", type, " [", rows, "] on ", d, ", got ", shape_of(t), " on ",
                    t.device()));
  return {t.data_ptr(), 0};
}

// sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, return_logprobs, stream)
PyObject* sample_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "sample_tokens takes 8 arguments");
  try {
    const at::Tensor &x = tensor(a[0], "logits"), &u = tensor(a[1], "uniforms");
    on_gpu(x, "logits");
    const auto dtype = x.scalar_type();
    const int code = dtype == at::kBFloat16 ? PKV_BF16 : dtype == at::kHalf ? PKV_FP16 : dtype == at::kFloat ? PKV_FP32 : -1;
    if (code < 0) refuse(c10::str("logits must be bfloat16, float16 or float32, got ", dtype));
    if (x.dim() != 2 || x.size(1) < 1 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1)))
      refuse(c10::str("logits must be [rows, vocab], contiguous in vocab and not empty there, got ", shape_of(x)));
    const int64_t rows = x.size(0), vocab = x.size(1);
    if (vocab > 1000000 || rows > 65535) refuse(c10::str("at most 65535 rows of 1000000 tokens, got ", x.sizes()));
    const c10::Device dev = x.device();
    if (u.scalar_type() != at::kFloat || u.dim() != 1 || u.size(0) != rows || !u.is_contiguous() || u.device() != dev)
      refuse(c10::str("uniforms must be contiguous float32 [", rows, "] on ", dev, ", got ", shape_of(u), " on ", u.device()));
    const Setting t = setting(a[2], "temperature", 1.0, false, rows, dev), k = setting(a[3], "top_k", 0.0, true, rows, dev),
                  p = setting(a[4], "top_p", 1.0, false, rows, dev), m = setting(a[5], "min_p", 0.0, false, rows, dev);
    if (!t.rows && t.all < 0) refuse("temperature must not be negative (0: the largest logit)");
    const bool logs = truth(a[6]);
    at::Tensor tokens = at::empty({rows}, at::TensorOptions().dtype(at::kLong).device(dev)), lp;
    if (logs) lp = at::empty({rows}, at::TensorOptions().dtype(at::kFloat).device(dev));
    if (rows > 0) {
      // of this call alone, from torch's allocator: of the current stream, or of the graph it captures
      const size_t bytes = lib_pkv_sample_workspace_bytes(int32_t(rows), int32_t(vocab));
      at::Tensor ws = at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(dev));
      check(lib_pkv_sample(x.data_ptr(), rows > 1 ? x.stride(0) : vocab, code, u.data_ptr<float>(),
                           static_cast<const float*>(t.rows), float(t.all), static_cast<const int32_t*>(k.rows),
                           int32_t(k.all), static_cast<const float*>(p.rows), float(p.all),
                           static_cast<const float*>(m.rows), float(m.all),
                           tokens.data_ptr<int64_t>(), logs ? lp.data_ptr<float>() : nullptr, int32_t(rows),
                           int32_t(vocab), ws.data_ptr(), bytes, address(a[7])),
            "pkv_sample");
    }
    if (!logs) return THPVariable_Wrap(tokens);
    return Py_BuildValue("(NN)", THPVariable_Wrap(tokens), THPVariable_Wrap(lp));
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// attach(handle of a loaded libprism_kv.so, the exception class for its errors)
PyObject* attach(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "attach takes 2 arguments");
  void* lib = PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
#define FIND(name)                                                                  \
  if (!(lib_##name = reinterpret_cast<decltype(lib_##name)>(dlsym(lib, #name)))) \
    return PyErr_Format(PyExc_RuntimeError, "%s not in the library", #name);
  ENTRIES(FIND)
  Py_XDECREF(g_error);
  Py_INCREF(g_error = a[1]);
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(attach), METHOD(rotate_qk), METHOD(new_batch), METHOD(packed_rope_append),
                         METHOD(packed_attention), METHOD(packed_key_weights), METHOD(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_fastcall", "per-layer calls into libprism_kv.so", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall() { return PyModule_Create(&module_def); }
