// fa2_torch.cpp - fa2/_torch_call.so: the common calls of fa2.kernel.attention and of the serving operators
// (fa2.rotary, fa2.packed, fa2.paged, fa2.pages), made natively.
//
// attention()'s checks, policy, allocations and launch took 11-17 us per call in Python and ctypes
// (a causal call of B1 H4 N256 D64 11.2 us, a split-KV one 16.5), more than the kernels of a short
// prompt or a decoding step run for (5-10 us), so back-to-back calls waited for the host. Here the
// same steps on at::Tensor take about 4 us, the launch included.
//
// call() takes exactly the calls that need nothing else: plain dense GPU tensors of the current
// device that satisfy every check of attention() and the library's 16-byte rule, with default
// tiles, packing and split count. Anything else returns None, and attention()'s Python does it: it
// raises the reference's errors, copies tensors the kernel cannot load, switches devices, honours
// the overrides. No state is kept from one call to the next.
#include <Python.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/PythonTorchFunctionTLS.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "fa2_fwd.h"

namespace {

constexpr double kLog2e = 1.4426950408889634;       // fa2/kernel.py: LOG2E
constexpr int64_t kMaxKvRowStride = int64_t(1) << 22;  // fa2/kernel.py: _MAX_KV_ROW_STRIDE
constexpr int kMaxDevices = 64;

// The device's CU count, as torch.cuda.get_device_properties reports it; 0 if unknown.
int cu_count(int dev) {
  static std::atomic<int> cus[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return 0;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
      (void)hipGetLastError();
      return 0;
    }
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// A tensor whose memory the kernel may address through data_ptr: no subclass, no wrapper of a
// transform, strided and on the GPU.
bool plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.dim() == 4 && t.layout() == at::kStrided && t.is_cuda() &&
         t.has_storage() && !t.is_conj() && !t.is_neg() && !at::isTensorSubclassLike(t);
}

// The element strides the library takes (0 for a dimension of one element, which it never steps),
// and whether its 16-byte loads can address the tensor: fa2/kernel.py's _loadable.
bool strides_of(const at::Tensor& t, int64_t max_row, int64_t (&s)[4]) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || t.stride(3) != 1) return false;
  for (int i = 0; i < 3; ++i) {
    s[i] = t.size(i) == 1 ? 0 : t.stride(i);
    if (s[i] % 8) return false;
  }
  s[3] = 1;
  return s[2] <= max_row;
}

// attention()'s policy at the default tiles: packing, split count and workspace. The count is the one
// that runs, which needs the smaller workspace, unless the workspace has room for the key-norm table:
// the kernel that uses the table takes fa2_num_splits's count, as fa2_launch_splits's contract says.
struct Policy {
  int32_t bm = 0, bn = 0, pack = 1, splits = 1;
  size_t ws_bytes = 0;
};
bool policy_of(int32_t B, int32_t hq, int32_t hkv, int32_t nq, int32_t nkv, int32_t D, int32_t dtype,
               int32_t causal, int32_t cus, Policy* out) {
  Policy p;
  if (fa2_default_config(D, &p.bm, &p.bn, nullptr, nullptr) != FA2_OK) return false;
  if (fa2_should_pack_gqa(nq, hq / hkv, p.bm)) p.pack = hq / hkv;
  if (!causal) p.splits = fa2_num_splits(B, hq, hkv, nq, nkv, D, 0, p.bm, p.bn, cus);
  p.ws_bytes = fa2_workspace_bytes_for(B, hq, hkv, nq, nkv, D, dtype, causal, p.splits);
  if (p.splits > 1 && p.ws_bytes == fa2_workspace_bytes(B, hq, nq, D, p.splits)) {
    p.splits = fa2_launch_splits(B, hq, hkv, nq, nkv, D, 0, p.bm, p.bn, cus, p.splits);
    p.ws_bytes = fa2_workspace_bytes(B, hq, nq, D, p.splits);
  }
  *out = p;
  return true;
}

// policy(batch, h_q, h_kv, n_q, n_kv, head_dim, dtype, causal, cus) -> (pack, splits, workspace bytes)
// of a call of these sizes on a GPU of `cus` CUs (dtype: the C ABI's code). No GPU call.
PyObject* policy(PyObject*, PyObject* args) {
  int B, hq, hkv, nq, nkv, D, dtype, causal, cus;
  if (!PyArg_ParseTuple(args, "iiiiiiiii", &B, &hq, &hkv, &nq, &nkv, &D, &dtype, &causal, &cus))
    return nullptr;
  Policy p;
  if (B < 1 || hkv < 1 || hq < 1 || hq % hkv || nq < 1 || nkv < 1 || cus < 1 ||
      !policy_of(B, hq, hkv, nq, nkv, D, dtype, causal, cus, &p)) {
    PyErr_SetString(PyExc_ValueError, "sizes that attention() rejects");
    return nullptr;
  }
  return Py_BuildValue("iin", p.pack, p.splits, (Py_ssize_t)p.ws_bytes);
}

// call(q, k, v, causal, sm_scale, return_lse) -> attention()'s result, or None (see above)
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6) {
    PyErr_SetString(PyExc_TypeError, "call(q, k, v, causal, sm_scale, return_lse)");
    return nullptr;
  }
  if (!plain(args[0]) || !plain(args[1]) || !plain(args[2]) ||
      c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  const int causal = PyObject_IsTrue(args[3]);
  const int want_lse = PyObject_IsTrue(args[5]);
  if (causal < 0 || want_lse < 0) return nullptr;

  // ---- attention()'s checks (fa2/kernel.py:218-228 of the reference)
  const int64_t B = q.size(0), hq = q.size(1), nq = q.size(2), D = q.size(3);
  const int64_t hkv = k.size(1), nkv = k.size(2);
  const auto dtype = q.scalar_type();
  if ((dtype != at::kHalf && dtype != at::kBFloat16) || k.scalar_type() != dtype ||
      v.scalar_type() != dtype || k.sizes() != v.sizes() || k.size(0) != B || k.size(3) != D ||
      (D != 16 && D != 32 && D != 64 && D != 128))
    Py_RETURN_NONE;
  if (B < 1 || hkv < 1 || hq < 1 || nq < 1 || nkv < 1 || hq % hkv || (causal && nq != nkv) ||
      B > INT32_MAX || hq > INT32_MAX || nq > INT32_MAX || nkv > INT32_MAX)
    Py_RETURN_NONE;
  const auto device = q.device();
  if (k.device() != device || v.device() != device || device.index() != c10::hip::current_device())
    Py_RETURN_NONE;
  double sm_scale = 1.0 / std::sqrt((double)D);
  if (args[4] != Py_None) {
    if (!PyFloat_CheckExact(args[4])) Py_RETURN_NONE;
    sm_scale = PyFloat_AS_DOUBLE(args[4]);
    if (!(sm_scale > 0)) Py_RETURN_NONE;
  }
  int64_t sq[4], sk[4], sv[4], so[4];
  if (!strides_of(q, INT64_MAX, sq) || !strides_of(k, kMaxKvRowStride, sk) ||
      !strides_of(v, kMaxKvRowStride, sv))
    Py_RETURN_NONE;

  const int cus = causal ? 1 : cu_count(device.index());
  const int32_t code = dtype == at::kBFloat16 ? FA2_DTYPE_BF16 : FA2_DTYPE_F16;
  Policy p;
  if (cus < 1 || nq > INT32_MAX / (hq / hkv) ||
      !policy_of((int32_t)B, (int32_t)hq, (int32_t)hkv, (int32_t)nq, (int32_t)nkv, (int32_t)D, code,
                 causal, cus, &p))
    Py_RETURN_NONE;

  // ---- outputs, workspace, launch
  at::Tensor out = at::empty_like(q);
  if (!strides_of(out, INT64_MAX, so)) Py_RETURN_NONE;
  at::Tensor lse, ws;
  if (want_lse) lse = at::empty({B, hq, nq}, q.options().dtype(at::kFloat));
  if (p.ws_bytes) ws = at::empty({(int64_t)p.ws_bytes}, q.options().dtype(at::kByte));
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void *qp = q.data_ptr(), *kp = k.data_ptr(), *vp = v.data_ptr();
  void* op = out.data_ptr();
  float* lp = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  void* wp = p.ws_bytes ? ws.data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS  // as ctypes does around a foreign call
  rc = fa2_attn_fwd_ex(qp, kp, vp, op, sq, sk, sv, so, (int32_t)B, (int32_t)hq, (int32_t)hkv,
                       (int32_t)nq, (int32_t)nkv, (int32_t)D, code, causal, p.pack, p.bm, p.bn,
                       (float)(sm_scale * kLog2e), lp, p.splits, wp, p.ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;  // nothing ran: attention() repeats the call and raises
  PyObject* o = THPVariable_Wrap(std::move(out));
  if (!o || !want_lse) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  if (!l) {
    Py_DECREF(o);
    return nullptr;
  }
  PyObject* both = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return both;
  END_HANDLE_TH_ERRORS
}

// ---- the serving operators: each takes its Python function's call when every tensor is plain, on the current
// device and as the kernels address it, and returns None otherwise. What the C ABI checks is left to it: a
// refused call returns None too, and Python repeats it and raises. Python's own work for such calls took 13-46 us
// (a rotation 16 us, a cache write and read back 46), their kernels 4-10.

// A plain tensor of `dim` dimensions on the current device, or null
const at::Tensor* tensor_of(PyObject* o, int64_t dim, at::ScalarType type, c10::Device device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.dim() != dim || t.layout() != at::kStrided || !t.is_cuda() || !t.has_storage() ||
      t.is_conj() || t.is_neg() || t.scalar_type() != type || t.device() != device || at::isTensorSubclassLike(t))
    return nullptr;
  for (int64_t i = 0; i < dim; ++i)
    if (t.size(i) > INT32_MAX) return nullptr;
  return &t;
}
// ... that is also dense
const at::Tensor* dense_of(PyObject* o, int64_t dim, at::ScalarType type, c10::Device device) {
  const at::Tensor* t = tensor_of(o, dim, type, device);
  return t && t->is_contiguous() ? t : nullptr;
}
// The type and device of a call's rows: fp16 or bf16, on the current device; false otherwise
bool rows_type(PyObject* o, at::ScalarType* type, c10::Device* device) {
  if (!THPVariable_CheckExact(o) || c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled())
    return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda()) return false;
  *type = t.scalar_type();
  *device = t.device();
  return (*type == at::kHalf || *type == at::kBFloat16) && device->index() == c10::hip::current_device();
}
int32_t code_of(at::ScalarType type) { return type == at::kBFloat16 ? FA2_DTYPE_BF16 : FA2_DTYPE_F16; }

// The strides of all but the last dimension (0 for a dimension of one element), if the last has stride 1 and
// the kernels' loads can address the rest; `multiple` elements to 16 bytes
bool row_strides(const at::Tensor& t, int64_t multiple, int64_t* s) {
  const int64_t n = t.dim() - 1;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || t.stride(n) != 1) return false;
  for (int64_t i = 0; i < n; ++i) {
    s[i] = t.size(i) == 1 ? 0 : t.stride(i);
    if (s[i] < 0 || s[i] % multiple) return false;
  }
  return true;
}

// k, v, k_scale, v_scale at args[0 .. 3] and table, cu, lens at args[4 .. 6]
bool cache_and_sequences(PyObject* const* args, at::ScalarType rows, c10::Device device, int64_t n_tokens,
                         fa2_cache* c, fa2_sequences* q) {
  const bool e4m3 = THPVariable_CheckExact(args[0]) &&
                    THPVariable_Unpack(args[0]).scalar_type() == at::kFloat8_e4m3fn;
  const at::ScalarType type = e4m3 ? at::kFloat8_e4m3fn : rows;
  const at::Tensor *k = tensor_of(args[0], 4, type, device), *v = tensor_of(args[1], 4, type, device);
  if (!k || !v || k->sizes() != v->sizes()) return false;
  *c = fa2_cache{};
  c->k = k->data_ptr();
  c->v = v->data_ptr();
  if (!row_strides(*k, e4m3 ? 16 : 8, c->k_stride) || !row_strides(*v, e4m3 ? 16 : 8, c->v_stride)) return false;
  if (e4m3) {
    const at::Tensor *ks = tensor_of(args[2], 3, at::kFloat8_e8m0fnu, device);
    const at::Tensor *vs = tensor_of(args[3], 3, at::kFloat8_e8m0fnu, device);
    if (!ks || !vs || ks->sizes() != k->sizes().slice(0, 3) || vs->sizes() != ks->sizes()) return false;
    c->k_scale = ks->data_ptr();
    c->v_scale = vs->data_ptr();
    for (int i = 0; i < 3; ++i) {
      c->k_scale_stride[i] = ks->size(i) == 1 ? 0 : ks->stride(i);
      c->v_scale_stride[i] = vs->size(i) == 1 ? 0 : vs->stride(i);
    }
  }
  c->n_pages = (int32_t)k->size(0);
  c->h_kv = (int32_t)k->size(1);
  c->page_size = (int32_t)k->size(2);
  c->head_dim = (int32_t)k->size(3);
  c->cache_dtype = e4m3 ? FA2_DTYPE_E4M3 : code_of(rows);
  const at::Tensor *table = tensor_of(args[4], 2, at::kInt, device), *cu = dense_of(args[5], 1, at::kInt, device);
  const at::Tensor* lens = dense_of(args[6], 1, at::kInt, device);
  if (!table || !cu || !lens || cu->size(0) != lens->size(0) + 1 || table->size(0) != lens->size(0) ||
      (table->size(1) > 1 && table->stride(1) != 1) || n_tokens > INT32_MAX)
    return false;
  *q = fa2_sequences{(const int32_t*)cu->data_ptr(), (const int32_t*)lens->data_ptr(), (const int32_t*)table->data_ptr(),
                     table->size(0) == 1 ? 0 : table->stride(0), (int32_t)lens->size(0), (int32_t)n_tokens,
                     (int32_t)table->size(1)};
  return true;
}

// freqs (or None), interleaved, scale
bool rotation_of(PyObject* freqs, PyObject* interleaved, PyObject* scale, c10::Device device, fa2_rotation* r) {
  const at::Tensor* f = dense_of(freqs, 1, at::kDouble, device);
  if (!f || !PyFloat_CheckExact(scale) || !PyBool_Check(interleaved)) return false;
  *r = fa2_rotation{(const double*)f->data_ptr(), (int32_t)f->size(0), interleaved == Py_True, PyFloat_AS_DOUBLE(scale)};
  return true;
}

// sm_scale * log2 e of a call (None: 1 / sqrt(head_dim)); 0 if it is not a plain positive float
float qk_scale_of(PyObject* o, int64_t head_dim) {
  double s = 1.0 / std::sqrt((double)head_dim);
  if (o != Py_None) {
    if (!PyFloat_CheckExact(o)) return 0.f;
    s = PyFloat_AS_DOUBLE(o);
  }
  return s > 0 ? (float)(s * kLog2e) : 0.f;
}

// The caller's out (or a new tensor like q), if the kernels can address it
bool out_of(PyObject* o, const at::Tensor& q, at::Tensor* out, int64_t* s) {
  if (o == Py_None) {
    *out = at::empty_like(q);
  } else {
    const at::Tensor* t = tensor_of(o, q.dim(), q.scalar_type(), q.device());
    if (!t || t->sizes() != q.sizes()) return false;
    *out = *t;
  }
  return row_strides(*out, 8, s);
}

PyObject* pair_of(at::Tensor a, at::Tensor b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = x ? THPVariable_Wrap(std::move(b)) : nullptr;
  PyObject* both = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

bool arguments(const char* what, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", what, want, n);
  return false;
}

// rotary(x, positions, freqs, interleaved, scale, out)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("rotary", n_args, 6)) return nullptr;
  at::ScalarType type;
  c10::Device device(c10::kCPU);
  if (!rows_type(args[0], &type, &device)) Py_RETURN_NONE;
  const bool packed = THPVariable_Unpack(args[0]).dim() == 3;
  const at::Tensor* x = tensor_of(args[0], packed ? 3 : 4, type, device);
  if (!x || x->numel() == 0 || !THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
  const at::ScalarType ptype = THPVariable_Unpack(args[1]).scalar_type();
  if (ptype != at::kInt && ptype != at::kLong) Py_RETURN_NONE;
  const bool each = !packed && THPVariable_Unpack(args[1]).dim() == 2;  // positions of every batch row
  const at::Tensor* pos = tensor_of(args[1], each ? 2 : 1, ptype, device);
  const int64_t B = packed ? 1 : x->size(0), H = x->size(1), N = packed ? x->size(0) : x->size(2);
  if (!pos || pos->size(each) != N || (each && pos->size(0) != B)) Py_RETURN_NONE;
  fa2_rotation rot;
  at::Tensor out;
  int64_t xs[3], os[3], xt[3], ot[3];
  if (!rotation_of(args[2], args[3], args[4], device, &rot) || !row_strides(*x, 8, xt) || !out_of(args[5], *x, &out, ot))
    Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i) {  // [b, h, n] of a packed [n, h]
    xs[i] = !packed ? xt[i] : i == 0 ? 0 : i == 1 ? xt[1] : xt[0];
    os[i] = !packed ? ot[i] : i == 0 ? 0 : i == 1 ? ot[1] : ot[0];
  }
  const int64_t ps[2] = {each ? pos->stride(0) : 0, pos->stride(each)};
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void* xp = x->data_ptr();
  const void* pp = pos->data_ptr();
  void* op = out.data_ptr();
  const int64_t D = x->size(packed ? 2 : 3);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fa2_rotary(xp, op, xs, os, pp, ptype == at::kLong ? 8 : 4, ps, &rot, (int32_t)B, (int32_t)H, (int32_t)N,
                  (int32_t)D, code_of(type), stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A HeadNorm's weight and eps at args[0] and args[1] (None: no norm)
bool norm_of(PyObject* const* args, int64_t head_dim, c10::Device device, const float** weight, double* eps) {
  *weight = nullptr;
  *eps = 0.0;
  if (args[0] == Py_None) return true;
  const at::Tensor* w = dense_of(args[0], 1, at::kFloat, device);
  if (!w || w->size(0) != head_dim || !PyFloat_CheckExact(args[1])) return false;
  *weight = (const float*)w->data_ptr();
  *eps = PyFloat_AS_DOUBLE(args[1]);
  return true;
}

// A plan's axes (None: one) and the positions of n tokens (of `batch` of them each), as the kernels take them
bool axes_of(PyObject* axes, PyObject* positions, int64_t batch, int64_t n, c10::Device device, fa2_turn* t, const void** p,
             int32_t* bytes, int64_t (&stride)[3]) {
  t->axes = nullptr;
  t->n_axes = 1;
  const bool several = axes != Py_None;
  if (several) {
    const at::Tensor* a = dense_of(axes, 1, at::kInt, device);
    if (!a || a->size(0) != t->rotation.half) return false;
    t->axes = (const int32_t*)a->data_ptr();
  }
  if (!THPVariable_CheckExact(positions)) return false;
  const at::Tensor& x = THPVariable_Unpack(positions);
  const at::ScalarType type = x.defined() ? x.scalar_type() : at::kFloat;
  if (type != at::kInt && type != at::kLong) return false;
  const int64_t dim = x.dim() - several;  // of one axis
  if (dim != 1 && (dim != 2 || batch == 0)) return false;
  const at::Tensor* at = tensor_of(positions, x.dim(), type, device);
  if (!at || at->size(x.dim() - 1) != n || (dim == 2 && at->size(several) != batch) || (several && at->size(0) < 1)) return false;
  if (several) t->n_axes = (int32_t)at->size(0);
  stride[0] = several ? at->stride(0) : 0;
  stride[1] = dim == 2 ? at->stride(several) : 0;
  stride[2] = at->stride(x.dim() - 1);
  *p = at->data_ptr();
  *bytes = type == at::kLong ? 8 : 4;
  return true;
}

// rotary_qk(q, k, positions, freqs, interleaved, scale, axes, q_weight, q_eps, k_weight, k_eps, q_out, k_out) ->
// (q_out, k_out); k may be None, and so is its result then
PyObject* rotary_qk(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("rotary_qk", n_args, 13)) return nullptr;
  at::ScalarType type;
  c10::Device device(c10::kCPU);
  if (!rows_type(args[0], &type, &device)) Py_RETURN_NONE;
  const bool packed = THPVariable_Unpack(args[0]).dim() == 3, has_k = args[1] != Py_None;
  const at::Tensor* q = tensor_of(args[0], packed ? 3 : 4, type, device);
  const at::Tensor* k = has_k ? tensor_of(args[1], packed ? 3 : 4, type, device) : nullptr;
  if (!q || q->numel() == 0 || (has_k && (!k || k->numel() == 0)) || (!has_k && (args[9] != Py_None || args[12] != Py_None)))
    Py_RETURN_NONE;
  const int64_t B = packed ? 1 : q->size(0), N = packed ? q->size(0) : q->size(2), D = q->size(packed ? 2 : 3);
  if (has_k && ((packed ? k->size(0) : k->size(2)) != N || (!packed && k->size(0) != B) || k->size(packed ? 2 : 3) != D))
    Py_RETURN_NONE;
  fa2_turn turn;
  const void* pp;
  int32_t bytes;
  int64_t ps[3], t[4][3], s[4][3] = {};
  at::Tensor q_out, k_out;
  if (!rotation_of(args[3], args[4], args[5], device, &turn.rotation) ||
      !axes_of(args[6], args[2], packed ? 0 : B, N, device, &turn, &pp, &bytes, ps) ||
      !norm_of(args + 7, D, device, &turn.q_weight, &turn.q_eps) || !norm_of(args + 9, D, device, &turn.k_weight, &turn.k_eps) ||
      !row_strides(*q, 8, t[0]) || !out_of(args[11], *q, &q_out, t[2]) ||
      (has_k && (!row_strides(*k, 8, t[1]) || !out_of(args[12], *k, &k_out, t[3]))))
    Py_RETURN_NONE;
  for (int x = 0; x < 4; ++x)
    for (int i = 0; i < 3 && (has_k || x % 2 == 0); ++i)  // [b, h, n] of a packed [n, h]
      s[x][i] = !packed ? t[x][i] : i == 0 ? 0 : i == 1 ? t[x][1] : t[x][0];
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void *qp = q->data_ptr(), *kp = has_k ? k->data_ptr() : nullptr;
  void *qo = q_out.data_ptr(), *ko = has_k ? k_out.data_ptr() : nullptr;
  const int32_t hq = (int32_t)q->size(1), hk = has_k ? (int32_t)k->size(1) : 0;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fa2_rotary_qk(qp, kp, qo, ko, s[0], s[1], s[2], s[3], pp, bytes, ps, &turn, (int32_t)B, hq, hk, (int32_t)N, (int32_t)D,
                     code_of(type), stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  if (has_k) return pair_of(std::move(q_out), std::move(k_out));
  PyObject* o = THPVariable_Wrap(std::move(q_out));
  PyObject* both = o ? PyTuple_Pack(2, o, Py_None) : nullptr;
  Py_XDECREF(o);
  return both;
  END_HANDLE_TH_ERRORS
}

// cache_write(k_cache, v_cache, k_scale, v_scale, table, cu, lens, k, v, freqs, interleaved, scale, axes, q, q_out) -> q_out, or
// True without q; cache_write_turned with q_weight, q_eps, k_weight, k_eps and positions (or None) behind them
PyObject* write_any(PyObject* const* args, bool turned) {
  at::ScalarType type;
  c10::Device device(c10::kCPU);
  if (!rows_type(args[7], &type, &device)) Py_RETURN_NONE;
  const at::Tensor *k = tensor_of(args[7], 3, type, device), *v = tensor_of(args[8], 3, type, device);
  fa2_cache c;
  fa2_sequences s;
  if (!k || !v || k->sizes() != v->sizes() || k->numel() == 0 ||
      !cache_and_sequences(args, type, device, k->size(0), &c, &s) || k->size(1) != c.h_kv || k->size(2) != c.head_dim)
    Py_RETURN_NONE;
  int64_t ks[2], vs[2], qs[2], os[2], ps[3] = {};
  fa2_turn turn;
  const void* pp = nullptr;
  int32_t bytes = 0;
  const bool turn_k = args[9] != Py_None, has_q = args[13] != Py_None;
  const at::Tensor* q = nullptr;
  at::Tensor out;
  if (!row_strides(*k, 8, ks) || !row_strides(*v, 8, vs) ||
      (turn_k && !rotation_of(args[9], args[10], args[11], device, &turn.rotation)) || (has_q && !turn_k) ||
      (!has_q && args[14] != Py_None))
    Py_RETURN_NONE;
  if (turned) {
    turn.axes = nullptr;
    turn.n_axes = 1;
    if (!turn_k || (!has_q && args[15] != Py_None) || !norm_of(args + 15, c.head_dim, device, &turn.q_weight, &turn.q_eps) ||
        !norm_of(args + 17, c.head_dim, device, &turn.k_weight, &turn.k_eps) ||
        (args[19] != Py_None ? !axes_of(args[12], args[19], 0, k->size(0), device, &turn, &pp, &bytes, ps)
                             : args[12] != Py_None))
      Py_RETURN_NONE;
  }
  if (has_q) {
    q = tensor_of(args[13], 3, type, device);
    if (!q || q->size(0) != k->size(0) || q->size(2) != k->size(2) || q->size(1) < 1 || !row_strides(*q, 8, qs) ||
        !out_of(args[14], *q, &out, os))
      Py_RETURN_NONE;
  }
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void *kp = k->data_ptr(), *vp = v->data_ptr(), *qp = has_q ? q->data_ptr() : nullptr;
  void* op = has_q ? out.data_ptr() : nullptr;
  const int32_t hq = has_q ? (int32_t)q->size(1) : 0;
  const int64_t p2[2] = {ps[0], ps[2]};
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (turned)
    rc = fa2_cache_write_turned(&c, &s, kp, vp, ks, vs, qp, op, qs, os, hq, pp, bytes, p2, &turn, code_of(type), stream);
  else
    rc = fa2_cache_write(&c, &s, kp, vp, ks, vs, qp, op, qs, os, hq, turn_k ? &turn.rotation : nullptr, code_of(type), stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  if (!has_q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
}
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  return arguments("cache_write", n_args, 15) ? write_any(args, false) : nullptr;
  END_HANDLE_TH_ERRORS
}
PyObject* cache_write_turned(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  return arguments("cache_write_turned", n_args, 20) ? write_any(args, true) : nullptr;
  END_HANDLE_TH_ERRORS
}

// A pool's free and count at args[0] and args[1], the table at args[2], two int32 [S] at args[3] and args[4]: plain, dense
// (the table in its rows) and on the current device
struct Pages {
  const at::Tensor *free, *count, *table, *a, *b;
  int64_t table_stride;
};
bool pages_of(PyObject* const* args, Pages* p) {
  if (!THPVariable_CheckExact(args[0]) || c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled()) return false;
  const at::Tensor& f = THPVariable_Unpack(args[0]);
  if (!f.defined() || !f.is_cuda() || f.device().index() != c10::hip::current_device()) return false;
  p->free = dense_of(args[0], 1, at::kInt, f.device());
  p->count = dense_of(args[1], 1, at::kInt, f.device());
  p->table = tensor_of(args[2], 2, at::kInt, f.device());
  p->a = dense_of(args[3], 1, at::kInt, f.device());
  p->b = dense_of(args[4], 1, at::kInt, f.device());
  if (!p->free || !p->count || !p->table || !p->a || !p->b || p->count->numel() != 1) return false;
  const int64_t S = p->table->size(0), P = p->table->size(1);
  p->table_stride = S == 1 ? 0 : p->table->stride(0);
  return S > 0 && p->a->size(0) == S && p->b->size(0) == S && (P <= 1 || p->table->stride(1) == 1) &&
         (S == 1 || P == 0 || p->table_stride >= P);
}

// pages_extend(free, count, table, lens, new, page_size, n_tokens) -> (count, cu, lens, positions, slots)
PyObject* pages_extend(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("pages_extend", n_args, 7)) return nullptr;
  Pages p;
  if (!pages_of(args, &p) || !PyLong_CheckExact(args[5]) || !PyLong_CheckExact(args[6])) Py_RETURN_NONE;
  int overflow = 0, overflow2 = 0;
  const long long page = PyLong_AsLongLongAndOverflow(args[5], &overflow), n = PyLong_AsLongLongAndOverflow(args[6], &overflow2);
  if (overflow || overflow2 || page < 1 || page > INT32_MAX || n < 0 || n > INT32_MAX) Py_RETURN_NONE;
  const int64_t S = p.table->size(0);
  const auto options = p.free->options();
  at::Tensor out[5] = {at::empty({1}, options), at::empty({S + 1}, options), at::empty({S}, options), at::empty({n}, options),
                       at::empty({n}, options.dtype(at::kLong))};
  void* stream = c10::hip::getCurrentHIPStream(p.free->device().index()).stream();
  int32_t* to[4];
  for (int i = 0; i < 4; ++i) to[i] = (int32_t*)out[i].data_ptr();
  int64_t* slots = (int64_t*)out[4].data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fa2_pages_extend((const int32_t*)p.free->data_ptr(), (int32_t)p.free->size(0), (const int32_t*)p.count->data_ptr(), to[0],
                        (int32_t*)p.table->data_ptr(), p.table_stride, (int32_t)S, (int32_t)p.table->size(1), (int32_t)page,
                        (const int32_t*)p.a->data_ptr(), (const int32_t*)p.b->data_ptr(), to[2], to[1], to[3], slots, (int32_t)n,
                        stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  PyObject* all = PyTuple_New(5);
  for (int i = 0; all && i < 5; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(out[i]));
    if (o)
      PyTuple_SET_ITEM(all, i, o);
    else
      Py_CLEAR(all);
  }
  return all;
  END_HANDLE_TH_ERRORS
}

// pages_release(free, count, table, first, last) -> count
PyObject* pages_release(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("pages_release", n_args, 5)) return nullptr;
  Pages p;
  if (!pages_of(args, &p)) Py_RETURN_NONE;
  const int64_t S = p.table->size(0);
  at::Tensor count = at::empty({1}, p.free->options()), counts = at::empty({S + 1}, p.free->options());
  void* stream = c10::hip::getCurrentHIPStream(p.free->device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fa2_pages_release((int32_t*)p.free->data_ptr(), (int32_t)p.free->size(0), (const int32_t*)p.count->data_ptr(),
                         (int32_t*)count.data_ptr(), (const int32_t*)p.table->data_ptr(), p.table_stride, (int32_t)S,
                         (int32_t)p.table->size(1), (const int32_t*)p.a->data_ptr(), (const int32_t*)p.b->data_ptr(),
                         (int32_t*)counts.data_ptr(), stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(count));
  END_HANDLE_TH_ERRORS
}

// cache_read(k_cache, v_cache, k_scale, v_scale, table, cu, lens, n_tokens, dtype) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("cache_read", n_args, 9)) return nullptr;
  if (!THPVariable_CheckExact(args[0]) || !PyLong_CheckExact(args[7]) || c10::impl::dispatch_mode_enabled() ||
      at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const at::Tensor& kc = THPVariable_Unpack(args[0]);
  int overflow = 0;
  const long long n = PyLong_AsLongLongAndOverflow(args[7], &overflow);
  if (overflow || n < 1 || n > INT32_MAX || !kc.defined() || !kc.is_cuda() ||
      kc.device().index() != c10::hip::current_device() || !THPDtype_Check(args[8]))
    Py_RETURN_NONE;
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[8])->scalar_type;
  fa2_cache c;
  fa2_sequences s;
  if ((type != at::kHalf && type != at::kBFloat16) || !cache_and_sequences(args, type, kc.device(), n, &c, &s))
    Py_RETURN_NONE;
  const auto options = kc.options().dtype(type);
  at::Tensor k = at::empty({n, c.h_kv, c.head_dim}, options), v = at::empty({n, c.h_kv, c.head_dim}, options);
  int64_t st[2];
  if (!row_strides(k, 8, st)) Py_RETURN_NONE;
  void* stream = c10::hip::getCurrentHIPStream(kc.device().index()).stream();
  void *kp = k.data_ptr(), *vp = v.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fa2_cache_read(&c, &s, kp, vp, st, st, code_of(type), stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  return pair_of(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// window (None: all keys) and sinks at args[0] and args[1], as the C ABI takes them: *window 0 without one
bool window_of(PyObject* const* args, int causal, int32_t* window, int32_t* sinks) {
  if (!PyLong_CheckExact(args[1])) return false;
  int overflow = 0;
  const long long s = PyLong_AsLongLongAndOverflow(args[1], &overflow);
  if (overflow || s < 0) return false;
  *window = *sinks = 0;
  if (args[0] == Py_None) return s == 0;
  if (!PyLong_CheckExact(args[0]) || !causal) return false;
  const long long w = PyLong_AsLongLongAndOverflow(args[0], &overflow);
  if (overflow || w < 1) return false;
  *window = (int32_t)(w < INT32_MAX ? w : INT32_MAX);
  *sinks = (int32_t)(s < INT32_MAX ? s : INT32_MAX);
  return true;
}

// attn_packed(q, k, v, cu, cu_kv, causal, sm_scale, return_lse, out, window, sinks)
PyObject* attn_packed(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("attn_packed", n_args, 11)) return nullptr;
  at::ScalarType type;
  c10::Device device(c10::kCPU);
  if (!rows_type(args[0], &type, &device)) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(args[0], 3, type, device), *k = tensor_of(args[1], 3, type, device);
  const at::Tensor *v = tensor_of(args[2], 3, type, device), *cu = dense_of(args[3], 1, at::kInt, device);
  const at::Tensor* cu_kv = args[4] == Py_None ? nullptr : dense_of(args[4], 1, at::kInt, device);
  const int causal = PyObject_IsTrue(args[5]), want_lse = PyObject_IsTrue(args[7]);
  if (causal < 0 || want_lse < 0) return nullptr;
  if (!q || !k || !v || !cu || (args[4] != Py_None && !cu_kv) || q->numel() == 0 || k->sizes() != v->sizes() ||
      k->size(2) != q->size(2) || k->size(1) < 1 || q->size(1) % k->size(1) || cu->size(0) < 1 ||
      (cu_kv ? cu_kv->size(0) != cu->size(0) : k->size(0) != q->size(0)))
    Py_RETURN_NONE;
  const float scale = qk_scale_of(args[6], q->size(2));
  int64_t qs[2], ks[2], vs[2], os[2];
  int32_t window, sinks;
  at::Tensor out, lse;
  if (scale == 0.f || !window_of(args + 9, causal, &window, &sinks) || !row_strides(*q, 8, qs) || !row_strides(*k, 8, ks) || !row_strides(*v, 8, vs) ||
      !out_of(args[8], *q, &out, os))
    Py_RETURN_NONE;
  const int32_t T = (int32_t)q->size(0), hq = (int32_t)q->size(1), hkv = (int32_t)k->size(1);
  if (want_lse) lse = at::empty({hq, T}, q->options().dtype(at::kFloat));
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
  void* op = out.data_ptr();
  float* lp = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  const int32_t *cp = (const int32_t*)cu->data_ptr(), *ckp = cu_kv ? (const int32_t*)cu_kv->data_ptr() : nullptr;
  const int32_t n_seq = (int32_t)cu->size(0) - 1, T_kv = (int32_t)k->size(0), D = (int32_t)q->size(2);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (window)
    rc = fa2_attn_packed_window(qp, kp, vp, op, qs, ks, vs, os, cp, ckp, n_seq, T, T_kv, hq, hkv, D, code_of(type), window,
                                sinks, scale, lp, stream);
  else
    rc = fa2_attn_packed(qp, kp, vp, op, qs, ks, vs, os, cp, ckp, n_seq, T, T_kv, hq, hkv, D, code_of(type), causal, scale,
                         lp, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  return want_lse ? pair_of(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// attn_paged(k_cache, v_cache, k_scale, v_scale, table, cu, lens, q, causal, sm_scale, return_lse, out, window, sinks,
// shared)
PyObject* attn_paged(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!arguments("attn_paged", n_args, 15)) return nullptr;
  at::ScalarType type;
  c10::Device device(c10::kCPU);
  if (!rows_type(args[7], &type, &device)) Py_RETURN_NONE;
  const at::Tensor* q = tensor_of(args[7], 3, type, device);
  const int causal = PyObject_IsTrue(args[8]), want_lse = PyObject_IsTrue(args[10]);
  if (causal < 0 || want_lse < 0) return nullptr;
  fa2_cache c;
  fa2_sequences s;
  if (!q || q->numel() == 0 || !cache_and_sequences(args, type, device, q->size(0), &c, &s) || q->size(2) != c.head_dim ||
      c.h_kv < 1 || q->size(1) % c.h_kv)
    Py_RETURN_NONE;
  const float scale = qk_scale_of(args[9], q->size(2));
  const int cus = cu_count(device.index());
  int64_t qs[2], os[2];
  int32_t window, sinks;
  at::Tensor out, lse, ws;
  const at::Tensor* shared = args[14] == Py_None ? nullptr : dense_of(args[14], 1, at::kInt, device);
  if (!window_of(args + 12, causal, &window, &sinks) || (args[14] != Py_None && (!shared || shared->numel() != 1 || window)))
    Py_RETURN_NONE;
  if (scale == 0.f || cus < 1 || !row_strides(*q, 8, qs) || !out_of(args[11], *q, &out, os)) Py_RETURN_NONE;
  const int32_t T = (int32_t)q->size(0), hq = (int32_t)q->size(1);
  if (want_lse) lse = at::empty({hq, T}, q->options().dtype(at::kFloat));
  const int64_t keys = (int64_t)s.max_pages * c.page_size;
  const size_t n_ws =
      shared   ? fa2_paged_shared_workspace_bytes(hq, c.h_kv, c.head_dim, T, s.n_seq, cus)
      : window ? fa2_paged_window_workspace_bytes(hq, c.h_kv, c.head_dim, c.cache_dtype, T, s.n_seq, keys, window, sinks, cus)
               : fa2_paged_workspace_bytes(hq, c.h_kv, c.head_dim, c.cache_dtype, T, s.n_seq, keys, cus);
  if (n_ws) ws = at::empty({(int64_t)n_ws}, q->options().dtype(at::kByte));
  void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
  const void* qp = q->data_ptr();
  void* op = out.data_ptr();
  float* lp = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  void* wp = n_ws ? ws.data_ptr() : nullptr;
  const int32_t* sp = shared ? (const int32_t*)shared->data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (shared)
    rc = fa2_attn_paged_shared(qp, op, qs, os, &c, &s, sp, hq, code_of(type), causal, scale, lp, wp, n_ws, stream);
  else if (window)
    rc = fa2_attn_paged_window(qp, op, qs, os, &c, &s, hq, code_of(type), window, sinks, scale, lp, wp, n_ws, stream);
  else
    rc = fa2_attn_paged(qp, op, qs, os, &c, &s, hq, code_of(type), causal, scale, lp, wp, n_ws, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA2_OK) Py_RETURN_NONE;
  return want_lse ? pair_of(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define FA2_FAST(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, "its Python function's call, or None"}
PyMethodDef methods[] = {
    FA2_FAST(rotary), FA2_FAST(cache_write), FA2_FAST(cache_read), FA2_FAST(attn_packed), FA2_FAST(attn_paged),
    FA2_FAST(rotary_qk), FA2_FAST(cache_write_turned), FA2_FAST(pages_extend), FA2_FAST(pages_release),
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     "call(q, k, v, causal, sm_scale, return_lse) -> attention()'s result, or None"},
    {"policy", policy, METH_VARARGS,
     "policy(batch, h_q, h_kv, n_q, n_kv, head_dim, dtype, causal, cus) -> (pack, splits, workspace bytes)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_call", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: fa2/_lib.py's build_id() of the torch and Python compiled against (csrc/build.py); another
// one does not use this module.
PyMODINIT_FUNC PyInit__torch_call() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", FA2_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
