// The host side of the hot entry points in native code: argument checks, strides, the launch.
//
// An eager decode step at batch 1 spends its time on the host: ops.attn_decode_append took 27 us
// of Python (25 stride reads, 45 ctypes conversions, stream and workspace look-ups) around two
// kernels of 15 us. Each function here takes exactly the calls whose arguments need no conversion
// (tensors of the package's layouts and types on one device, outside graph capture) and returns
// None for every other one, which then goes the Python way, with its conversions and its errors;
// an int is the status of a launch that was rejected or failed. Nothing is kept between calls.
#include <Python.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include "../../include/forge_attn.h"

namespace {

using at::Tensor;

// A tensor as plain memory on a GPU: no subclass, functorch wrapper, fake tensor or forward-mode dual.
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
         t.has_storage() && !t.is_conj() && !t.is_neg() && !t._fw_grad(0).defined() &&
         !t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched,
                                                   c10::DispatchKey::FuncTorchGradWrapper,
                                                   c10::DispatchKey::Functionalize, c10::DispatchKey::Python}));
}

// The tensor behind a Python argument (a Parameter counts as one); false for anything that is no
// plain GPU tensor.
bool take(PyObject* o, Tensor& t) {
  if (!THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return plain(t);
}

// The same where None is allowed (t stays undefined).
bool take_opt(PyObject* o, Tensor& t) { return o == Py_None || take(o, t); }

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FORGE_F32;
    case at::kBFloat16: return FORGE_BF16;
    case at::kHalf: return FORGE_F16;
    default: return -1;
  }
}

// fp32 norm gain of D values
bool gain_ok(const Tensor& w, int64_t D, c10::Device dev) {
  return !w.defined() ||
         (w.scalar_type() == at::kFloat && w.is_contiguous() && w.numel() == D && w.device() == dev);
}

struct Rope {
  const float* cos = nullptr;
  const float* sin = nullptr;
  int64_t sb = 0, st = 0;
};

// fp32 tables [T, D] or [1 or B, T, D] with equal strides
bool rope_ok(const Tensor& c, const Tensor& s, int64_t B, int64_t T, int64_t D, c10::Device dev, Rope& r) {
  if (!c.defined() && !s.defined()) return true;
  if (!c.defined() || !s.defined()) return false;
  const int64_t d = c.dim();
  if ((d != 2 && d != 3) || c.sizes() != s.sizes() || c.strides() != s.strides() || c.size(d - 1) != D ||
      c.size(d - 2) != T || c.stride(d - 1) != 1 || c.scalar_type() != at::kFloat || s.scalar_type() != at::kFloat ||
      c.device() != dev || s.device() != dev)
    return false;
  if (d == 3 && c.size(0) != 1 && c.size(0) != B) return false;
  r.cos = static_cast<const float*>(ptr(c));
  r.sin = static_cast<const float*>(ptr(s));
  r.sb = d == 3 && c.size(0) == B && B > 1 ? c.stride(0) : 0;
  r.st = c.stride(d - 2);
  return true;
}

bool as_int(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool as_float(PyObject* o, float& v) {
  if (!PyFloat_CheckExact(o)) return false;
  v = (float)PyFloat_AS_DOUBLE(o);
  return true;
}

bool capturing() {
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

// Gives the GIL up for its scope (no Python object is touched there): an allocation may have to free
// and synchronise, and a launch waits while the stream's queue is full.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// The buffer of (device, stream) from the caller's workspace table (ops._STREAM_WS: cleared buffers,
// the most recently used last), taken out of the table while a call uses it, so that no other thread
// launches on it in between, and put back once the call is launched.
struct StreamWorkspace {
  PyObject *table, *key = nullptr, *buf = nullptr;
  void* ptr = nullptr;
  size_t bytes = 0;

  StreamWorkspace(PyObject* table, int dev, hipStream_t stream, size_t need) : table(table) {
    if (!need) return;
    key = Py_BuildValue("(iK)", dev, (unsigned long long)(uintptr_t)stream);
    PyObject* b = key ? PyDict_GetItemWithError(table, key) : nullptr;
    if (b && THPVariable_CheckExact(b) && (size_t)THPVariable_Unpack(b).numel() >= need) {
      Py_INCREF(b);
      if (PyDict_DelItem(table, key) == 0) buf = b;
      else Py_DECREF(b);
    }
    if (PyErr_Occurred()) PyErr_Clear();
    if (!buf) return;
    ptr = THPVariable_Unpack(buf).data_ptr();
    bytes = (size_t)THPVariable_Unpack(buf).numel();
  }
  void put_back() {
    if (buf && PyDict_SetItem(table, key, buf) != 0) PyErr_Clear();
  }
  ~StreamWorkspace() {
    Py_XDECREF(buf);
    Py_XDECREF(key);
  }
};

PyObject* result(int st, const Tensor& out) {
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(out);
}

// decode_append(table, q, k, v, k_cache, v_cache, scale, pos | None, pos_dev | None, row_pos | None,
//               max_kv_len | None, window, q_weight | None, k_weight | None, eps, norm_q, norm_k, norm_v,
//               cos | None, sin | None, chunk)
PyObject* decode_append_impl(PyObject* const* a) {
  Tensor q, k, v, kc, vc, pos_dev, row_pos, qw, kw, cos, sin;
  if (!take(a[1], q) || !take(a[2], k) || !take(a[3], v) || !take(a[4], kc) || !take(a[5], vc) ||
      !take_opt(a[8], pos_dev) || !take_opt(a[9], row_pos) || !take_opt(a[12], qw) || !take_opt(a[13], kw) ||
      !take_opt(a[18], cos) || !take_opt(a[19], sin))
    return nullptr;
  float scale, eps;
  int64_t window, chunk, pos = 0, max_kv = -1;
  if (!as_float(a[6], scale) || !as_float(a[14], eps) || !as_int(a[11], window) || !as_int(a[20], chunk) ||
      (a[7] != Py_None && !as_int(a[7], pos)) || (a[10] != Py_None && !as_int(a[10], max_kv)))
    return nullptr;
  const bool norm_q = a[15] == Py_True, norm_k = a[16] == Py_True, norm_v = a[17] == Py_True;
  if (q.dim() != 4 || k.dim() != 4 || kc.dim() != 4 || k.sizes() != v.sizes() || kc.sizes() != vc.sizes() ||
      kc.strides() != vc.strides())
    return nullptr;
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), K = kc.size(1), max_len = kc.size(2);
  const int dt = dtype_of(q);
  const c10::Device dev = q.device();
  if (dt < 0 || K <= 0 || H % K || kc.size(0) != B || kc.size(3) != D || k.size(0) != B || k.size(1) != K ||
      k.size(2) != T || k.size(3) != D)
    return nullptr;
  for (const Tensor* t : {&k, &v, &kc, &vc})
    if (t->scalar_type() != q.scalar_type() || t->device() != dev || t->stride(3) != 1) return nullptr;
  if (q.stride(3) != 1) return nullptr;
  if (row_pos.defined()) {
    if (row_pos.scalar_type() != at::kInt || row_pos.numel() != B || row_pos.device() != dev || !row_pos.is_contiguous())
      return nullptr;
    pos_dev.reset();
    pos = 0;
  } else if (pos_dev.defined()) {
    if (pos_dev.scalar_type() != at::kLong || pos_dev.device() != dev) return nullptr;
    pos = 0;
  }
  Rope r;
  if (!rope_ok(cos, sin, B, T, D, dev, r) || !gain_ok(qw, D, dev) || !gain_ok(kw, D, dev)) return nullptr;
  if (pos < 0 || pos > max_len) return nullptr;
  if (max_kv < 0) max_kv = !row_pos.defined() && !pos_dev.defined() ? pos + T : max_len;
  max_kv = std::max<int64_t>(1, std::min(max_kv, max_len));
  if (window < 0 || window > INT_MAX || chunk > INT_MAX || c10::hip::current_device() != dev.index()) return nullptr;
  if (chunk <= 0) {
    const int64_t span = window > 0 && window + 16 < max_len ? window + 16 : max_len;  // ops.decode_chunk
    chunk = (row_pos.defined() ? forge_attn_decode_chunk : forge_attn_decode_chunk_uniform)(dt, (int)B, (int)T, (int)H,
                                                                                          (int)K, (int)D, span);
  }
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  const size_t need = forge_attn_decode_workspace_bytes(dt, (int)B, (int)T, (int)H, (int)K, (int)D, max_kv, (int)chunk);
  if (need && capturing()) return nullptr;
  StreamWorkspace ws(a[0], dev.index(), stream, need);
  if (need && !ws.ptr) return nullptr;
  const int rope = r.cos ? FORGE_ROPE : 0;
  Tensor out;
  int st;
  {
    NoGil unlocked;
    out = at::empty({B, T, H, D}, q.options().requires_grad(false));
    st = forge_attn_decode_append(
        dt, (int)B, (int)T, (int)H, (int)K, (int)D, ptr(q), q.stride(0), q.stride(1), q.stride(2),
        norm_q ? static_cast<const float*>(ptr(qw)) : nullptr, eps, (norm_q ? FORGE_NORM_QK : 0) | rope, ptr(k),
        k.stride(0), k.stride(1), k.stride(2), ptr(v), v.stride(0), v.stride(1), v.stride(2),
        norm_k ? static_cast<const float*>(ptr(kw)) : nullptr,
        (norm_k ? FORGE_NORM_QK : 0) | rope | (norm_v ? FORGE_NORM_V : 0), r.cos, r.sin, r.sb, r.st, kc.data_ptr(),
        vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), max_len, static_cast<const int32_t*>(ptr(row_pos)),
        static_cast<const int64_t*>(ptr(pos_dev)), pos, max_kv, (int)window, scale, (int)chunk, out.data_ptr(),
        out.stride(0), out.stride(1), out.stride(2), ws.ptr, ws.bytes, ws.ptr ? FORGE_WS_ZEROED : 0, stream);
  }
  if (st == 0) ws.put_back();
  return result(st, out);
}

// kv_append(k, v, k_cache, v_cache, pos, k_weight | None, eps, norm_k, norm_v, cos | None, sin | None): host position
PyObject* kv_append_impl(PyObject* const* a) {
  Tensor k, v, kc, vc, kw, cos, sin;
  if (!take(a[0], k) || !take(a[1], v) || !take(a[2], kc) || !take(a[3], vc) || !take_opt(a[5], kw) ||
      !take_opt(a[9], cos) || !take_opt(a[10], sin))
    return nullptr;
  float eps;
  int64_t pos;
  if (!as_int(a[4], pos) || !as_float(a[6], eps)) return nullptr;
  const bool norm_k = a[7] == Py_True, norm_v = a[8] == Py_True;
  if (k.dim() != 4 || kc.dim() != 4 || k.sizes() != v.sizes() || kc.sizes() != vc.sizes() ||
      kc.strides() != vc.strides())
    return nullptr;
  const int64_t B = k.size(0), K = k.size(1), T = k.size(2), D = k.size(3);
  const int dt = dtype_of(kc);
  const c10::Device dev = k.device();
  if (dt < 0 || kc.size(0) != B || kc.size(1) != K || kc.size(3) != D || c10::hip::current_device() != dev.index())
    return nullptr;
  for (const Tensor* t : {&k, &v, &kc, &vc})
    if (t->scalar_type() != k.scalar_type() || t->device() != dev || t->stride(3) != 1) return nullptr;
  Rope r;
  if (!rope_ok(cos, sin, B, T, D, dev, r) || !gain_ok(kw, D, dev)) return nullptr;
  const int flags = (norm_k ? FORGE_NORM_QK : 0) | (r.cos ? FORGE_ROPE : 0) | (norm_v ? FORGE_NORM_V : 0);
  int st;
  {
    NoGil unlocked;
    st = forge_kv_append(
        dt, (int)B, (int)T, (int)K, (int)D, ptr(k), k.stride(0), k.stride(1), k.stride(2), ptr(v), v.stride(0),
        v.stride(1), v.stride(2), kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), kc.size(2),
        nullptr, nullptr, pos, norm_k ? static_cast<const float*>(ptr(kw)) : nullptr, eps, flags, r.cos, r.sin, r.sb,
        r.st, c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return PyLong_FromLong(st);
}

// prefill(q, k, v, scale, offset, window, q_weight | None, eps, norm_q, cos | None, sin | None): bf16/fp16 through
// forge_attn_prefill_ws, fp32 through forge_attn_prefill_f32
PyObject* prefill_impl(PyObject* const* a) {
  Tensor q, k, v, qw, cos, sin;
  if (!take(a[0], q) || !take(a[1], k) || !take(a[2], v) || !take_opt(a[6], qw) || !take_opt(a[9], cos) ||
      !take_opt(a[10], sin))
    return nullptr;
  float scale, eps;
  int64_t offset, window;
  if (!as_float(a[3], scale) || !as_int(a[4], offset) || !as_int(a[5], window) || !as_float(a[7], eps)) return nullptr;
  const bool norm_q = a[8] == Py_True;
  if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides()) return nullptr;
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), K = k.size(1);
  const int dt = dtype_of(q);
  const c10::Device dev = q.device();
  if (dt < 0 || K <= 0 || H % K || k.size(0) != B || k.size(3) != D || offset < 0 || k.size(2) - T < offset ||
      window < 0 || window > INT_MAX || q.stride(3) != 1 || c10::hip::current_device() != dev.index())
    return nullptr;
  for (const Tensor* t : {&k, &v})
    if (t->scalar_type() != q.scalar_type() || t->device() != dev || t->stride(3) != 1) return nullptr;
  Rope r;
  if ((cos.defined() && cos.dim() != 2) || !rope_ok(cos, sin, B, T, D, dev, r) || !gain_ok(qw, D, dev)) return nullptr;
  const bool f32 = dt == FORGE_F32;
  if (f32 ? D != 32 && D != 64 && D != 128 : D != 64 && D != 128 && D != 256 && D != 512) return nullptr;
  const int flags = (norm_q ? FORGE_NORM_QK : 0) | (r.cos ? FORGE_ROPE : 0);
  const float* w = norm_q ? static_cast<const float*>(ptr(qw)) : nullptr;
  const auto opts = q.options().requires_grad(false);
  Tensor out, ws;
  int st;
  {
    NoGil unlocked;
    out = at::empty({B, T, H, D}, opts);
    const size_t need =
        f32 ? forge_attn_prefill_f32_workspace_bytes((int)B, (int)T, (int)H, (int)K, (int)D, offset, (int)window)
            : forge_attn_prefill_workspace_bytes(dt, (int)B, (int)T, (int)H, (int)K, (int)D, offset, (int)window);
    if (need) {
      try {
        ws = at::empty({(int64_t)need}, opts.dtype(at::kByte));
      } catch (const c10::OutOfMemoryError&) {   // the launch is not split then
      }
    }
    void* wp = ws.defined() ? ws.data_ptr() : nullptr;
    const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    st = f32 ? forge_attn_prefill_f32((int)B, (int)T, (int)H, (int)K, (int)D, ptr(q), q.stride(0), q.stride(1),
                                      q.stride(2), w, eps, flags, r.cos, r.sin, r.st, ptr(k), ptr(v), k.stride(0),
                                      k.stride(1), k.stride(2), offset, (int)window, scale, out.data_ptr(),
                                      out.stride(0), out.stride(1), out.stride(2), wp, need, stream)
             : forge_attn_prefill_ws(dt, (int)B, (int)T, (int)H, (int)K, (int)D, ptr(q), q.stride(0), q.stride(1),
                                     q.stride(2), w, eps, flags, r.cos, r.sin, r.st, ptr(k), ptr(v), k.stride(0),
                                     k.stride(1), k.stride(2), offset, (int)window, scale, nullptr, 0, out.data_ptr(),
                                     out.stride(0), out.stride(1), out.stride(2), wp, need, stream);
  }
  return result(st, out);
}

// linear_small(x, w, bias | None, w_up | None, gain | None, eps, norm, residual | None): contiguous x [..., K] of at
// most 16 rows, w and w_up [N, K], residual [..., N]
PyObject* linear_small_impl(PyObject* const* a) {
  Tensor x, w, b, up, gain, res;
  if (!take(a[0], x) || !take(a[1], w) || !take_opt(a[2], b) || !take_opt(a[3], up) || !take_opt(a[4], gain) ||
      !take_opt(a[7], res))
    return nullptr;
  float eps;
  if (!as_float(a[5], eps) || x.dim() < 1 || w.dim() != 2) return nullptr;
  const bool norm = a[6] == Py_True;
  const int64_t K = x.size(-1), N = w.size(0);
  const int dt = dtype_of(x);
  const c10::Device dev = x.device();
  if (K <= 0 || K % 32 || (dt != FORGE_BF16 && dt != FORGE_F16) || !x.is_contiguous() || x.numel() < K ||
      x.numel() > 16 * K || w.size(1) != K || !w.is_contiguous() || c10::hip::current_device() != dev.index())
    return nullptr;
  for (const Tensor* t : {&w, &b, &up, &res})
    if (t->defined() && (t->scalar_type() != x.scalar_type() || t->device() != dev || !t->is_contiguous())) return nullptr;
  if ((b.defined() && b.numel() != N) || (up.defined() && up.sizes() != w.sizes())) return nullptr;
  if (norm && !gain.defined()) return nullptr;
  if (gain.defined() && ((gain.scalar_type() != at::kFloat && gain.scalar_type() != x.scalar_type()) ||
                         gain.device() != dev || !gain.is_contiguous() || gain.numel() != K))
    return nullptr;
  const int64_t M = x.numel() / K;
  if (res.defined() && res.numel() != M * N) return nullptr;
  if (N > INT_MAX || K > INT_MAX || M > forge_linear_small_rows((int)N, (int)K, norm, up.defined(), res.defined()))
    return nullptr;   // torch's calls are faster there
  if (((uintptr_t)ptr(x) | (uintptr_t)ptr(w) | (uintptr_t)ptr(up) | (uintptr_t)ptr(gain)) % 16) return nullptr;
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor out;
  int st;
  {
    NoGil unlocked;
    out = at::empty(shape, x.options().requires_grad(false));
    st = forge_linear_small(dt, (int)M, (int)N, (int)K, ptr(x), K, ptr(w), ptr(up), K, ptr(b), ptr(gain),
                            gain.defined() ? dtype_of(gain) : FORGE_F32, norm, eps, ptr(res), N, out.data_ptr(), N,
                            c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return result(st, out);
}

// tensors_are(tensors, ids, state, w): whether the tuple of tensors is the recorded one, by id and by
// (data_ptr, version) each, of w's dtype and device (w: Attention's fused q/k/v weights)
PyObject* tensors_are_impl(PyObject* const* a) {
  if (!PyTuple_CheckExact(a[0]) || !PyTuple_CheckExact(a[1]) || !PyTuple_CheckExact(a[2])) return nullptr;
  Tensor w;
  if (!take(a[3], w)) return nullptr;
  const Py_ssize_t n = PyTuple_GET_SIZE(a[0]);
  if (PyTuple_GET_SIZE(a[1]) != n || PyTuple_GET_SIZE(a[2]) != n) Py_RETURN_FALSE;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyTuple_GET_ITEM(a[0], i);
    PyObject* st = PyTuple_GET_ITEM(a[2], i);
    if (!THPVariable_Check(o) || !PyTuple_CheckExact(st) || PyTuple_GET_SIZE(st) < 2) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!plain(t) || t.is_inference()) return nullptr;
    if (t.scalar_type() != w.scalar_type() || t.device() != w.device()) Py_RETURN_FALSE;
    if (PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[1], i)) != o ||
        PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(st, 0)) != (unsigned long long)(uintptr_t)t.const_data_ptr() ||
        PyLong_AsLongLong(PyTuple_GET_ITEM(st, 1)) != (long long)t._version()) {
      PyErr_Clear();
      Py_RETURN_FALSE;
    }
  }
  Py_RETURN_TRUE;
}

// A tensor [.., .., .., D] that the paged kernels take as it is: the last dimension contiguous, pointer and strides
// multiples of 16 bytes (ops._aligned), its strides with 0 for dimensions of one element (ops._strides3).
bool strides16(const Tensor& t, int64_t (&s)[3]) {
  const int64_t e16 = 16 / t.element_size();
  if (t.dim() != 4 || t.stride(3) != 1 || (uintptr_t)t.const_data_ptr() % 16) return false;
  for (int i = 0; i < 3; ++i) {
    s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (s[i] < 0 || s[i] % e16) return false;
  }
  return true;
}

// int32 [B] on dev
bool rows_ok(const Tensor& t, int64_t B, c10::Device dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.is_contiguous() && t.device() == dev;
}

struct Pages {
  int64_t s[3], B, size, max, stride;
  int n;
};

// pools [n, K, size, D] and table [B, max] of one cache (ops._pages)
bool pages_ok(const Tensor& kp, const Tensor& vp, const Tensor& table, int64_t B, c10::Device dev, Pages& p) {
  int64_t sv[3];
  if (kp.dim() != 4 || kp.sizes() != vp.sizes() || kp.scalar_type() != vp.scalar_type() || kp.device() != dev ||
      vp.device() != dev || !strides16(kp, p.s) || !strides16(vp, sv) || !std::equal(p.s, p.s + 3, sv))
    return false;
  p.size = kp.size(2);
  if (p.size < 16 || p.size > INT_MAX || (p.size & (p.size - 1)) || kp.size(0) < 1 || kp.size(0) > INT_MAX) return false;
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != B || table.size(1) < 1 ||
      table.size(1) > INT_MAX || table.stride(1) != 1 || table.device() != dev)
    return false;
  p.n = (int)kp.size(0);
  p.max = table.size(1);
  p.stride = B > 1 ? table.stride(0) : 0;
  return p.stride >= 0;
}

// kv_append_paged(k, v, k_pages, v_pages, table, row_pos, new_lens | None, k_weight | None, eps, norm_k, norm_v,
//                 cos | None, sin | None)
PyObject* kv_append_paged_impl(PyObject* const* a) {
  Tensor k, v, kp, vp, table, row_pos, news, kw, cos, sin;
  if (!take(a[0], k) || !take(a[1], v) || !take(a[2], kp) || !take(a[3], vp) || !take(a[4], table) ||
      !take(a[5], row_pos) || !take_opt(a[6], news) || !take_opt(a[7], kw) || !take_opt(a[11], cos) || !take_opt(a[12], sin))
    return nullptr;
  float eps;
  if (!as_float(a[8], eps) || k.dim() != 4 || k.sizes() != v.sizes()) return nullptr;
  const bool norm_k = a[9] == Py_True, norm_v = a[10] == Py_True;
  const int64_t B = k.size(0), K = k.size(1), T = k.size(2), D = k.size(3);
  const int dt = dtype_of(kp);
  const c10::Device dev = k.device();
  Pages p;
  int64_t sk[3], sv[3];
  if (dt < 0 || k.scalar_type() != kp.scalar_type() || v.scalar_type() != kp.scalar_type() || v.device() != dev ||
      c10::hip::current_device() != dev.index() || !strides16(k, sk) || !strides16(v, sv) ||
      !pages_ok(kp, vp, table, B, dev, p) || kp.size(1) != K || kp.size(3) != D || !rows_ok(row_pos, B, dev) ||
      (news.defined() && !rows_ok(news, B, dev)))
    return nullptr;
  Rope r;
  if (!rope_ok(cos, sin, B, T, D, dev, r) || !gain_ok(kw, D, dev)) return nullptr;
  const int flags = (norm_k ? FORGE_NORM_QK : 0) | (r.cos ? FORGE_ROPE : 0) | (norm_v ? FORGE_NORM_V : 0);
  int st;
  {
    NoGil unlocked;
    st = forge_kv_append_paged(dt, (int)B, (int)T, (int)K, (int)D, ptr(k), sk[0], sk[1], sk[2], ptr(v), sv[0], sv[1], sv[2],
                               kp.data_ptr(), vp.data_ptr(), p.s[0], p.s[1], p.s[2], p.n, (int)p.size,
                               static_cast<const int32_t*>(ptr(table)), p.stride, (int)p.max,
                               static_cast<const int32_t*>(ptr(row_pos)), static_cast<const int32_t*>(ptr(news)),
                               norm_k ? static_cast<const float*>(ptr(kw)) : nullptr, eps, flags, r.cos, r.sin, r.sb, r.st,
                               c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return st >= 0 ? PyLong_FromLong(st) : nullptr;   // (a rejected call gets its error the Python way)
}

// What attn_paged and attn_sinks have in common: q, its norm and tables, window and sinks, the output and the partials.
struct NewTokens {
  Tensor q, qw, cos, sin, out, ws;
  float scale, eps;
  int64_t window, sinks, sq[3], B, H, T, D;
  int dt, flags;
  const float* w;
  Rope r;
  size_t need = 0;

  bool take_args(const Tensor& cache) {
    if (q.dim() != 4 || cache.dim() != 4 || !strides16(q, sq)) return false;
    B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
    dt = dtype_of(q);
    const c10::Device dev = q.device();
    const int64_t K = cache.size(1);
    if (dt < 0 || K <= 0 || H % K || cache.size(3) != D || cache.scalar_type() != q.scalar_type() || B < 1 || T < 1 ||
        B > INT_MAX || H > INT_MAX || T > INT_MAX || window < 0 || sinks < 0 || window > INT_MAX / 2 ||
        sinks > INT_MAX / 2 || (sinks && !window) || c10::hip::current_device() != dev.index())
      return false;
    if (!rope_ok(cos, sin, B, T, D, dev, r) || !gain_ok(qw, D, dev) || (uintptr_t)ptr(qw) % 16) return false;
    return true;
  }
  void size(int64_t K, int64_t max_kv, bool tree = false) {
    need = (tree ? forge_attn_tree_workspace_bytes : forge_attn_paged_workspace_bytes)(
        dt, (int)B, (int)T, (int)H, (int)K, (int)D, max_kv, (int)window, (int)sinks);
  }
  // Calls of few partials outside graph capture use their stream's workspace (ops._PagedPartials)
  bool keep() const { return need && need <= ((size_t)32 << 20) && !capturing(); }
  void set_flags(bool norm_q) {
    flags = (norm_q ? FORGE_NORM_QK : 0) | (r.cos ? FORGE_ROPE : 0);
    w = norm_q ? static_cast<const float*>(ptr(qw)) : nullptr;
  }
  // (without the GIL) the output, and memory for the partials of a split launch where the stream's workspace does not
  // serve; without it nothing is split
  void allocate(bool kept) {
    const auto opts = q.options().requires_grad(false);
    out = at::empty({B, T, H, D}, opts);
    if (!need || kept) return;
    try {
      ws = at::empty({(int64_t)need}, opts.dtype(at::kByte));
    } catch (const c10::OutOfMemoryError&) {
    }
  }
};

// attn_paged(table of workspaces, q, k_pages, v_pages, table, row_pos, new_lens | None, scale, max_kv_len | None, window, sinks,
//            q_weight | None, eps, norm_q, cos | None, sin | None)
PyObject* attn_paged_impl(PyObject* const* a) {
  NewTokens n;
  Tensor kp, vp, table, row_pos, news;
  int64_t max_kv = 0;
  if (!take(a[1], n.q) || !take(a[2], kp) || !take(a[3], vp) || !take(a[4], table) || !take(a[5], row_pos) ||
      !take_opt(a[6], news) || !as_float(a[7], n.scale) || (a[8] != Py_None && !as_int(a[8], max_kv)) ||
      !as_int(a[9], n.window) || !as_int(a[10], n.sinks) || !take_opt(a[11], n.qw) || !as_float(a[12], n.eps) ||
      !take_opt(a[14], n.cos) || !take_opt(a[15], n.sin))
    return nullptr;
  if (!n.take_args(kp)) return nullptr;
  const c10::Device dev = n.q.device();
  Pages p;
  if (!pages_ok(kp, vp, table, n.B, dev, p) || !rows_ok(row_pos, n.B, dev) || (news.defined() && !rows_ok(news, n.B, dev)))
    return nullptr;
  const int64_t most = p.max * p.size, K = kp.size(1);
  max_kv = a[8] == Py_None ? most : std::min(max_kv, most);
  if (max_kv < 1) return nullptr;
  n.set_flags(a[13] == Py_True);
  n.size(K, max_kv);
  const bool kept = n.keep();
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  StreamWorkspace ws(a[0], dev.index(), stream, kept ? n.need : 0);
  if (kept && !ws.ptr) return nullptr;   // (made the Python way)
  int st;
  {
    NoGil unlocked;
    n.allocate(kept);
    st = forge_attn_paged(n.dt, (int)n.B, (int)n.T, (int)n.H, (int)K, (int)n.D, ptr(n.q), n.sq[0], n.sq[1], n.sq[2], n.w,
                          n.eps, n.flags, n.r.cos, n.r.sin, n.r.sb, n.r.st, ptr(kp), ptr(vp), p.s[0], p.s[1], p.s[2], p.n,
                          (int)p.size, static_cast<const int32_t*>(ptr(table)), p.stride, (int)p.max,
                          static_cast<const int32_t*>(ptr(row_pos)), static_cast<const int32_t*>(ptr(news)), max_kv,
                          (int)n.window, (int)n.sinks, n.scale, n.out.data_ptr(), n.out.stride(0), n.out.stride(1),
                          n.out.stride(2), kept ? ws.ptr : n.ws.defined() ? n.ws.data_ptr() : nullptr,
                          kept ? ws.bytes : n.need, kept ? FORGE_WS_ZEROED : 0, stream);
  }
  if (st == 0) ws.put_back();
  return st < 0 ? nullptr : result(st, n.out);
}

// attn_sinks(table of workspaces, q, k_cache, v_cache, scale, window, sinks, pos | None, pos_dev | None, row_pos | None, max_kv_len | None,
//            q_weight | None, eps, norm_q, cos | None, sin | None, fixed_cut)
PyObject* attn_sinks_impl(PyObject* const* a) {
  NewTokens n;
  Tensor kc, vc, pos_dev, row_pos;
  int64_t pos = 0, max_kv = INT64_MAX, sk[3], sv[3];
  if (!take(a[1], n.q) || !take(a[2], kc) || !take(a[3], vc) || !as_float(a[4], n.scale) || !as_int(a[5], n.window) ||
      !as_int(a[6], n.sinks) || (a[7] != Py_None && !as_int(a[7], pos)) || !take_opt(a[8], pos_dev) ||
      !take_opt(a[9], row_pos) || (a[10] != Py_None && !as_int(a[10], max_kv)) || !take_opt(a[11], n.qw) ||
      !as_float(a[12], n.eps) || !take_opt(a[14], n.cos) || !take_opt(a[15], n.sin))
    return nullptr;
  if (!n.take_args(kc) || n.window < 1) return nullptr;
  const c10::Device dev = n.q.device();
  if (kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type() || kc.device() != dev || vc.device() != dev ||
      kc.size(0) != n.B || !strides16(kc, sk) || !strides16(vc, sv) || !std::equal(sk, sk + 3, sv))
    return nullptr;
  const int64_t K = kc.size(1), max_len = kc.size(2);
  if (row_pos.defined()) {
    if (!rows_ok(row_pos, n.B, dev)) return nullptr;
    pos_dev.reset();
    pos = 0;
  } else if (pos_dev.defined()) {
    if (pos_dev.scalar_type() != at::kLong || pos_dev.numel() < 1 || pos_dev.device() != dev) return nullptr;
    pos = 0;
  } else {
    if (pos < 0 || pos > max_len - n.T) return nullptr;
    max_kv = pos + n.T;
  }
  max_kv = std::min(max_kv, max_len);
  if (max_kv < 1) return nullptr;
  n.set_flags(a[13] == Py_True);
  if (a[16] == Py_True) {
    if (n.T > FORGE_FIXED_CUT_MAX_T) return nullptr;
    n.flags |= FORGE_FIXED_CUT;
    n.need = forge_attn_sinks_fixed_workspace_bytes(n.dt, (int)n.B, (int)n.T, (int)n.H, (int)K, (int)n.D, max_len,
                                                    (int)n.window, (int)n.sinks);
  } else {
    n.size(K, max_kv);
  }
  const bool kept = n.keep();
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  StreamWorkspace ws(a[0], dev.index(), stream, kept ? n.need : 0);
  if (kept && !ws.ptr) return nullptr;   // (made the Python way)
  int st;
  {
    NoGil unlocked;
    n.allocate(kept);
    if ((n.flags & FORGE_FIXED_CUT) && n.need && !kept && !n.ws.defined()) return nullptr;   // (raised the Python way)
    st = forge_attn_sinks(n.dt, (int)n.B, (int)n.T, (int)n.H, (int)K, (int)n.D, ptr(n.q), n.sq[0], n.sq[1], n.sq[2], n.w,
                          n.eps, n.flags, n.r.cos, n.r.sin, n.r.sb, n.r.st, ptr(kc), ptr(vc), sk[0], sk[1],
                          max_len > 1 ? sk[2] : n.D, max_len, static_cast<const int32_t*>(ptr(row_pos)),
                          static_cast<const int64_t*>(ptr(pos_dev)), pos, max_kv, (int)n.window, (int)n.sinks, n.scale,
                          n.out.data_ptr(), n.out.stride(0), n.out.stride(1), n.out.stride(2),
                          kept ? ws.ptr : n.ws.defined() ? n.ws.data_ptr() : nullptr,
                          kept ? ws.bytes : n.need, kept ? FORGE_WS_ZEROED : 0, stream);
  }
  if (st == 0) ws.put_back();
  return st < 0 ? nullptr : result(st, n.out);
}

// A tree's bits [B, T, words] or [T, words] and depths [B, T] or [T] (ops._tree_args)
struct Tree {
  Tensor mask, depth, news;
  int64_t mb = 0, mt = 0, db = 0;
  bool ok(int64_t B, int64_t T, int64_t window, c10::Device dev) {
    const int64_t words = (T + 63) / 64, d = mask.dim();
    if (T > FORGE_TREE_MAX_TOKENS || mask.scalar_type() != at::kLong || mask.device() != dev || (d != 2 && d != 3) ||
        mask.size(d - 1) != words || mask.size(d - 2) != T || (d == 3 && mask.size(0) != B) ||
        (words > 1 && mask.stride(d - 1) != 1) || (window && !depth.defined()))
      return false;
    mt = T > 1 ? mask.stride(d - 2) : 0;
    mb = d == 3 && B > 1 ? mask.stride(0) : 0;
    if (mt < 0 || mb < 0) return false;
    if (depth.defined()) {
      const int64_t e = depth.dim();
      if (depth.scalar_type() != at::kInt || depth.device() != dev || (e != 1 && e != 2) || depth.size(e - 1) != T ||
          (e == 2 && depth.size(0) != B) || (T > 1 && depth.stride(e - 1) != 1))
        return false;
      db = e == 2 && B > 1 ? depth.stride(0) : 0;
    }
    return !news.defined() || rows_ok(news, B, dev);
  }
};

// What attn_tree and attn_tree_paged share once their caches are checked.
PyObject* launch_tree(PyObject* table, NewTokens& n, Tree& t, const Tensor& kc, const Tensor& vc, const int64_t (&sk)[3],
                      int64_t sks, int n_pages, int64_t page_size, const Tensor& pages, int64_t s_table, int64_t max_pages,
                      const Tensor& row_pos, const Tensor& pos_dev, int64_t pos, int64_t max_kv, bool norm_q) {
  const c10::Device dev = n.q.device();
  const int64_t K = kc.size(1);
  n.set_flags(norm_q);
  n.size(K, max_kv, true);
  const bool kept = n.keep();
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  StreamWorkspace ws(table, dev.index(), stream, kept ? n.need : 0);
  if (kept && !ws.ptr) return nullptr;   // (made the Python way)
  int st;
  {
    NoGil unlocked;
    n.allocate(kept);
    st = forge_attn_tree(n.dt, (int)n.B, (int)n.T, (int)n.H, (int)K, (int)n.D, ptr(n.q), n.sq[0], n.sq[1], n.sq[2], n.w, n.eps,
                         n.flags, n.r.cos, n.r.sin, n.r.sb, n.r.st, ptr(kc), ptr(vc), sk[0], sk[1], sks, n_pages, page_size,
                         static_cast<const int32_t*>(ptr(pages)), s_table, (int)max_pages,
                         static_cast<const int32_t*>(ptr(row_pos)), static_cast<const int64_t*>(ptr(pos_dev)), pos,
                         static_cast<const int32_t*>(ptr(t.news)), max_kv, (int)n.window, (int)n.sinks, n.scale,
                         static_cast<const int64_t*>(ptr(t.mask)), t.mb, t.mt, static_cast<const int32_t*>(ptr(t.depth)), t.db,
                         n.out.data_ptr(), n.out.stride(0), n.out.stride(1), n.out.stride(2),
                         kept ? ws.ptr : n.ws.defined() ? n.ws.data_ptr() : nullptr, kept ? ws.bytes : n.need,
                         kept ? FORGE_WS_ZEROED : 0, stream);
  }
  if (st == 0) ws.put_back();
  return st < 0 ? nullptr : result(st, n.out);
}

// attn_tree(table of workspaces, q, k_cache, v_cache, mask, scale, pos | None, pos_dev | None, row_pos | None, depth | None,
//           new_lens | None, max_kv_len | None, window, sinks, q_weight | None, eps, norm_q, cos | None, sin | None)
PyObject* attn_tree_impl(PyObject* const* a) {
  NewTokens n;
  Tree t;
  Tensor kc, vc, pos_dev, row_pos;
  int64_t pos = 0, max_kv = INT64_MAX, sk[3], sv[3];
  if (!take(a[1], n.q) || !take(a[2], kc) || !take(a[3], vc) || !take(a[4], t.mask) || !as_float(a[5], n.scale) ||
      (a[6] != Py_None && !as_int(a[6], pos)) || !take_opt(a[7], pos_dev) || !take_opt(a[8], row_pos) ||
      !take_opt(a[9], t.depth) || !take_opt(a[10], t.news) || (a[11] != Py_None && !as_int(a[11], max_kv)) ||
      !as_int(a[12], n.window) || !as_int(a[13], n.sinks) || !take_opt(a[14], n.qw) || !as_float(a[15], n.eps) ||
      !take_opt(a[17], n.cos) || !take_opt(a[18], n.sin))
    return nullptr;
  if (!n.take_args(kc) || (a[6] != Py_None) + pos_dev.defined() + row_pos.defined() > 1) return nullptr;
  const c10::Device dev = n.q.device();
  if (kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type() || kc.device() != dev || vc.device() != dev ||
      kc.size(0) != n.B || !strides16(kc, sk) || !strides16(vc, sv) || !std::equal(sk, sk + 3, sv) ||
      !t.ok(n.B, n.T, n.window, dev))
    return nullptr;
  const int64_t max_len = kc.size(2);
  if (row_pos.defined()) {
    if (!rows_ok(row_pos, n.B, dev)) return nullptr;
  } else if (pos_dev.defined()) {
    if (pos_dev.scalar_type() != at::kLong || pos_dev.numel() < 1 || pos_dev.device() != dev) return nullptr;
  } else {
    if (pos < 0 || pos > max_len - n.T) return nullptr;
    max_kv = pos + n.T;
  }
  max_kv = std::min(max_kv, max_len);
  if (max_kv < 1) return nullptr;
  return launch_tree(a[0], n, t, kc, vc, sk, max_len > 1 ? sk[2] : n.D, 1, max_len, Tensor(), 0, 0, row_pos, pos_dev, pos, max_kv,
                     a[16] == Py_True);
}

// attn_tree_paged(table of workspaces, q, k_pages, v_pages, table, row_pos, mask, scale, depth | None, new_lens | None,
//                 max_kv_len | None, window, sinks, q_weight | None, eps, norm_q, cos | None, sin | None)
PyObject* attn_tree_paged_impl(PyObject* const* a) {
  NewTokens n;
  Tree t;
  Tensor kp, vp, table, row_pos;
  int64_t max_kv = INT64_MAX;
  if (!take(a[1], n.q) || !take(a[2], kp) || !take(a[3], vp) || !take(a[4], table) || !take(a[5], row_pos) ||
      !take(a[6], t.mask) || !as_float(a[7], n.scale) || !take_opt(a[8], t.depth) || !take_opt(a[9], t.news) ||
      (a[10] != Py_None && !as_int(a[10], max_kv)) || !as_int(a[11], n.window) || !as_int(a[12], n.sinks) ||
      !take_opt(a[13], n.qw) || !as_float(a[14], n.eps) || !take_opt(a[16], n.cos) || !take_opt(a[17], n.sin))
    return nullptr;
  if (!n.take_args(kp)) return nullptr;
  const c10::Device dev = n.q.device();
  Pages p;
  if (!pages_ok(kp, vp, table, n.B, dev, p) || !rows_ok(row_pos, n.B, dev) || !t.ok(n.B, n.T, n.window, dev)) return nullptr;
  max_kv = std::min(max_kv, p.max * p.size);
  if (max_kv < 1) return nullptr;
  return launch_tree(a[0], n, t, kp, vp, p.s, p.s[2], p.n, p.size, table, p.stride, p.max, row_pos, Tensor(), 0, max_kv,
                     a[15] == Py_True);
}

PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const Tensor& t : ts)
    if (r) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}

// tree_mask(parents, new_lens | None)
PyObject* tree_mask_impl(PyObject* const* a) {
  Tensor parents, news;
  if (!take(a[0], parents) || !take_opt(a[1], news)) return nullptr;
  const c10::Device dev = parents.device();
  if (parents.scalar_type() != at::kInt || parents.dim() != 2 || c10::hip::current_device() != dev.index()) return nullptr;
  const int64_t B = parents.size(0), T = parents.size(1);
  if (B < 1 || B > INT_MAX || T < 1 || T > FORGE_TREE_MAX_TOKENS || (T > 1 && parents.stride(1) != 1) ||
      (news.defined() && !rows_ok(news, B, dev)))
    return nullptr;
  Tensor mask, depth;
  int st;
  {
    NoGil unlocked;
    mask = at::empty({B, T, (T + 63) / 64}, parents.options().dtype(at::kLong));
    depth = at::empty({B, T}, parents.options());
    st = forge_tree_mask((int)B, (int)T, static_cast<const int32_t*>(ptr(parents)), B > 1 ? parents.stride(0) : 0,
                         static_cast<const int32_t*>(ptr(news)), static_cast<int64_t*>(mask.data_ptr()),
                         static_cast<int32_t*>(depth.data_ptr()), c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  if (st) return st < 0 ? nullptr : PyLong_FromLong(st);
  return tuple_of({mask, depth});
}

// [B, T] of a type on dev with its rows contiguous, or undefined
bool rows2_ok(const Tensor& t, at::ScalarType type, int64_t B, int64_t T, c10::Device dev, int64_t& stride) {
  stride = 0;
  if (!t.defined()) return true;
  if (t.scalar_type() != type || t.dim() != 2 || t.size(0) != B || t.size(1) != T || t.device() != dev ||
      (T > 1 && t.stride(1) != 1))
    return false;
  if (B > 1) stride = t.stride(0);
  return true;
}

// verify_drafts(table of workspaces, logits, tokens, parents | None, uniform | None, temperature, draft_probs | None, new_lens | None)
PyObject* verify_drafts_impl(PyObject* const* a) {
  Tensor logits, tokens, parents, uniform, temps, probs, news;
  if (!take(a[1], logits) || !take(a[2], tokens) || !take_opt(a[3], parents) || !take_opt(a[4], uniform) ||
      !take_opt(a[6], probs) || !take_opt(a[7], news))
    return nullptr;
  double heat = 0.0;
  if (PyFloat_CheckExact(a[5])) heat = PyFloat_AS_DOUBLE(a[5]);
  else if (!take(a[5], temps)) return nullptr;
  const c10::Device dev = logits.device();
  const int dt = dtype_of(logits);
  if (dt < 0 || logits.dim() != 3 || c10::hip::current_device() != dev.index()) return nullptr;
  const int64_t B = logits.size(0), T = logits.size(1), V = logits.size(2);
  int64_t st_, sp, su;
  if (B < 1 || B > INT_MAX || T < 1 || T > FORGE_TREE_MAX_TOKENS || V < 1 || V > INT_MAX || (V > 1 && logits.stride(2) != 1) ||
      !rows2_ok(tokens, at::kLong, B, T, dev, st_) || !rows2_ok(parents, at::kInt, B, T, dev, sp) ||
      !rows2_ok(uniform, at::kFloat, B, T, dev, su) || (news.defined() && !rows_ok(news, B, dev)))
    return nullptr;
  if (temps.defined() && (temps.scalar_type() != at::kFloat || temps.dim() != 1 || temps.size(0) != B ||
                          !temps.is_contiguous() || temps.device() != dev))
    return nullptr;
  if ((temps.defined() || heat != 0.0) && !uniform.defined()) return nullptr;
  if (T == 1) probs.reset();
  int pdt = 0;
  if (probs.defined()) {
    pdt = dtype_of(probs);
    if ((pdt != FORGE_F32 && pdt != dt) || probs.dim() != 3 || probs.size(0) != B ||
        (probs.size(1) != T && probs.size(1) != T - 1) || probs.size(2) != V || (V > 1 && probs.stride(2) != 1) ||
        probs.device() != dev)
      return nullptr;
  }
  const size_t need = forge_verify_drafts_workspace_bytes((int)B, (int)T, (int)V, probs.defined());
  if (!need) return nullptr;
  const bool kept = need <= ((size_t)32 << 20) && !capturing();
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  StreamWorkspace sw(a[0], dev.index(), stream, kept ? need : 0);
  if (kept && !sw.ptr) return nullptr;   // (made the Python way)
  Tensor out, path, count, ws;
  int st;
  {
    NoGil unlocked;
    out = at::empty({B, T}, tokens.options());
    path = at::empty({B, T}, tokens.options().dtype(at::kInt));
    count = at::empty({B}, tokens.options().dtype(at::kInt));
    if (!kept) ws = at::empty({(int64_t)need}, tokens.options().dtype(at::kByte));
    st = forge_verify_drafts(dt, (int)B, (int)T, (int)V, ptr(logits), logits.stride(0), logits.stride(1),
                             static_cast<const int64_t*>(ptr(tokens)), st_, static_cast<const int32_t*>(ptr(parents)), sp,
                             static_cast<const float*>(ptr(uniform)), su, static_cast<const float*>(ptr(temps)), heat, pdt,
                             ptr(probs), probs.defined() ? probs.stride(0) : 0, probs.defined() ? probs.stride(1) : 0,
                             static_cast<const int32_t*>(ptr(news)), static_cast<int64_t*>(out.data_ptr()),
                             static_cast<int32_t*>(path.data_ptr()), static_cast<int32_t*>(count.data_ptr()),
                             kept ? sw.ptr : ws.data_ptr(), kept ? sw.bytes : need, kept ? FORGE_WS_ZEROED : 0, stream);
  }
  if (st == 0) sw.put_back();
  if (st) return st < 0 ? nullptr : PyLong_FromLong(st);
  return tuple_of({out, path, count});
}

// The K and V caches of layers of one shape and layout (ops._layer_groups takes the others)
struct Layers {
  std::vector<const void*> k, v;
  Tensor first;
  int64_t s[3];
  bool take_lists(PyObject* ks, PyObject* vs) {
    const auto sequence = [](PyObject* o) { return PyList_CheckExact(o) || PyTuple_CheckExact(o); };
    if (!sequence(ks) || !sequence(vs)) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(ks);
    if (n < 1 || PySequence_Fast_GET_SIZE(vs) != n) return false;
    k.reserve(n);
    v.reserve(n);
    for (Py_ssize_t i = 0; i < 2 * n; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(i < n ? ks : vs, i % n);
      if (i == 0) {
        if (!take(o, first) || first.dim() != 4 || dtype_of(first) < 0 || first.size(3) * first.element_size() % 16 ||
            !strides16(first, s) || c10::hip::current_device() != first.device().index())
          return false;
        for (int d = 0; d < 4; ++d)
          if (first.stride(d) == 0 && first.size(d) > 1) return false;
        k.push_back(first.const_data_ptr());
        continue;
      }
      // (the others are plain tensors if they are what the first is; of 56 the full look takes longer than the launch)
      if (!THPVariable_CheckExact(o)) return false;
      const Tensor& t = THPVariable_Unpack(o);
      const c10::TensorImpl *x = t.unsafeGetTensorImpl(), *y = first.unsafeGetTensorImpl();
      if (!t.defined() || x->key_set() != y->key_set() || x->is_python_dispatch() || !x->has_storage() ||
          x->dtype() != y->dtype() || x->device() != y->device() || x->sizes() != y->sizes() || x->strides() != y->strides() ||
          t._fw_grad(0).defined())
        return false;
      const void* at = t.const_data_ptr();
      if ((uintptr_t)at % 16) return false;
      (i < n ? k : v).push_back(at);
    }
    return true;
  }
};

PyObject* status(int st) { return st < 0 ? nullptr : PyLong_FromLong(st); }

// kv_compact(k_caches, v_caches, path, count, pos | None, pos_dev | None, row_pos | None)
PyObject* kv_compact_impl(PyObject* const* a) {
  Layers l;
  Tensor path, count, pos_dev, row_pos;
  int64_t pos = 0, sp;
  if (!take(a[2], path) || !take(a[3], count) || (a[4] != Py_None && !as_int(a[4], pos)) || !take_opt(a[5], pos_dev) ||
      !take_opt(a[6], row_pos) || !l.take_lists(a[0], a[1]))
    return nullptr;
  const c10::Device dev = l.first.device();
  const int64_t B = l.first.size(0), max_len = l.first.size(2);
  if (path.dim() != 2 || B < 1 || max_len < 1 || path.size(1) < 1 || path.size(1) > INT_MAX || pos < 0 ||
      !rows2_ok(path, at::kInt, B, path.size(1), dev, sp) || !rows_ok(count, B, dev) ||
      (row_pos.defined() && !rows_ok(row_pos, B, dev)) ||
      (pos_dev.defined() && (pos_dev.scalar_type() != at::kLong || pos_dev.numel() < 1 || pos_dev.device() != dev)) ||
      (a[4] != Py_None) + pos_dev.defined() + row_pos.defined() > 1)
    return nullptr;
  int st;
  {
    NoGil unlocked;
    st = forge_kv_compact((int)l.first.element_size(), (int)l.k.size(), (int)B, (int)l.first.size(1), (int)l.first.size(3),
                          l.k.data(), l.v.data(), l.s[0], l.s[1], l.s[2], (int)B, max_len, nullptr, 0, 0,
                          static_cast<const int32_t*>(ptr(row_pos)), static_cast<const int64_t*>(ptr(pos_dev)), pos,
                          static_cast<const int32_t*>(ptr(path)), sp, (int)path.size(1),
                          static_cast<const int32_t*>(ptr(count)), c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return status(st);
}

// kv_compact_paged(k_pools, v_pools, table, row_pos, path, count)
PyObject* kv_compact_paged_impl(PyObject* const* a) {
  Layers l;
  Tensor table, row_pos, path, count;
  int64_t sp;
  if (!take(a[2], table) || !take(a[3], row_pos) || !take(a[4], path) || !take(a[5], count) || !l.take_lists(a[0], a[1]))
    return nullptr;
  const c10::Device dev = l.first.device();
  if (path.dim() != 2) return nullptr;
  const int64_t B = path.size(0), T = path.size(1);
  Pages p;
  if (B < 1 || T < 1 || T > INT_MAX || !rows2_ok(path, at::kInt, B, T, dev, sp) || !rows_ok(count, B, dev) ||
      !rows_ok(row_pos, B, dev) || !pages_ok(l.first, l.first, table, B, dev, p))
    return nullptr;
  int st;
  {
    NoGil unlocked;
    st = forge_kv_compact((int)l.first.element_size(), (int)l.k.size(), (int)B, (int)l.first.size(1), (int)l.first.size(3),
                          l.k.data(), l.v.data(), l.s[0], l.s[1], l.s[2], p.n, p.size,
                          static_cast<const int32_t*>(ptr(table)), p.stride, (int)p.max,
                          static_cast<const int32_t*>(ptr(row_pos)), nullptr, 0, static_cast<const int32_t*>(ptr(path)), sp,
                          (int)T, static_cast<const int32_t*>(ptr(count)), c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return status(st);
}

// copy_pages(k_pools, v_pools, src, dst), the page numbers as tensors
PyObject* copy_pages_impl(PyObject* const* a) {
  Layers l;
  Tensor src, dst;
  if (!take(a[2], src) || !take(a[3], dst) || !l.take_lists(a[0], a[1])) return nullptr;
  const c10::Device dev = l.first.device();
  const int64_t n = src.numel(), size = l.first.size(2);
  if (src.dim() != 1 || n < 1 || n > INT_MAX || !rows_ok(src, n, dev) || !rows_ok(dst, n, dev) || size > INT_MAX ||
      l.first.size(0) < 1 || l.first.size(0) > INT_MAX)
    return nullptr;
  int st;
  {
    NoGil unlocked;
    st = forge_copy_pages((int)l.first.element_size(), (int)l.k.size(), (int)l.first.size(1), (int)l.first.size(3), l.k.data(),
                          l.v.data(), l.s[0], l.s[1], l.s[2], (int)l.first.size(0), (int)size, (int)n,
                          static_cast<const int32_t*>(ptr(src)), static_cast<const int32_t*>(ptr(dst)),
                          c10::hip::getCurrentHIPStream(dev.index()).stream());
  }
  return status(st);
}

// An exception on the way (out of memory, for one) goes the Python way too, which raises it there.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    PyObject* r = F(args);
    if (r) return r;
    if (PyErr_Occurred()) PyErr_Clear();
  } catch (...) {
    PyErr_Clear();
  }
  Py_RETURN_NONE;
}

#define FORGE_ENTRY(NAME, N) \
  {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<NAME##_impl, N>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FORGE_ENTRY(decode_append, 21), FORGE_ENTRY(kv_append, 11), FORGE_ENTRY(prefill, 11),
    FORGE_ENTRY(linear_small, 8),   FORGE_ENTRY(tensors_are, 4), FORGE_ENTRY(kv_append_paged, 13),
    FORGE_ENTRY(attn_paged, 16),    FORGE_ENTRY(attn_sinks, 17), FORGE_ENTRY(tree_mask, 2),
    FORGE_ENTRY(attn_tree, 19),     FORGE_ENTRY(attn_tree_paged, 18), FORGE_ENTRY(verify_drafts, 8),
    FORGE_ENTRY(kv_compact, 7),     FORGE_ENTRY(kv_compact_paged, 6), FORGE_ENTRY(copy_pages, 4), {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_forge_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__forge_host(void) { return PyModule_Create(&module); }
