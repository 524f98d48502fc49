// CPython extension `mqk._front`: the Python entry points' checks, output
// allocations and native call in C++, for ordinary calls.
//
// A decode-size kernel takes 5-16 us, and the Python of one call (a dozen tensors
// checked attribute by attribute, three torch.empty, two ctypes calls) took 11-30 us,
// so those calls ran at the host's pace.  Measured per call, host only: mqk.fused_qkv_rope
// 13.7 -> 7.7 us, fused_qkv_rope_ex with the input norm and the paged write 19.1 -> 10.0 us,
// its W4A16 twin 29.9 -> 8.9 us, a LinearW4A16 11.3 -> 6.0 us (what is left is mostly the
// launches themselves).
//
// Every function returns a result only if the call is an ordinary one: plain dense
// tensors on the current device with the expected types and shapes, contiguous and
// 16-byte aligned, no tensor subclass, functorch wrapper or torch mode, and a
// workspace that is there and large enough.  Anything else -- an error to raise, a
// tensor to copy or convert, another device, a workspace to make -- returns None, and
// the Python code beside it, which remains the definition of the entry point, takes
// the call.  A native failure returns the status for Python to raise.
//
// The GIL is released where a call can wait for the driver: the output allocations and
// the launches (a full queue, or one whose host function needs the GIL).  Every pointer
// is read from its tensor before; 0.1 us of a call.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <dlfcn.h>

#include <cmath>

#include "../../include/mqk.h"

namespace {

// Entry points of the loaded libmqk.so (bind()).
struct Lib {
  decltype(&mqk_fused_qkv_rope_bf16) bf16 = nullptr;
  decltype(&mqk_fused_qkv_rope_f32) f32 = nullptr;
  decltype(&mqk_fused_qkv_rope_f16_ws) f16 = nullptr;
  decltype(&mqk_fused_qkv_rope_f16_workspace_size) f16_size = nullptr;
  decltype(&mqk_fused_qkv_rope_workspace_size) size = nullptr;
  decltype(&mqk_fused_qkv_rope_ex_workspace_size) ex_size = nullptr;
  decltype(&mqk_fused_qkv_rope_w4a16_workspace_size) w4_size = nullptr;
  decltype(&mqk_fused_qkv_rope_ex_bf16) ex = nullptr;
  decltype(&mqk_fused_qkv_rope_ex_w4a16) ex_w4 = nullptr;
  decltype(&mqk_w4a16_gemm_workspace_size) gemm_size = nullptr;
  decltype(&mqk_w4a16_gemm_ex) gemm = nullptr;
  decltype(&mqk_attn_prefill) attn = nullptr;
  decltype(&mqk_attn_prefill_workspace_size) attn_size = nullptr;
  decltype(&mqk_kv4_write) kv4_write = nullptr;
  decltype(&mqk_kv4_read) kv4_read = nullptr;
  decltype(&mqk_kv4_attn) kv4_attn = nullptr;
  decltype(&mqk_kv4_attn_workspace_size) kv4_attn_size = nullptr;
  decltype(&mqk_kv4_evict) kv4_evict = nullptr;
  decltype(&mqk_paged_tables) paged_tables = nullptr;
  decltype(&mqk_paged_attn) paged_attn = nullptr;
  decltype(&mqk_paged_attn_workspace_size) paged_attn_size = nullptr;
  decltype(&mqk_paged_bounds) paged_bounds = nullptr;
  decltype(&mqk_paged_select) paged_select = nullptr;
  decltype(&mqk_paged_select_workspace_size) paged_select_size = nullptr;
} g_lib;

PyObject* g_workspaces = nullptr;  // mqk._native._workspaces: {(device index, stream): uint8 tensor}
PyObject* g_raw_stream = nullptr;  // torch's raw current-stream accessor
PyObject* g_parameter = nullptr;   // torch.nn.Parameter
PyObject* g_capturing = nullptr;   // mqk._native.capturing: is the current stream being captured?
bool g_bound = false;

constexpr float kEps = 1e-6f;  // the op's fixed QK-Norm epsilon

// A tensor argument of an ordinary call: exactly torch.Tensor or Parameter, dense
// strided on the GPU, and no key but the ones a plain (or autograd) tensor carries.
const at::Tensor* plain(PyObject* o) {
  PyTypeObject* t = Py_TYPE(o);
  if (reinterpret_cast<PyObject*>(t) != THPVariableClass && reinterpret_cast<PyObject*>(t) != g_parameter) return nullptr;
  const at::Tensor& v = THPVariable_Unpack(o);
  static const c10::DispatchKeySet allowed =
      c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView,
                            c10::DispatchKey::AutocastCUDA});
  if (!v.defined() || v.layout() != c10::kStrided || !v.is_cuda() || !allowed.has_all(v.key_set()))
    return nullptr;
  return &v;
}

struct Call {
  c10::DeviceIndex dev = -1;
  bool ok = true;

  // An operand read through 16-byte loads: on the call's device, of type `type`,
  // contiguous and aligned.
  const at::Tensor* operand(PyObject* o, at::ScalarType type) {
    const at::Tensor* t = ok ? plain(o) : nullptr;
    if (!t || t->scalar_type() != type || !t->is_contiguous() || (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) != 0 ||
        (dev >= 0 && t->get_device() != dev)) {
      ok = false;
      return nullptr;
    }
    dev = t->get_device();
    return t;
  }
  // Numbers that are read one by one: contiguous int32, aligned as such.
  const at::Tensor* numbers(PyObject* o) {
    const at::Tensor* t = ok ? plain(o) : nullptr;
    if (!t || t->scalar_type() != at::kInt || !t->is_contiguous() || (dev >= 0 && t->get_device() != dev)) {
      ok = false;
      return nullptr;
    }
    dev = t->get_device();
    return t;
  }
  // ... or None (null); int32 tensors of n entries
  const int32_t* ints(PyObject* o, int64_t n) {
    if (o == Py_None) return nullptr;
    const at::Tensor* t = operand(o, at::kInt);
    if (ok && t->numel() != n) ok = false;
    return ok ? t->data_ptr<int32_t>() : nullptr;
  }
};

// Without the GIL while it lives.  Nothing in its scope touches a Python object.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

template <class T>
const T* ptr(const at::Tensor* t) {
  return static_cast<const T*>(t->data_ptr());
}

bool current_device_is(c10::DeviceIndex dev) {
  static const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
  return guard.getDevice().index() == dev;
}

bool modes_off() {
  return !at::impl::torch_function_mode_enabled() && !c10::impl::TorchDispatchModeTLS::any_modes_set();
}

// The raw current stream of device dev, as a Python int (new reference).
PyObject* stream_of(c10::DeviceIndex dev) {
  PyObject* index = PyLong_FromLong(dev);
  if (!index) return nullptr;
  PyObject* s = PyObject_CallOneArg(g_raw_stream, index);
  Py_DECREF(index);
  return s;
}

// The workspace of (dev, stream) if it holds n bytes; none needed for n == 0.  False:
// absent or too small (Python makes or grows it).
struct Workspace {
  at::Tensor buf;  // (held: another thread may replace it while the GIL is released)
  void* ptr = nullptr;
  size_t bytes = 0;
};
bool workspace(c10::DeviceIndex dev, PyObject* stream, size_t n, Workspace* ws) {
  if (n == 0) return true;
  PyObject* key = Py_BuildValue("(iO)", int(dev), stream);
  if (!key) {
    PyErr_Clear();
    return false;
  }
  PyObject* buf = PyDict_GetItem(g_workspaces, key);  // (borrowed)
  Py_DECREF(key);
  if (!buf || !THPVariable_Check(buf)) return false;
  const at::Tensor& t = THPVariable_Unpack(buf);
  if (size_t(t.numel()) < n) return false;
  ws->buf = t;
  ws->ptr = t.data_ptr();
  ws->bytes = size_t(t.numel());
  return true;
}

// Whether the current stream is being captured (also when that cannot be told).
bool capturing() {
  PyObject* r = PyObject_CallNoArgs(g_capturing);
  if (!r) {
    PyErr_Clear();
    return true;
  }
  const bool yes = r != Py_False;
  Py_DECREF(r);
  return yes;
}

// head_dim 64 and 128 (128-column blocks of whole heads) are taken here; other sizes in Python.
bool blocks_of(int64_t D, int64_t hq, int64_t hkv, int* bq, int* bkv) {
  if (D != 128 && D != 64) return false;
  if (hq < 1 || hkv < 1 || hq > 1 << 20 || hkv > 1 << 20) return false;
  *bq = int(hq * D / 128);
  *bkv = int(hkv * D / 128);
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, c10::DeviceIndex dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::DeviceType::CUDA, dev)));
}

PyObject* wrap3(at::Tensor q, at::Tensor k, at::Tensor v) {
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  at::Tensor* t[3] = {&q, &k, &v};
  for (int i = 0; i < 3; ++i) {
    PyObject* o;
    if (t[i]->defined()) {
      o = THPVariable_Wrap(*t[i]);
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    if (!o) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i, o);
  }
  return out;
}

// Norm weights and RoPE tables shared by the fronts: gamma [D], cos / sin [rows, D].
struct Rope {
  const at::Tensor *gq, *gk, *cos, *sin;
  int64_t D = 0, rows = 0;
  bool read(Call& c, PyObject* const* a, at::ScalarType type) {
    gq = c.operand(a[0], type);
    gk = c.operand(a[1], type);
    cos = c.operand(a[2], type);
    sin = c.operand(a[3], type);
    if (!c.ok || gq->dim() != 1 || gk->dim() != 1 || cos->dim() != 2 || sin->dim() != 2) return false;
    D = gq->size(0);
    rows = cos->size(0);
    return gk->size(0) == D && cos->size(1) == D && sin->size(1) == D && sin->size(0) == rows && rows >= 1;
  }
};

// fused(x, w_q, w_k, w_v, q_norm_w, k_norm_w, cos, sin, positions)
PyObject* fused(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !g_bound || !modes_off()) return none();
  const at::Tensor* x0 = plain(a[0]);
  if (!x0) return none();
  const at::ScalarType type = x0->scalar_type();
  if (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat) return none();
  Call c;
  const at::Tensor* x = c.operand(a[0], type);
  const at::Tensor* w[3];
  for (int i = 0; i < 3; ++i) w[i] = c.operand(a[1 + i], type);
  Rope r;
  if (!c.ok || !r.read(c, a + 4, type) || x->dim() != 3) return none();
  const int64_t B = x->size(0), S = x->size(1), H = x->size(2), T = B * S, D = r.D;
  for (int i = 0; i < 3; ++i)
    if (w[i]->dim() != 2 || w[i]->size(1) != H) return none();
  const int64_t hq = w[0]->size(0) / D, hkv = w[1]->size(0) / D;
  int bq, bkv;
  if (T == 0 || !blocks_of(D, hq, hkv, &bq, &bkv) || w[0]->size(0) != hq * D || w[1]->size(0) != hkv * D ||
      w[2]->size(0) != hkv * D)
    return none();
  const int32_t* pos = c.ints(a[8], T);
  if (!c.ok || !current_device_is(c.dev)) return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  size_t need = 0;
  if (type == at::kBFloat16) need = g_lib.size(T, bq, bkv, H);
  else if (type == at::kHalf) need = g_lib.f16_size(T, int(hq), int(hkv), H, int(D));
  if (type == at::kHalf && need > 0 && capturing()) {  // (a workspace of the graph's own: Python)
    Py_DECREF(stream);
    return none();
  }
  Workspace ws;
  const bool have = workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const void* in[8] = {x->data_ptr(),    w[0]->data_ptr(), w[1]->data_ptr(),  w[2]->data_ptr(),
                       r.gq->data_ptr(), r.gk->data_ptr(), r.cos->data_ptr(), r.sin->data_ptr()};
  at::Tensor q, k, v;
  int st;
  {
    Unlocked unlocked;
    q = fresh({B, S, hq, D}, type, c.dev);
    k = fresh({B, S, hkv, D}, type, c.dev);
    v = fresh({B, S, hkv, D}, type, c.dev);
    if (type == at::kFloat) {
      auto p = [&](int i) { return static_cast<const float*>(in[i]); };
      st = g_lib.f32(p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), pos, T, S, H, int(hq), int(hkv), int(D), r.rows, kEps,
                     static_cast<float*>(q.data_ptr()), static_cast<float*>(k.data_ptr()),
                     static_cast<float*>(v.data_ptr()), hs);
    } else {
      auto p = [&](int i) { return static_cast<const uint16_t*>(in[i]); };
      auto o = [](at::Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); };
      const auto fn = type == at::kHalf ? g_lib.f16 : g_lib.bf16;
      st = fn(p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), pos, T, S, H, int(hq), int(hkv), int(D), r.rows, kEps, o(q),
              o(k), o(v), ws.ptr, ws.bytes, hs);
    }
  }
  if (st != 0) return PyLong_FromLong(st);
  return wrap3(std::move(q), std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// The optional features: a = (positions, cu_seqlens, seq_pos0, input_norm_w, input_eps,
// k_cache, v_cache, block_table, kv_seq, kv_pos, return_kv).
struct Ext {
  mqk_fused_ext ext{};
  mqk_paged_kv kv{};
  const int32_t* pos = nullptr;
  bool return_kv = true;
  bool read(Call& c, PyObject* const* a, int64_t T, int64_t H, int64_t hkv, int64_t D) {
    pos = c.ints(a[0], T);
    if (a[1] != Py_None) {
      if (a[0] != Py_None) return false;
      const at::Tensor* cu = c.operand(a[1], at::kInt);
      if (!c.ok || cu->dim() != 1 || cu->numel() < 2) return false;
      ext.cu_seqlens = cu->data_ptr<int32_t>();
      ext.n_seqs = cu->numel() - 1;
      ext.seq_pos0 = c.ints(a[2], ext.n_seqs);
    } else if (a[2] != Py_None) {
      return false;
    }
    if (a[3] != Py_None) {
      const at::Tensor* g = c.operand(a[3], at::kBFloat16);
      if (!c.ok || g->dim() != 1 || g->size(0) != H || !PyFloat_CheckExact(a[4])) return false;
      ext.in_gamma = static_cast<const uint16_t*>(g->data_ptr());
      ext.in_eps = float(PyFloat_AS_DOUBLE(a[4]));
    }
    const bool cache = a[5] != Py_None;
    if (cache != (a[6] != Py_None) || cache != (a[7] != Py_None)) return false;
    if (!cache && (a[8] != Py_None || a[9] != Py_None)) return false;
    if (cache) {
      const at::Tensor* kc = c.operand(a[5], at::kBFloat16);
      const at::Tensor* vc = c.operand(a[6], at::kBFloat16);
      const at::Tensor* bt = c.operand(a[7], at::kInt);
      if (!c.ok || kc->dim() != 4 || kc->size(2) != hkv || kc->size(3) != D || vc->sizes() != kc->sizes() || bt->dim() != 2)
        return false;
      if (a[0] != Py_None && (a[8] == Py_None || a[9] == Py_None)) return false;
      kv.kv_seq = c.ints(a[8], T);
      kv.kv_pos = c.ints(a[9], T);
      kv.k_cache = static_cast<uint16_t*>(kc->data_ptr());
      kv.v_cache = static_cast<uint16_t*>(vc->data_ptr());
      kv.block_table = bt->data_ptr<int32_t>();
      kv.bt_rows = bt->size(0);
      kv.bt_cols = bt->size(1);
      kv.num_blocks = kc->size(0);
      kv.block_size = int32_t(kc->size(1));
      ext.kv = &kv;
    }
    if (!PyBool_Check(a[10])) return false;
    return_kv = a[10] == Py_True;
    return c.ok && (return_kv || cache);
  }
};

// x [B, S, hidden], or [T, hidden] with cu_seqlens: leading output dims and S.
bool lead_shape(const at::Tensor& x, bool varlen, int64_t* lead, int* n_lead, int64_t* S) {
  if (x.dim() == 3) {
    lead[0] = x.size(0);
    lead[1] = x.size(1);
    *n_lead = 2;
    *S = x.size(1);
    return true;
  }
  if (x.dim() == 2 && varlen) {
    lead[0] = x.size(0);
    *n_lead = 1;
    *S = x.size(0);
    return true;
  }
  return false;
}

// Outputs [*lead, heads, D] in bf16 (k and v undefined without return_kv).
struct Outputs {
  at::Tensor q, k, v;
  void make(const int64_t* lead, int n_lead, int64_t hq, int64_t hkv, int64_t D, bool kv, c10::DeviceIndex dev) {
    int64_t s[4] = {lead[0], lead[1], 0, 0};
    auto one = [&](int64_t h) {
      s[n_lead] = h;
      s[n_lead + 1] = D;
      return fresh(at::IntArrayRef(s, size_t(n_lead) + 2), at::kBFloat16, dev);
    };
    q = one(hq);
    if (kv) {
      k = one(hkv);
      v = one(hkv);
    }
  }
  static uint16_t* ptr(const at::Tensor& t) { return t.defined() ? static_cast<uint16_t*>(t.data_ptr()) : nullptr; }
};

// ex(x, w_q, w_k, w_v, q_norm_w, k_norm_w, cos, sin, <Ext's eleven>)
PyObject* fused_ex(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 19 || !g_bound || !modes_off()) return none();
  Call c;
  const at::Tensor* x = c.operand(a[0], at::kBFloat16);
  const at::Tensor* w[3];
  for (int i = 0; i < 3; ++i) w[i] = c.operand(a[1 + i], at::kBFloat16);
  Rope r;
  int64_t lead[2] = {0, 0}, S = 0;
  int n_lead = 0;
  if (!c.ok || !r.read(c, a + 4, at::kBFloat16) || !lead_shape(*x, a[9] != Py_None, lead, &n_lead, &S)) return none();
  const int64_t H = x->size(-1), D = r.D;
  for (int i = 0; i < 3; ++i)
    if (w[i]->dim() != 2 || w[i]->size(1) != H) return none();
  const int64_t hq = w[0]->size(0) / D, hkv = w[1]->size(0) / D, T = H > 0 ? x->numel() / H : 0;
  int bq, bkv;
  if (T == 0 || !blocks_of(D, hq, hkv, &bq, &bkv) || w[0]->size(0) != hq * D || w[1]->size(0) != hkv * D ||
      w[2]->size(0) != hkv * D)
    return none();
  Ext e;
  if (!e.read(c, a + 8, T, H, hkv, D) || !current_device_is(c.dev)) return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, g_lib.ex_size(T, bq, bkv, H, &e.ext), &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const uint16_t* in[8] = {ptr<uint16_t>(x),    ptr<uint16_t>(w[0]), ptr<uint16_t>(w[1]),  ptr<uint16_t>(w[2]),
                           ptr<uint16_t>(r.gq), ptr<uint16_t>(r.gk), ptr<uint16_t>(r.cos), ptr<uint16_t>(r.sin)};
  Outputs o;
  int st;
  {
    Unlocked unlocked;
    o.make(lead, n_lead, hq, hkv, D, e.return_kv, c.dev);
    st = g_lib.ex(in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7], e.pos, T, S, H, int(hq), int(hkv), int(D), r.rows,
                  kEps, o.ptr(o.q), o.ptr(o.k), o.ptr(o.v), &e.ext, ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return wrap3(std::move(o.q), std::move(o.k), std::move(o.v));
  END_HANDLE_TH_ERRORS
}

// One projection's (qweight, scales, qzeros) for K inputs and group size g.
struct Int4 {
  const at::Tensor *qw, *sc, *qz;
  int64_t N = 0;
  int scale_type = 0;
  bool read(Call& c, PyObject* const* a, int64_t K, int64_t g) {
    qw = c.operand(a[0], at::kInt);
    qz = c.operand(a[2], at::kInt);
    if (!c.ok) return false;
    const at::Tensor* s0 = plain(a[1]);
    if (!s0 || (s0->scalar_type() != at::kBFloat16 && s0->scalar_type() != at::kHalf)) return false;
    scale_type = s0->scalar_type() == at::kHalf ? MQK_SCALE_FP16 : MQK_SCALE_BF16;
    sc = c.operand(a[1], s0->scalar_type());
    if (!c.ok || qw->dim() != 2 || sc->dim() != 2 || qz->dim() != 2) return false;
    N = qw->size(1);
    return N > 0 && N % 8 == 0 && qw->size(0) == K / 8 && sc->size(0) == K / g && sc->size(1) == N && qz->size(0) == K / g &&
           qz->size(1) == N / 8;
  }
};

bool group_of(PyObject* o, int64_t K, int64_t* g) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *g = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *g > 0 && *g <= 1 << 24 && K % *g == 0 && K % 8 == 0;
}

// ex_w4(x, 9 int4 tensors, q_norm_w, k_norm_w, cos, sin, <Ext's eleven>, group_size)
PyObject* fused_ex_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 26 || !g_bound || !modes_off()) return none();
  Call c;
  const at::Tensor* x = c.operand(a[0], at::kBFloat16);
  int64_t lead[2] = {0, 0}, S = 0, g = 0;
  int n_lead = 0;
  if (!c.ok || !lead_shape(*x, a[15] != Py_None, lead, &n_lead, &S)) return none();
  const int64_t H = x->size(-1), T = H > 0 ? x->numel() / H : 0;
  if (T == 0 || !group_of(a[25], H, &g)) return none();
  Int4 w[3];
  for (int i = 0; i < 3; ++i)
    if (!w[i].read(c, a + 1 + 3 * i, H, g)) return none();
  if (w[1].scale_type != w[0].scale_type || w[2].scale_type != w[0].scale_type) return none();
  Rope r;
  if (!r.read(c, a + 10, at::kBFloat16)) return none();
  const int64_t D = r.D, hq = w[0].N / D, hkv = w[1].N / D;
  int bq, bkv;
  if (!blocks_of(D, hq, hkv, &bq, &bkv) || w[0].N != hq * D || w[1].N != hkv * D || w[2].N != hkv * D) return none();
  Ext e;
  if (!e.read(c, a + 14, T, H, hkv, D) || !current_device_is(c.dev)) return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const size_t need = g_lib.w4_size(T, bq, bkv, H, &e.ext);
  // (a captured call that unpacks its weights has a workspace of the graph's own: Python)
  const bool own = need > g_lib.ex_size(T, bq, bkv, H, &e.ext) && capturing();
  const bool have = !own && workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const uint16_t* in[5] = {ptr<uint16_t>(x), ptr<uint16_t>(r.gq), ptr<uint16_t>(r.gk), ptr<uint16_t>(r.cos),
                           ptr<uint16_t>(r.sin)};
  const int32_t *qw[3], *qz[3];
  const void* sc[3];
  for (int i = 0; i < 3; ++i) {
    qw[i] = ptr<int32_t>(w[i].qw);
    sc[i] = w[i].sc->data_ptr();
    qz[i] = ptr<int32_t>(w[i].qz);
  }
  Outputs o;
  int st;
  {
    Unlocked unlocked;
    o.make(lead, n_lead, hq, hkv, D, e.return_kv, c.dev);
    st = g_lib.ex_w4(in[0], qw[0], sc[0], qz[0], qw[1], sc[1], qz[1], qw[2], sc[2], qz[2], int(g), w[0].scale_type, in[1],
                     in[2], in[3], in[4], e.pos, T, S, H, int(hq), int(hkv), int(D), r.rows, kEps, o.ptr(o.q), o.ptr(o.k),
                     o.ptr(o.v), &e.ext, ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return wrap3(std::move(o.q), std::move(o.k), std::move(o.v));
  END_HANDLE_TH_ERRORS
}

// gemm(x [M, K], qweight, scales, qzeros, group_size)
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !g_bound || !modes_off()) return none();
  Call c;
  const at::Tensor* x = c.operand(a[0], at::kBFloat16);
  int64_t g = 0;
  if (!c.ok || x->dim() != 2) return none();
  const int64_t M = x->size(0), K = x->size(1);
  Int4 w;
  if (M == 0 || !group_of(a[4], K, &g) || !w.read(c, a + 1, K, g) || !current_device_is(c.dev)) return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, g_lib.gemm_size(M, K, w.N), &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const uint16_t* xp = ptr<uint16_t>(x);
  const int32_t *qw = ptr<int32_t>(w.qw), *qz = ptr<int32_t>(w.qz);
  const void* sc = w.sc->data_ptr();
  at::Tensor out;
  int st;
  {
    Unlocked unlocked;
    out = fresh({M, w.N}, at::kBFloat16, c.dev);
    st = g_lib.gemm(xp, qw, sc, qz, M, K, w.N, int(g), w.scale_type, static_cast<uint16_t*>(out.data_ptr()), ws.ptr,
                    ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// --- attention -----------------------------------------------------------------------

// Heads of tokens that the kernels read where they are: [T, H, D] or [B, S, H, D] of type
// `type`, dense along the head, token and head strides of whole 16-byte chunks.
struct Heads {
  const at::Tensor* t = nullptr;
  int64_t T = 0, H = 0, D = 0;
  mqk_attn_tensor desc{};
  bool read(Call& c, PyObject* o, at::ScalarType type) {
    t = plain(o);
    if (!t || t->scalar_type() != type || (c.dev >= 0 && t->get_device() != c.dev)) return false;
    const int64_t d = t->dim();
    if (d != 3 && d != 4) return false;
    const int64_t step = 16 / int64_t(t->element_size());
    H = t->size(d - 2);
    D = t->size(d - 1);
    T = d == 4 ? t->size(0) * t->size(1) : t->size(0);
    if (T == 0 || H == 0 || D == 0) return false;
    desc.token_stride = t->stride(d - 3);
    desc.head_stride = t->stride(d - 2);
    if (d == 4 && t->size(0) > 1 && t->stride(0) != t->size(1) * t->stride(1)) return false;
    if (t->stride(d - 1) != 1 || desc.token_stride < 0 || desc.head_stride < 0 || desc.token_stride % step != 0 ||
        desc.head_stride % step != 0)
      return false;
    desc.data = t->data_ptr();
    if ((reinterpret_cast<uintptr_t>(desc.data) & 15u) != 0) return false;
    c.dev = t->get_device();
    return true;
  }
};

// The bytes between a tensor's first element and its last one, and whether two meet.
bool meet(const at::Tensor& x, const at::Tensor& y) {
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + uintptr_t(last + 1) * t.element_size();
  };
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.data_ptr()), b = reinterpret_cast<uintptr_t>(y.data_ptr());
  return a < end(y) && b < end(x);
}

int dtype_of(at::ScalarType type) {
  return type == at::kBFloat16 ? MQK_BF16 : type == at::kHalf ? MQK_F16 : type == at::kFloat ? MQK_F32 : -1;
}

// None: D ** -0.5; an ordinary positive float; else false.
bool scale_of(PyObject* o, int64_t D, float* scale) {
  if (o == Py_None) {
    *scale = float(1.0 / std::sqrt(double(D)));
    return true;
  }
  if (!PyFloat_CheckExact(o)) return false;
  const double v = PyFloat_AS_DOUBLE(o);
  *scale = float(v);
  return v > 0.0 && v <= 1e30;
}

// attn_prefill(q, k, v, cu_seqlens, cu_seqlens_k, scale, out)
PyObject* attn_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_bound || !modes_off()) return none();
  const at::Tensor* q0 = plain(a[0]);
  if (!q0) return none();
  const at::ScalarType type = q0->scalar_type();
  const int dtype = dtype_of(type);
  Call c;
  Heads q, k, v;
  if (dtype < 0 || !q.read(c, a[0], type) || !k.read(c, a[1], type) || !v.read(c, a[2], type)) return none();
  const int64_t D = q.D;
  if (k.T != v.T || k.H != v.H || k.D != D || v.D != D || q.H % k.H != 0 || D % 8 != 0 || D > 256 ||
      q.t->dim() != k.t->dim() || k.t->sizes() != v.t->sizes())
    return none();
  float scale;
  if (!scale_of(a[5], D, &scale)) return none();
  const int32_t *cu = nullptr, *cu_k = nullptr;
  int64_t seqs = 1;
  if (a[3] != Py_None) {
    const at::Tensor* t = c.operand(a[3], at::kInt);
    if (!c.ok || t->dim() != 1 || t->numel() < 2) return none();
    cu = t->data_ptr<int32_t>();
    seqs = t->numel() - 1;
    if (a[4] != Py_None) {
      const at::Tensor* u = c.operand(a[4], at::kInt);
      if (!c.ok || u->dim() != 1 || u->numel() != seqs + 1) return none();
      cu_k = u->data_ptr<int32_t>();
    } else if (q.T != k.T) {
      return none();
    }
  } else {
    if (a[4] != Py_None) return none();
    if (q.t->dim() == 4) {
      seqs = q.t->size(0);
      if (k.t->size(0) != seqs) return none();
    }
  }
  if (!current_device_is(c.dev)) return none();
  const size_t need = g_lib.attn_size(dtype, q.T, k.T, seqs, cu != nullptr, int(q.H), int(k.H), int(D));
  if (need > 0 && capturing()) return none();  // (a workspace of the graph's own: Python)
  const bool fill = a[6] == Py_None;
  at::Tensor out;
  if (!fill) {
    const at::Tensor* t = c.operand(a[6], type);
    if (!c.ok || t->sizes() != q.t->sizes() || meet(*t, *q.t) || meet(*t, *k.t) || meet(*t, *v.t)) return none();
    out = *t;
  }
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const c10::DimVector shape(q.t->sizes().begin(), q.t->sizes().end());
  int st;
  {
    Unlocked unlocked;
    if (fill) out = fresh(shape, type, c.dev);
    st = g_lib.attn(&q.desc, &k.desc, &v.desc, dtype, cu, cu_k, q.T, k.T, seqs, int(q.H), int(k.H), int(D), scale, fill,
                    out.data_ptr(), ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A 4-bit cache [num_blocks, Hkv, 9 D], its block table and the sequences' lengths.
struct Cache4 {
  const at::Tensor* t = nullptr;
  mqk_kv4_cache desc{};
  const int32_t* lens = nullptr;
  at::ScalarType type{};
  bool read(Call& c, PyObject* cache, PyObject* table, PyObject* seq_lens) {
    t = plain(cache);
    if (!t) return false;
    type = t->scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return false;
    t = c.operand(cache, type);
    const at::Tensor* bt = c.operand(table, at::kInt);
    const at::Tensor* n = c.operand(seq_lens, at::kInt);
    if (!c.ok || t->dim() != 3 || (t->size(2) != 9 * 64 && t->size(2) != 9 * 128) || t->size(0) < 1 || t->size(1) < 1 ||
        bt->dim() != 2 || bt->size(0) < 1 || bt->size(1) < 1 || n->dim() != 1 || n->numel() != bt->size(0))
      return false;
    desc.cache = t->data_ptr();
    desc.block_table = bt->data_ptr<int32_t>();
    desc.num_blocks = t->size(0);
    desc.bt_cols = bt->size(1);
    desc.n_seqs = bt->size(0);
    desc.dtype = dtype_of(type);
    desc.Hkv = int(t->size(1));
    desc.D = int(t->size(2) / 9);
    lens = n->data_ptr<int32_t>();
    return true;
  }
  // [num_blocks, Hkv, 16] float32, or None where that is allowed
  const at::Tensor* marks = nullptr;
  bool scores(Call& c, PyObject* o, bool need, float** to) {
    *to = nullptr;
    if (o == Py_None) return !need;
    marks = c.operand(o, at::kFloat);
    if (!c.ok || marks->dim() != 3 || marks->size(0) != t->size(0) || marks->size(1) != t->size(1) || marks->size(2) != 16)
      return false;
    *to = marks->data_ptr<float>();
    return true;
  }
  // offsets [n_seqs + 1], or None for equally many tokens a sequence
  bool offsets(Call& c, PyObject* o, int64_t T, const int32_t** to) const {
    *to = nullptr;
    if (o == Py_None) return T % desc.n_seqs == 0;
    const at::Tensor* u = c.operand(o, at::kInt);
    if (!c.ok || u->dim() != 1 || u->numel() != desc.n_seqs + 1) return false;
    *to = u->data_ptr<int32_t>();
    return true;
  }
};

// kv4_write(k, v, cache, block_table, seq_lens, cu_seqlens, scores)
PyObject* kv4_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_bound || !modes_off()) return none();
  Call c;
  Cache4 cache;
  Heads k, v;
  const int32_t* cu;
  float* scores;
  if (!cache.read(c, a[2], a[3], a[4]) || !k.read(c, a[0], cache.type) || !v.read(c, a[1], cache.type) ||
      k.t->sizes() != v.t->sizes() || k.H != cache.desc.Hkv || k.D != cache.desc.D ||
      !cache.offsets(c, a[5], k.T, &cu) || !cache.scores(c, a[6], false, &scores) || !current_device_is(c.dev))
    return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  int st;
  {
    Unlocked unlocked;
    st = g_lib.kv4_write(&k.desc, &v.desc, &cache.desc, cache.lens, cu, k.T, scores, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// An exact Python int (no bool) within [lo, hi].
bool int_of(PyObject* o, int64_t lo, int64_t hi, int64_t* to) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  *to = v;
  return overflow == 0 && v >= lo && v <= hi;
}

PyObject* wrap2(at::Tensor x, at::Tensor y) {
  PyObject* px = THPVariable_Wrap(std::move(x));
  PyObject* py = px ? THPVariable_Wrap(std::move(y)) : nullptr;
  PyObject* out = py ? PyTuple_Pack(2, px, py) : nullptr;
  Py_XDECREF(px);
  Py_XDECREF(py);
  return out;
}

// kv4_read(cache, block_table, seq_lens, n_tokens, cu_seqlens)
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !g_bound || !modes_off()) return none();
  Call c;
  Cache4 cache;
  int64_t T;
  const int32_t* cu;
  if (!int_of(a[3], 1, 0x7FFF0000ll, &T) || !cache.read(c, a[0], a[1], a[2]) || !cache.offsets(c, a[4], T, &cu) ||
      !current_device_is(c.dev))
    return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  at::Tensor k, v;
  int st;
  {
    Unlocked unlocked;
    k = fresh({T, cache.desc.Hkv, cache.desc.D}, cache.type, c.dev);
    v = fresh({T, cache.desc.Hkv, cache.desc.D}, cache.type, c.dev);
    st = g_lib.kv4_read(&cache.desc, cache.lens, cu, T, k.data_ptr(), v.data_ptr(), hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return wrap2(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// kv4_attn(q, cache, block_table, seq_lens, scale, scores, out)
PyObject* kv4_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_bound || !modes_off()) return none();
  Call c;
  Cache4 cache;
  if (!cache.read(c, a[1], a[2], a[3])) return none();
  const at::Tensor* q = c.operand(a[0], cache.type);
  if (!c.ok || (q->dim() != 3 && q->dim() != 4) || q->numel() == 0) return none();
  const int64_t d = q->dim(), S = d == 4 ? q->size(1) : 1, hq = q->size(d - 2);
  float scale;
  float* scores;
  if (q->size(0) != cache.desc.n_seqs || q->size(d - 1) != cache.desc.D || hq % cache.desc.Hkv != 0 || hq > 1 << 20 ||
      !scale_of(a[4], cache.desc.D, &scale) || !cache.scores(c, a[5], false, &scores))
    return none();
  at::Tensor out;
  const bool make = a[6] == Py_None;
  if (!make) {
    const at::Tensor* t = c.operand(a[6], cache.type);
    if (!c.ok || t->sizes() != q->sizes() || meet(*t, *q) || meet(*t, *cache.t) ||
        (cache.marks && meet(*t, *cache.marks)))
      return none();
    out = *t;
  }
  if (!current_device_is(c.dev)) return none();
  const size_t need = g_lib.kv4_attn_size(&cache.desc, S, int(hq), scores != nullptr);
  if (need > 0 && capturing()) return none();  // (a workspace of the graph's own: Python)
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const void* qp = q->data_ptr();
  const c10::DimVector shape(q->sizes().begin(), q->sizes().end());
  int st;
  {
    Unlocked unlocked;
    if (make) out = fresh(shape, cache.type, c.dev);
    st = g_lib.kv4_attn(qp, &cache.desc, cache.lens, S, int(hq), scale, scores, out.data_ptr(), ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// kv4_evict(cache, scores, block_table, seq_lens, budget, recent)
PyObject* kv4_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !g_bound || !modes_off()) return none();
  Call c;
  Cache4 cache;
  int64_t budget, recent;
  float* scores;
  if (!cache.read(c, a[0], a[2], a[3]) || !cache.scores(c, a[1], true, &scores) || !int_of(a[4], 1, 1 << 24, &budget) ||
      !int_of(a[5], 0, budget, &recent) || !current_device_is(c.dev))
    return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  at::Tensor lens, kept;
  int st;
  {
    Unlocked unlocked;
    lens = fresh({cache.desc.n_seqs}, at::kInt, c.dev);
    kept = fresh({cache.desc.n_seqs, cache.desc.Hkv, budget}, at::kInt, c.dev);
    st = g_lib.kv4_evict(&cache.desc, scores, cache.lens, int(budget), int(recent), lens.data_ptr<int32_t>(),
                         kept.data_ptr<int32_t>(), hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return wrap2(std::move(lens), std::move(kept));
  END_HANDLE_TH_ERRORS
}

// A tensor of n numbers of its own in `whole`'s memory, from byte `at` on.
at::Tensor piece(const at::Tensor& whole, at::ScalarType type, int64_t at, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                          c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  t.unsafeGetTensorImpl()->set_storage_offset(at / int64_t(c10::elementSize(type)));
  return t;
}

// paged_tables(seq_lens, new_lens, block_table, free_pages, n_tokens, page, cursor)
PyObject* paged_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_bound || !modes_off()) return none();
  Call c;
  int64_t T, page;
  const at::Tensor* bt = c.numbers(a[2]);
  if (!c.ok || bt->dim() != 2 || bt->size(0) < 1 || bt->size(1) < 1 || !int_of(a[4], 0, 0x7FFF0000ll, &T) ||
      !int_of(a[5], 1, 1 << 20, &page))
    return none();
  const at::Tensor* in[4] = {};
  for (int i : {0, 1, 3}) {
    in[i] = c.numbers(a[i]);
    if (!c.ok || in[i]->dim() != 1 || in[i]->numel() == 0 || meet(*in[i], *bt)) return none();
  }
  const int64_t seqs = bt->size(0);
  if (in[0]->numel() != seqs || in[1]->numel() != seqs) return none();
  const int32_t* cursor = nullptr;
  if (a[6] != Py_None) {
    const at::Tensor* t = c.numbers(a[6]);
    if (!c.ok || t->dim() != 1 || t->numel() != 1 || meet(*t, *bt)) return none();
    cursor = t->data_ptr<int32_t>();
  }
  if (!current_device_is(c.dev)) return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  const int32_t *old = in[0]->data_ptr<int32_t>(), *add = in[1]->data_ptr<int32_t>(), *list = in[3]->data_ptr<int32_t>();
  const int64_t listed = in[3]->numel(), cols = bt->size(1);
  int32_t* table = bt->data_ptr<int32_t>();
  at::Tensor out[6];
  int st;
  {
    Unlocked unlocked;
    // six outputs in one allocation, 16-byte aligned: allocating each took as long as the kernel
    const int64_t sizes[6] = {seqs, seqs + 1, T, T, T, 1};
    int64_t at[6], bytes = 0;
    for (int i = 0; i < 6; ++i) {
      at[i] = bytes;
      bytes += (sizes[i] * (i == 4 ? 8 : 4) + 15) / 16 * 16;
    }
    const at::Tensor whole = fresh({bytes}, at::kByte, c.dev);
    for (int i = 0; i < 6; ++i) out[i] = piece(whole, i == 4 ? at::kLong : at::kInt, at[i], sizes[i]);
    auto p = [&](int i) { return out[i].data_ptr<int32_t>(); };
    st = g_lib.paged_tables(old, add, seqs, table, cols, list, listed, cursor, int(page), T, p(0), p(1), p(2), p(3),
                            out[4].data_ptr<int64_t>(), p(5), hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  PyObject* all = PyTuple_New(6);
  if (!all) return nullptr;
  for (int i = 0; i < 6; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(out[i]));
    if (!o) {
      Py_DECREF(all);
      return nullptr;
    }
    PyTuple_SET_ITEM(all, i, o);
  }
  return all;
  END_HANDLE_TH_ERRORS
}

// Paged caches [num_blocks, page, Hkv, D] (`v` may be left out), or bounds [num_blocks, Hkv, 2, D]
// of one, its block table and the sequences' lengths.
struct Paged {
  const at::Tensor *k = nullptr, *v = nullptr, *table = nullptr, *n = nullptr;
  mqk_paged_cache desc{};
  const int32_t* lens = nullptr;
  at::ScalarType type{};
  bool read(Call& c, PyObject* keys, PyObject* values, bool box, int64_t page, PyObject* bt, PyObject* seq_lens) {
    k = plain(keys);
    if (!k) return false;
    type = k->scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return false;
    k = c.operand(keys, type);
    if (values) v = c.operand(values, type);
    table = c.numbers(bt);
    n = c.numbers(seq_lens);
    if (!c.ok || k->dim() != 4 || k->numel() == 0 || (v && v->sizes() != k->sizes()) || table->dim() != 2 ||
        table->size(0) < 1 || table->size(1) < 1 || n->dim() != 1 || n->numel() != table->size(0) ||
        (box && k->size(2) != 2))
      return false;
    desc.k = k->data_ptr();
    desc.v = v ? v->data_ptr() : nullptr;
    desc.block_table = table->data_ptr<int32_t>();
    desc.num_blocks = k->size(0);
    desc.bt_cols = table->size(1);
    desc.n_seqs = table->size(0);
    desc.dtype = dtype_of(type);
    const int64_t heads = box ? k->size(1) : k->size(2);
    if (!box) page = k->size(1);
    if (page % 8 != 0 || page > 1 << 20 || heads > 4096 || k->size(3) % 8 != 0 || k->size(3) > 256) return false;
    desc.page = int(page);
    desc.Hkv = int(heads);
    desc.D = int(k->size(3));
    lens = n->data_ptr<int32_t>();
    return true;
  }
  // q's tokens, cut by offsets [n_seqs + 1] (None: equally many a sequence)
  const at::Tensor* offs = nullptr;
  bool queries(Call& c, Heads& q, PyObject* o, PyObject* cu, const int32_t** to) {
    if (!q.read(c, o, type) || q.D != desc.D || q.H % desc.Hkv != 0 || q.H > 1 << 16) return false;
    return offsets(c, cu, q.T, to) && (*to || q.t->dim() != 4 || q.t->size(0) == desc.n_seqs);
  }
  bool offsets(Call& c, PyObject* o, int64_t T, const int32_t** to) {
    *to = nullptr;
    if (o == Py_None) return T % desc.n_seqs == 0;
    offs = c.numbers(o);
    if (!c.ok || offs->dim() != 1 || offs->numel() != desc.n_seqs + 1) return false;
    *to = offs->data_ptr<int32_t>();
    return true;
  }
  // whether t lies over anything that is read
  bool over(const at::Tensor& t) const {
    for (const at::Tensor* x : {k, v, table, n, offs})
      if (x && meet(t, *x)) return true;
    return false;
  }
};

// q's shape without its last `drop` dimensions, then `more`.
c10::DimVector lead(const at::Tensor& q, int drop, std::initializer_list<int64_t> more) {
  c10::DimVector s(q.sizes().begin(), q.sizes().end() - drop);
  s.insert(s.end(), more.begin(), more.end());
  return s;
}

// paged_attn(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, pages, scale, out)
PyObject* paged_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !g_bound || !modes_off()) return none();
  Call c;
  Paged cache;
  Heads q;
  const int32_t *cu, *pages = nullptr;
  int64_t listed = 0;
  float scale;
  if (!cache.read(c, a[1], a[2], false, 0, a[3], a[4]) || !cache.queries(c, q, a[0], a[5], &cu) ||
      !scale_of(a[7], q.D, &scale))
    return none();
  const at::Tensor* list = nullptr;
  if (a[6] != Py_None) {
    list = c.numbers(a[6]);
    if (!c.ok || list->dim() != q.t->dim() || list->numel() == 0) return none();
    listed = list->size(-1);
    const c10::DimVector want = lead(*q.t, 2, {cache.desc.Hkv, listed});
    if (list->sizes() != c10::IntArrayRef(want)) return none();
    pages = list->data_ptr<int32_t>();
  }
  at::Tensor out;
  const bool make = a[8] == Py_None;
  if (!make) {
    const at::Tensor* t = c.operand(a[8], cache.type);
    if (!c.ok || t->sizes() != q.t->sizes() || meet(*t, *q.t) || cache.over(*t) || (list && meet(*t, *list))) return none();
    out = *t;
  }
  if (!current_device_is(c.dev)) return none();
  const size_t need = g_lib.paged_attn_size(&cache.desc, q.T, int(q.H), cu != nullptr, listed);
  if (need > 0 && capturing()) return none();  // (a workspace of the graph's own: Python)
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const c10::DimVector shape(q.t->sizes().begin(), q.t->sizes().end());
  int st;
  {
    Unlocked unlocked;
    if (make) out = fresh(shape, cache.type, c.dev);
    st = g_lib.paged_attn(&q.desc, &cache.desc, cache.lens, cu, q.T, int(q.H), scale, pages, listed, make, out.data_ptr(),
                          ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_bounds(k_cache, bounds, block_table, seq_lens, n_tokens, cu_seqlens)
PyObject* paged_bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !g_bound || !modes_off()) return none();
  Call c;
  Paged cache;
  int64_t T = -1;
  const int32_t* cu = nullptr;
  if (!cache.read(c, a[0], nullptr, false, 0, a[2], a[3])) return none();
  if (a[4] == Py_None) {
    if (a[5] != Py_None) return none();
  } else if (!int_of(a[4], 1, 0x7FFF0000ll, &T) || !cache.offsets(c, a[5], T, &cu)) {
    return none();
  }
  const at::Tensor* to = c.operand(a[1], cache.type);
  if (!c.ok || to->dim() != 4 || to->size(0) != cache.desc.num_blocks || to->size(1) != cache.desc.Hkv ||
      to->size(2) != 2 || to->size(3) != cache.desc.D || cache.over(*to) || !current_device_is(c.dev))
    return none();
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  void* dst = to->data_ptr();
  int st;
  {
    Unlocked unlocked;
    st = g_lib.paged_bounds(&cache.desc, cache.lens, cu, T, dst, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_select(q, bounds, block_table, seq_lens, page, n_pages, cu_seqlens, first, recent)
PyObject* paged_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !g_bound || !modes_off()) return none();
  Call c;
  Paged cache;
  Heads q;
  const int32_t* cu;
  int64_t page, take, first, recent;
  if (!int_of(a[4], 8, 1 << 20, &page) || !int_of(a[5], 1, 1 << 24, &take) || !int_of(a[7], 0, take - 1, &first) ||
      !int_of(a[8], 1, take - first, &recent) || !cache.read(c, a[1], nullptr, true, page, a[2], a[3]) ||
      !cache.queries(c, q, a[0], a[6], &cu) || !current_device_is(c.dev))
    return none();
  const void* box = cache.desc.k;
  cache.desc.k = nullptr;
  const size_t need = g_lib.paged_select_size(&cache.desc, q.T);
  if (need > 0 && capturing()) return none();  // (a workspace of the graph's own: Python)
  PyObject* stream = stream_of(c.dev);
  if (!stream) return nullptr;
  Workspace ws;
  const bool have = workspace(c.dev, stream, need, &ws);
  void* hs = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!have) return none();
  const c10::DimVector shape = lead(*q.t, 2, {cache.desc.Hkv, take});
  at::Tensor out;
  int st;
  {
    Unlocked unlocked;
    out = fresh(shape, at::kInt, c.dev);
    st = g_lib.paged_select(&q.desc, box, &cache.desc, cache.lens, cu, q.T, int(q.H), take, int(first), int(recent),
                            out.data_ptr<int32_t>(), ws.ptr, ws.bytes, hs);
  }
  if (st != 0) return PyLong_FromLong(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind(dlopen handle of libmqk.so, workspaces dict, raw-stream accessor, Parameter class,
// capture check)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5 || !PyDict_Check(a[1]) || !PyCallable_Check(a[2]) || !PyType_Check(a[3]) || !PyCallable_Check(a[4])) {
    PyErr_SetString(PyExc_TypeError, "bind(handle, workspaces, raw_stream, parameter_class, capturing)");
    return nullptr;
  }
  void* h = PyLong_AsVoidPtr(a[0]);
  if (!h && PyErr_Occurred()) return nullptr;
  bool all = true;
  auto get = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(h, name));
    all = all && fn;
  };
  get(g_lib.bf16, "mqk_fused_qkv_rope_bf16");
  get(g_lib.f32, "mqk_fused_qkv_rope_f32");
  get(g_lib.f16, "mqk_fused_qkv_rope_f16_ws");
  get(g_lib.f16_size, "mqk_fused_qkv_rope_f16_workspace_size");
  get(g_lib.size, "mqk_fused_qkv_rope_workspace_size");
  get(g_lib.ex_size, "mqk_fused_qkv_rope_ex_workspace_size");
  get(g_lib.w4_size, "mqk_fused_qkv_rope_w4a16_workspace_size");
  get(g_lib.ex, "mqk_fused_qkv_rope_ex_bf16");
  get(g_lib.ex_w4, "mqk_fused_qkv_rope_ex_w4a16");
  get(g_lib.gemm_size, "mqk_w4a16_gemm_workspace_size");
  get(g_lib.gemm, "mqk_w4a16_gemm_ex");
  get(g_lib.attn, "mqk_attn_prefill");
  get(g_lib.attn_size, "mqk_attn_prefill_workspace_size");
  get(g_lib.kv4_write, "mqk_kv4_write");
  get(g_lib.kv4_read, "mqk_kv4_read");
  get(g_lib.kv4_attn, "mqk_kv4_attn");
  get(g_lib.kv4_attn_size, "mqk_kv4_attn_workspace_size");
  get(g_lib.kv4_evict, "mqk_kv4_evict");
  get(g_lib.paged_tables, "mqk_paged_tables");
  get(g_lib.paged_attn, "mqk_paged_attn");
  get(g_lib.paged_attn_size, "mqk_paged_attn_workspace_size");
  get(g_lib.paged_bounds, "mqk_paged_bounds");
  get(g_lib.paged_select, "mqk_paged_select");
  get(g_lib.paged_select_size, "mqk_paged_select_workspace_size");
  if (!all) {
    PyErr_SetString(PyExc_RuntimeError, "libmqk.so lacks an entry point mqk._front calls");
    return nullptr;
  }
  for (int i = 1; i < 5; ++i) Py_INCREF(a[i]);
  g_workspaces = a[1];
  g_raw_stream = a[2];
  g_parameter = a[3];
  g_capturing = a[4];
  g_bound = true;
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f));
}

PyMethodDef g_methods[] = {
    {"bind", fast(bind), METH_FASTCALL, "bind(libmqk handle, workspaces, raw stream accessor, Parameter class, capture check)"},
    {"fused", fast(fused), METH_FASTCALL, "fused_qkv_rope of an ordinary call: (q, k, v), a status, or None"},
    {"fused_ex", fast(fused_ex), METH_FASTCALL, "fused_qkv_rope_ex of an ordinary call"},
    {"fused_ex_w4", fast(fused_ex_w4), METH_FASTCALL, "fused_qkv_rope_w4a16_ex of an ordinary call"},
    {"gemm", fast(gemm), METH_FASTCALL, "w4a16_gemm of an ordinary call: the output, a status, or None"},
    {"attn_prefill", fast(attn_prefill), METH_FASTCALL, "attn_prefill of an ordinary call: the output, a status, or None"},
    {"kv4_write", fast(kv4_write), METH_FASTCALL, "kv4_write of an ordinary call: True, a status, or None"},
    {"kv4_read", fast(kv4_read), METH_FASTCALL, "kv4_read of an ordinary call: (k, v), a status, or None"},
    {"kv4_attn", fast(kv4_attn), METH_FASTCALL, "kv4_attn of an ordinary call: the output, a status, or None"},
    {"kv4_evict", fast(kv4_evict), METH_FASTCALL, "kv4_evict of an ordinary call: (new_lens, kept), a status, or None"},
    {"paged_tables", fast(paged_tables), METH_FASTCALL, "paged_tables of an ordinary call: its six outputs, a status, or None"},
    {"paged_attn", fast(paged_attn), METH_FASTCALL, "paged_attn of an ordinary call: the output, a status, or None"},
    {"paged_bounds", fast(paged_bounds), METH_FASTCALL, "paged_bounds of an ordinary call: True, a status, or None"},
    {"paged_select", fast(paged_select), METH_FASTCALL, "paged_select of an ordinary call: the output, a status, or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front() { return PyModule_Create(&g_module); }
