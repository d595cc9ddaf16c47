// The plain attention call (one band over one sequence or pack, no ring) from Python to the launches
// without Python in between: checks, output allocation, parameter block, launch, and the autograd node.
//
// Small calls are bounded by the host.  With the same steps in Python (ring_swa/sliding_window.py,
// ops/band_attn.py) one forward took 20 us for a kernel of 12, and forward + backward of 1024 tokens, 4
// heads, 143 us for 45 us of kernels: building the parameter block through ctypes, the Python autograd
// function, and the hand-over of the interpreter lock to the autograd thread.  Here they take 10.5 and 72.
//
// band_attn() only takes what it can answer: plain tensors on one GPU, in the layout and types the
// kernels take, with no tracing, transform or mode active that has to see the call.  For everything
// else it returns None and the Python route runs, which refuses or handles it.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <optional>

#include "../../include/rswa.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Entry points of the library that ring_swa._lib opened (bind)
struct {
  int (*fwd)(const rswa_attn_params*, void*) = nullptr;
  int (*bwd)(const rswa_attn_params*, void*) = nullptr;
  uint64_t (*bwd_bytes)(const rswa_attn_params*) = nullptr;
  PyObject* raise = nullptr;         // raises what a non-zero status means
  PyObject* python_bwd = nullptr;    // backward in Python, for the environment's switches and what has to be refused
} lib;

// With the interpreter lock only: Python changes the environment under it, and a getenv beside such a change
// may read the array that it has just freed.
bool env_switches() {
  TORCH_INTERNAL_ASSERT(PyGILState_Check());
  for (const char* name : {"RSWA_ADDRESSING", "RSWA_DKDV_FORM", "RSWA_DS_HANDOFF"}) {
    const char* v = std::getenv(name);
    if (v && *v) return true;
  }
  return false;
}

// Is anything active in this thread that has to see the operations of the call?
bool observed() {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  return tls.included_.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                                    c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                                    c10::DispatchKey::FuncTorchDynamicLayerBackMode,
                                                    c10::DispatchKey::Functionalize})) ||
         c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
         torch::jit::tracer::isTracing();
}

// A dense tensor on the GPU and nothing else: no subclass, wrapper, lazy conjugate or tangent
bool plain(const Tensor& t) {
  static const c10::DispatchKeySet known =
      c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA,
                           c10::DispatchKey::ADInplaceOrView});
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && (t.key_set().raw_repr() & ~known.raw_repr()) == 0 &&
         !t._fw_grad(0).defined();
}

// Queries, keys and values that the kernels take as they are?
bool fits(const Tensor& q, const Tensor& k, const Tensor& v, bool packed) {
  const int nd = packed ? 3 : 4;
  if (!plain(q) || !plain(k) || !plain(v)) return false;
  const auto type = q.scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || k.scalar_type() != type || v.scalar_type() != type) return false;
  if (q.dim() != nd || k.dim() != nd || v.dim() != nd || k.sizes() != v.sizes()) return false;
  if (q.device() != k.device() || q.device() != v.device()) return false;
  if (q.numel() == 0 || k.numel() == 0) return false;
  for (int d = 0; d < nd - 2; d++)
    if (q.size(d) != k.size(d) || q.size(d) >= (1 << 28)) return false;
  if (q.size(-1) != k.size(-1) || q.size(-2) % k.size(-2) != 0 || q.size(-2) >= (1 << 28)) return false;
  return q.stride(-1) == 1 && k.stride(-1) == 1 && v.stride(-1) == 1;
}

// ... and another tensor of q's type, shape and device
bool like(const Tensor& t, const Tensor& q) {
  return plain(t) && t.scalar_type() == q.scalar_type() && t.sizes() == q.sizes() && t.device() == q.device() &&
         t.stride(-1) == 1;
}

bool lse_of(const Tensor& t, const Tensor& q, bool packed) {
  if (!plain(t) || t.scalar_type() != at::kFloat || t.device() != q.device()) return false;
  return packed ? t.sizes().equals({q.size(1), q.size(0)}) : t.sizes().equals({q.size(0), q.size(2), q.size(1)});
}

struct Call {
  bool packed = false;
  int32_t window = 0, num_sink = 0;
  float scale = 0;
  Tensor cu;  // cu_seqlens of a pack; undefined: dense
};

void strides3(int64_t* dst, const Tensor& t, bool packed) {
  if (packed) {
    dst[0] = 0;
    dst[1] = t.stride(0);
    dst[2] = t.stride(1);
  } else {
    for (int i = 0; i < 3; i++) dst[i] = t.stride(i);
  }
}

// (as ring_swa/ops/band_attn.py:_params; causal, bottom-right aligned, one key range)
rswa_attn_params params(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                        const Tensor& lse) {
  rswa_attn_params p{};
  p.dtype = q.scalar_type() == at::kBFloat16 ? RSWA_BF16 : RSWA_F16;
  p.head_dim = (int32_t)q.size(-1);
  p.heads_q = (int32_t)q.size(-2);
  p.heads_kv = (int32_t)k.size(-2);
  if (c.packed) {
    p.batch = (int32_t)c.cu.numel() - 1;
    p.total_q = p.total_k = q.size(0);
    p.seqlen_q = p.seqlen_k = (int32_t)q.size(0);
    p.cu_seqlens_q = p.cu_seqlens_k = (const int32_t*)c.cu.data_ptr();
  } else {
    p.batch = (int32_t)q.size(0);
    p.seqlen_q = p.seqlen_k = (int32_t)q.size(1);
  }
  p.softmax_scale = c.scale;
  p.window_left = c.window;
  p.causal = 1;
  p.num_sink = c.num_sink;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  strides3(p.q_stride, q, c.packed);
  strides3(p.k_stride, k, c.packed);
  strides3(p.v_stride, v, c.packed);
  p.out = out.data_ptr();
  strides3(p.out_stride, out, c.packed);
  p.lse = (float*)lse.data_ptr();
  strides3(p.lse_stride, lse, c.packed);
  return p;
}

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

// 0, or the library's status with nothing launched
int forward(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, Tensor& out, Tensor& lse) {
  c10::DeviceGuard guard(q.device());
  out = at::empty(q.sizes(), q.options());
  const auto f32 = q.options().dtype(at::kFloat);
  lse = c.packed ? at::empty({q.size(1), q.size(0)}, f32) : at::empty({q.size(0), q.size(2), q.size(1)}, f32);
  const rswa_attn_params p = params(c, q, k, v, out, lse);
  void* const stream = stream_of(q);
  pybind11::gil_scoped_release others_run;  // (a launch waits where the queue is full)
  return lib.fwd(&p, stream);
}

[[noreturn]] void throw_python() {
  python_error err;
  err.persist();
  throw std::move(err);
}

struct Refused {};  // by the library, ahead of any launch: the Python route says why

struct BandNode : torch::autograd::Function<BandNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Call& c) {
    Tensor out, lse;
    if (::forward(c, q, k, v, out, lse) != RSWA_OK) throw Refused{};
    ctx->save_for_backward({q, k, v, out, lse});
    if (c.packed) ctx->saved_data["cu"] = c.cu;
    ctx->saved_data["mask"] = c10::IValue(c10::List<int64_t>({c.packed, c.window, c.num_sink}));
    ctx->saved_data["scale"] = (double)c.scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    const auto mask = ctx->saved_data["mask"].toIntList();
    const Call c{mask.get(0) != 0, (int32_t)mask.get(1), (int32_t)mask.get(2),
                 (float)ctx->saved_data["scale"].toDouble(),
                 mask.get(0) != 0 ? ctx->saved_data["cu"].toTensor() : Tensor()};
    Tensor dout = grads[0];
    if (dout.stride(-1) != 1) dout = dout.contiguous();
    const Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    // (hooks of saved tensors may give back others: what does not fit is for the Python route to refuse)
    const bool as_saved = fits(q, k, v, c.packed) && like(out, q) && like(dout, q) && lse_of(lse, q, c.packed) &&
                          (!c.packed || c.cu.device() == q.device());
    const bool switched = [] {  // (the thread that waits for the engine has let go of the lock: no cost to be seen)
      pybind11::gil_scoped_acquire gil;
      return env_switches();
    }();
    if (!as_saved || switched) {
      pybind11::gil_scoped_acquire gil;
      PyObject* r = PyObject_CallFunction(
          lib.python_bwd, "NNNNNNNNNdiNi", THPVariable_Wrap(q), THPVariable_Wrap(k), THPVariable_Wrap(v),
          THPVariable_Wrap(out), THPVariable_Wrap(lse), THPVariable_Wrap(dout), THPVariable_Wrap(dq),
          THPVariable_Wrap(dk), THPVariable_Wrap(dv), (double)c.scale, (int)c.window, THPVariable_Wrap(c.cu),
          (int)c.num_sink);
      if (!r) throw_python();
      Py_DECREF(r);
    } else {
      c10::DeviceGuard guard(q.device());
      rswa_attn_params p = params(c, q, k, v, out, lse);
      p.dout = dout.data_ptr();
      p.dq = dq.data_ptr();
      p.dk = dk.data_ptr();
      p.dv = dv.data_ptr();
      strides3(p.dout_stride, dout, c.packed);
      strides3(p.dq_stride, dq, c.packed);
      strides3(p.dk_stride, dk, c.packed);
      strides3(p.dv_stride, dv, c.packed);
      const Tensor ws = at::empty({(int64_t)lib.bwd_bytes(&p)}, q.options().dtype(at::kByte));
      p.workspace = ws.data_ptr();
      p.workspace_bytes = (uint64_t)ws.numel();
      const int rc = lib.bwd(&p, stream_of(q));
      if (rc != RSWA_OK) {
        pybind11::gil_scoped_acquire gil;
        PyObject* r = PyObject_CallFunction(lib.raise, "i", rc);
        Py_XDECREF(r);
        if (!r) throw_python();
      }
    }
    return {dq, dk, dv, Tensor()};
  }
};

// band_attn(q, k, v, window, softmax_scale or None, cu_seqlens or None, num_sink) -> out or None
PyObject* band_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !lib.fwd) Py_RETURN_NONE;
  for (int i = 0; i < 3; i++)
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
  const Tensor &q = THPVariable_Unpack(args[0]), &k = THPVariable_Unpack(args[1]), &v = THPVariable_Unpack(args[2]);
  Call c;
  c.packed = args[5] != Py_None;
  if (c.packed) {
    if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
    const Tensor& cu = c.cu = THPVariable_Unpack(args[5]);
    if (!plain(cu) || cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous() || cu.numel() < 2)
      Py_RETURN_NONE;
  }
  if (!fits(q, k, v, c.packed) || (c.packed && q.device() != c.cu.device()) || observed() || env_switches()) Py_RETURN_NONE;
  if (!PyLong_CheckExact(args[3]) || !PyLong_CheckExact(args[6])) Py_RETURN_NONE;
  int over = 0;
  const long long window = PyLong_AsLongLongAndOverflow(args[3], &over);
  if (over || window != (int32_t)window) Py_RETURN_NONE;
  const long long num_sink = PyLong_AsLongLongAndOverflow(args[6], &over);
  if (over || num_sink != (int32_t)num_sink) Py_RETURN_NONE;
  c.window = (int32_t)window;
  c.num_sink = (int32_t)num_sink;
  if (args[4] == Py_None) c.scale = (float)std::pow((double)q.size(-1), -0.5);
  else if (PyFloat_CheckExact(args[4])) c.scale = (float)PyFloat_AS_DOUBLE(args[4]);
  else Py_RETURN_NONE;
  Tensor out;
  if (c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    try {
      out = BandNode::apply(q, k, v, c);
    } catch (const Refused&) {
      Py_RETURN_NONE;
    }
  } else {
    Tensor lse;
    if (forward(c, q, k, v, out, lse) != RSWA_OK) Py_RETURN_NONE;
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- the calls over the 8-bit paged cache (ring_swa/ops/kv_cache.py makes the same in Python) --------------------
//
// A served token is a handful of kernels of 4 to 8 us; from Python the host takes 16 to 25 us for each of these calls (22
// to 31 under a torch function mode, such as a default device), here 4 to 9.  What they do not take (other types, tensors that need a gradient, modes) goes to Python, which refuses or
// handles it; a refusal of the library's is raised there too.

struct {
  int (*append)(const rswa_cache_params*, void*) = nullptr;
  int (*attn)(const rswa_cache_params*, void*) = nullptr;
  int (*weights)(const rswa_cache_params*, void*) = nullptr;
  int (*evict)(const rswa_cache_params*, void*) = nullptr;
  uint64_t (*attn_bytes)(const rswa_cache_params*) = nullptr;
  int (*read)(const rswa_cache_params*, void*) = nullptr;
  int (*draft_tree)(const rswa_tree_params*, void*) = nullptr;
  int (*tree_attn)(const rswa_draft_params*, void*) = nullptr;
  uint64_t (*tree_attn_bytes)(const rswa_draft_params*) = nullptr;
  int (*accept)(const rswa_draft_params*, void*) = nullptr;
  int (*verify)(const rswa_verify_params*, void*) = nullptr;
  uint64_t (*verify_bytes)(const rswa_verify_params*) = nullptr;
} cache_lib;

// A tensor argument that the calls take as it is; null: the Python route sees to it.
const Tensor* given(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return plain(t) ? &t : nullptr;
}

// (the calls have no backward: the Python route says so)
bool needs_grad(const Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }

// Dimensions from `from` on without gaps?  (A stride over one element is never used.)
bool dense_from(const Tensor& t, int64_t from) {
  int64_t step = 1;
  for (int64_t d = t.dim() - 1; d >= from; d--) {
    if (t.size(d) != 1 && t.stride(d) != step) return false;
    step *= t.size(d);
  }
  return true;
}

bool int_arg(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}

// 0, or the library's status with nothing launched
template <typename Params>
int launch_call(int (*entry)(const Params*, void*), const Params& p, c10::Device device) {
  void* const stream = (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream();
  pybind11::gil_scoped_release others_run;
  return entry(&p, stream);
}

struct CacheCall {
  rswa_cache_params p{};
  c10::Device device{c10::kCPU};
  bool packed = false;

  // (as ring_swa/ops/kv_cache.py:_cache_params; false: not a call for here)
  bool set(PyObject* cache, PyObject* table_o, PyObject* lens_o) {
    if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 4) return false;
    const Tensor* c[4];
    for (int i = 0; i < 4; i++)
      if (!(c[i] = given(PyTuple_GET_ITEM(cache, i))) || needs_grad(*c[i])) return false;
    const Tensor *table = given(table_o), *lens = given(lens_o);
    if (!table || !lens) return false;
    const Tensor &k = *c[0], &v = *c[1];
    if (k.dim() != 4 || v.dim() != 5 || table->dim() != 2 || lens->dim() != 1) return false;
    if (k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn ||
        c[2]->scalar_type() != at::kFloat8_e8m0fnu || c[3]->scalar_type() != at::kFloat8_e8m0fnu ||
        table->scalar_type() != at::kInt || lens->scalar_type() != at::kInt)
      return false;
    const int64_t pages = k.size(0), heads = k.size(1), size = k.size(2), dim = k.size(3);
    if (heads == 0 || pages >= INT32_MAX || table->size(0) >= INT32_MAX || table->size(1) >= INT32_MAX || size > 256)
      return false;
    if (!v.sizes().equals({pages, heads, size / 16, dim, 16}) || !c[2]->sizes().equals({pages, heads}) ||
        !c[3]->sizes().equals({pages, heads}) || lens->size(0) != table->size(0))
      return false;
    if (!dense_from(k, 2) || !dense_from(v, 2) || !dense_from(*table, 1) || !lens->is_contiguous()) return false;
    device = k.device();
    for (const Tensor* t : {c[1], c[2], c[3], table, lens})
      if (t->device() != device) return false;
    p.head_dim = (int32_t)dim;
    p.batch = (int32_t)table->size(0);
    p.heads_q = p.heads_kv = (int32_t)heads;
    p.page_size = (int32_t)size;
    p.num_pages = (int32_t)pages;
    p.max_pages = (int32_t)table->size(1);
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_scale = c[2]->data_ptr();
    p.v_scale = c[3]->data_ptr();
    for (int i = 0; i < 2; i++) {
      p.k_stride[i] = k.stride(i);
      p.v_stride[i] = v.stride(i);
      p.k_scale_stride[i] = c[2]->stride(i);
      p.v_scale_stride[i] = c[3]->stride(i);
    }
    p.page_table = (const int32_t*)table->data_ptr();
    p.page_table_stride = table->stride(0);
    p.seqlens = (const int32_t*)lens->data_ptr();
    return true;
  }

  // rows of queries, or of new keys
  bool rows(const Tensor& t, PyObject* cu_o) {
    const auto type = t.scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return false;
    if (needs_grad(t)) return false;
    packed = cu_o != Py_None;
    if (t.dim() != (packed ? 3 : 4) || t.size(-1) != p.head_dim || t.stride(-1) != 1 || t.device() != device)
      return false;
    for (int d = 0; d < t.dim(); d++)
      if (t.size(d) >= (1 << 28)) return false;
    p.dtype = type == at::kBFloat16 ? RSWA_BF16 : RSWA_F16;
    if (packed) {
      const Tensor* cu = given(cu_o);
      if (!cu || cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->size(0) != (int64_t)p.batch + 1 ||
          !cu->is_contiguous() || cu->device() != device)
        return false;
      p.total_q = t.size(0);
      p.cu_seqlens_q = (const int32_t*)cu->data_ptr();
    } else {
      if (t.size(0) != p.batch) return false;
      p.seqlen_q = (int32_t)t.size(1);
    }
    return true;
  }

  bool queries(const Tensor& q, PyObject* cu, PyObject* window_o, PyObject* scale_o, PyObject* sinks_o) {
    int64_t window, sinks;
    if (!rows(q, cu) || q.numel() == 0 || q.size(-2) % p.heads_kv != 0) return false;
    if (!int_arg(window_o, window) || !int_arg(sinks_o, sinks) || sinks < 0) return false;
    if (scale_o == Py_None) p.softmax_scale = (float)std::pow((double)p.head_dim, -0.5);
    else if (PyFloat_CheckExact(scale_o)) p.softmax_scale = (float)PyFloat_AS_DOUBLE(scale_o);
    else return false;
    p.heads_q = (int32_t)q.size(-2);
    p.window_left = (int32_t)std::max<int64_t>(-1, std::min<int64_t>(window, 1 << 28));
    p.num_sink = (int32_t)std::min<int64_t>(sinks, 1 << 28);
    p.q = q.data_ptr();
    strides3(p.q_stride, q, packed);
    return true;
  }

  Tensor results(const Tensor& q, bool want_lse, Tensor& lse) {
    Tensor out = at::empty(q.sizes(), q.options());
    p.out = out.data_ptr();
    strides3(p.out_stride, out, packed);
    if (want_lse) {
      const auto f32 = q.options().dtype(at::kFloat);
      lse = packed ? at::empty({q.size(1), q.size(0)}, f32) : at::empty({q.size(0), q.size(2), q.size(1)}, f32);
      p.lse = (float*)lse.data_ptr();
      strides3(p.lse_stride, lse, packed);
    }
    return out;
  }

  bool running_sums(const Tensor* w) {
    if (!w || w->scalar_type() != at::kFloat || w->dim() != 3 || w->size(0) != p.batch || w->size(1) != p.heads_kv ||
        !dense_from(*w, 2) || w->device() != device || w->size(2) >= INT32_MAX || needs_grad(*w))
      return false;
    int64_t span = w->size(2);  // of what the inner of the two strides has walked over
    const int inner = w->stride(0) < w->stride(1) ? 0 : 1;
    for (const int d : {inner, 1 - inner}) {
      if (w->size(d) > 1 && w->stride(d) < span) return false;  // (sums of different heads overlap)
      span += std::max<int64_t>(0, w->size(d) - 1) * w->stride(d);
    }
    p.weights = (float*)w->data_ptr();
    p.weights_stride[0] = w->stride(0);
    p.weights_stride[1] = w->stride(1);
    p.weights_len = (int32_t)w->size(2);
    return true;
  }

  // new keys and values, whose rows are `like`'s
  bool new_rows(const Tensor* k, const Tensor* v, const Tensor& like) {
    if (!k || !v || k->dim() != like.dim() || v->sizes() != k->sizes() || k->size(-2) != p.heads_kv) return false;
    for (int d = 0; d < k->dim(); d++)
      if (d != k->dim() - 2 && k->size(d) != like.size(d)) return false;
    for (const Tensor* t : {k, v})
      if (t->scalar_type() != like.scalar_type() || t->device() != device || t->stride(-1) != 1 || needs_grad(*t)) return false;
    p.new_k = k->data_ptr();
    p.new_v = v->data_ptr();
    strides3(p.new_k_stride, *k, packed);
    strides3(p.new_v_stride, *v, packed);
    return true;
  }

  // 0, or the library's status with nothing launched
  int launch(int (*entry)(const rswa_cache_params*, void*)) { return launch_call(entry, p, device); }
};

// An integer tensor whose rows are dense from `from` on, on the device; null otherwise.
const Tensor* ints(PyObject* o, at::ScalarType type, c10::IntArrayRef sizes, int64_t from, c10::Device device) {
  const Tensor* t = given(o);
  return t && t->scalar_type() == type && t->sizes() == sizes && t->device() == device && dense_from(*t, from) ? t : nullptr;
}

// cache_append(cache, k, v, page_table, seqlens, cu_seqlens or None) -> True, or None: not taken
PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 6 || !cache_lib.append || observed()) Py_RETURN_NONE;
  const Tensor *k = given(args[1]), *v = given(args[2]);
  if (!k || !v || !c.set(args[0], args[3], args[4]) || !c.rows(*k, args[5])) Py_RETURN_NONE;
  if (!c.new_rows(k, v, *k)) Py_RETURN_NONE;
  c10::DeviceGuard guard(c.device);
  if (c.launch(cache_lib.append) != RSWA_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// cache_attn(q, cache, page_table, seqlens, window, cu_seqlens or None, scale or None, sinks, return_lse)
//   -> out or (out, lse), or None: not taken
PyObject* cache_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 9 || !cache_lib.attn || observed() || !PyBool_Check(args[8])) Py_RETURN_NONE;
  const Tensor* q = given(args[0]);
  if (!q || !c.set(args[1], args[2], args[3]) || !c.queries(*q, args[5], args[4], args[6], args[7]) || c.p.max_pages == 0)
    Py_RETURN_NONE;
  c10::DeviceGuard guard(c.device);
  Tensor lse, workspace, out = c.results(*q, args[8] == Py_True, lse);
  if (const uint64_t bytes = cache_lib.attn_bytes(&c.p)) {
    workspace = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
    c.p.workspace = workspace.data_ptr();
    c.p.workspace_bytes = bytes;
  }
  if (c.launch(cache_lib.attn) != RSWA_OK) Py_RETURN_NONE;
  if (!lse.defined()) return THPVariable_Wrap(std::move(out));
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
  END_HANDLE_TH_ERRORS
}

// cache_weights(q, cache, page_table, seqlens, lse, weights, window, cu_seqlens or None, scale or None, sinks)
//   -> True, or None: not taken
PyObject* cache_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 10 || !cache_lib.weights || observed()) Py_RETURN_NONE;
  const Tensor *q = given(args[0]), *lse = given(args[4]);
  if (!q || !lse || !c.set(args[1], args[2], args[3]) || !c.queries(*q, args[7], args[6], args[8], args[9]) ||
      c.p.max_pages == 0 || !c.running_sums(given(args[5])) || !lse_of(*lse, *q, c.packed) || needs_grad(*lse))
    Py_RETURN_NONE;
  c.p.lse = (float*)lse->data_ptr();
  strides3(c.p.lse_stride, *lse, c.packed);
  c10::DeviceGuard guard(c.device);
  if (c.launch(cache_lib.weights) != RSWA_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// cache_evict(cache, weights, page_table, seqlens, new_page_table, budget, sinks, recent)
//   -> (seqlens, weights, kept), or None: not taken
PyObject* cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  int64_t budget, sinks, recent;
  if (n != 8 || !cache_lib.evict || observed()) Py_RETURN_NONE;
  if (!int_arg(args[5], budget) || !int_arg(args[6], sinks) || !int_arg(args[7], recent)) Py_RETURN_NONE;
  if (budget <= 0 || budget >= INT32_MAX || sinks < 0 || recent < 0 || sinks > budget - recent) Py_RETURN_NONE;
  const Tensor* to = given(args[4]);
  if (!to || !c.set(args[0], args[2], args[3]) || !c.running_sums(given(args[1]))) Py_RETURN_NONE;
  if (to->dim() != 2 || to->scalar_type() != at::kInt || to->size(0) != c.p.batch || !dense_from(*to, 1) ||
      to->device() != c.device || to->size(1) >= INT32_MAX)
    Py_RETURN_NONE;
  c10::DeviceGuard guard(c.device);
  const Tensor &w = THPVariable_Unpack(args[1]), &lens = THPVariable_Unpack(args[3]);
  Tensor new_lens = at::empty(lens.sizes(), lens.options()), new_w = at::empty(w.sizes(), w.options()),
         kept = at::empty({c.p.batch, c.p.heads_kv, budget}, lens.options());
  c.p.budget = (int32_t)budget;
  c.p.num_sink = (int32_t)sinks;
  c.p.num_recent = (int32_t)recent;
  c.p.new_page_table = (const int32_t*)to->data_ptr();
  c.p.new_page_table_stride = to->stride(0);
  c.p.new_max_pages = (int32_t)to->size(1);
  c.p.new_seqlens = (int32_t*)new_lens.data_ptr();
  c.p.new_weights = (float*)new_w.data_ptr();
  c.p.kept = (int32_t*)kept.data_ptr();
  if (c.launch(cache_lib.evict) != RSWA_OK) Py_RETURN_NONE;
  return Py_BuildValue("NNN", THPVariable_Wrap(std::move(new_lens)), THPVariable_Wrap(std::move(new_w)),
                       THPVariable_Wrap(std::move(kept)));
  END_HANDLE_TH_ERRORS
}

// cache_read(cache, k, v, page_table, first, cu_seqlens or None) -> True, or None: not taken
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 6 || !cache_lib.read || observed()) Py_RETURN_NONE;
  const Tensor *k = given(args[1]), *v = given(args[2]);
  if (!k || !v || !c.set(args[0], args[3], args[4]) || !c.rows(*k, args[5]) || !c.new_rows(k, v, *k)) Py_RETURN_NONE;
  c10::DeviceGuard guard(c.device);
  if (c.launch(cache_lib.read) != RSWA_OK) Py_RETURN_NONE;
  for (const Tensor* t : {k, v})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();  // (a graph that has saved them is to notice)
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// ---- drafted tokens (ring_swa/ops/drafts.py makes the same in Python) ---------------------------------------------

// cu_seqlens of a pack, or None
bool pack_of(PyObject* o, c10::Device device, const Tensor*& cu) {
  cu = nullptr;
  if (o == Py_None) return true;
  cu = given(o);
  return cu && cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) >= 1 && cu->size(0) < (1 << 28) &&
         cu->is_contiguous() && cu->device() == device;
}

// draft_tree(parents, cu_seqlens or None, max_nodes) -> (parents, depths, ancestors), or None: not taken
PyObject* draft_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t max_nodes;
  if (n != 3 || !cache_lib.draft_tree || observed() || !int_arg(args[2], max_nodes)) Py_RETURN_NONE;
  const Tensor *parents = given(args[0]), *cu;
  if (!parents || parents->scalar_type() != at::kInt || !pack_of(args[1], parents->device(), cu)) Py_RETURN_NONE;
  if (parents->dim() != (cu ? 1 : 2) || !dense_from(*parents, parents->dim() - 1) || max_nodes < 1 || max_nodes > 1024)
    Py_RETURN_NONE;
  for (int64_t d = 0; d < parents->dim(); d++)
    if (parents->size(d) >= (1 << 28)) Py_RETURN_NONE;
  rswa_tree_params p{};
  if (cu) {
    p.batch = (int32_t)(cu->size(0) - 1);
    p.total = parents->size(0);
    p.cu_seqlens = (const int32_t*)cu->data_ptr();
  } else {
    p.batch = (int32_t)parents->size(0);
    p.nodes = (int32_t)parents->size(1);
    p.parents_stride = parents->stride(0);
  }
  p.max_nodes = (int32_t)max_nodes;
  p.parents = (const int32_t*)parents->data_ptr();
  c10::DeviceGuard guard(parents->device());
  auto sizes = parents->sizes().vec();
  Tensor up = at::empty(sizes, parents->options()), depths = at::empty(sizes, parents->options());
  sizes.push_back((max_nodes + 63) / 64);
  Tensor ancestors = at::empty(sizes, parents->options().dtype(at::kLong));
  p.tree_parents = (int32_t*)up.data_ptr();
  p.depths = (int32_t*)depths.data_ptr();
  p.ancestors = (int64_t*)ancestors.data_ptr();
  if (launch_call(cache_lib.draft_tree, p, parents->device()) != RSWA_OK) Py_RETURN_NONE;
  return Py_BuildValue("NNN", THPVariable_Wrap(std::move(up)), THPVariable_Wrap(std::move(depths)),
                       THPVariable_Wrap(std::move(ancestors)));
  END_HANDLE_TH_ERRORS
}

// cache_tree_attn(q, k, v, tree, cache, page_table, seqlens, window, cu_seqlens or None, scale or None, sinks, return_lse)
//   -> out or (out, lse), or None: not taken
PyObject* cache_tree_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 12 || !cache_lib.tree_attn || observed() || !PyBool_Check(args[11])) Py_RETURN_NONE;
  if (!PyTuple_Check(args[3]) || PyTuple_GET_SIZE(args[3]) != 3) Py_RETURN_NONE;
  const Tensor* q = given(args[0]);
  if (!q || !c.set(args[4], args[5], args[6]) || !c.queries(*q, args[8], args[7], args[9], args[10])) Py_RETURN_NONE;
  if (!c.new_rows(given(args[1]), given(args[2]), *q)) Py_RETURN_NONE;
  const auto rows = q->sizes().slice(0, q->dim() - 2);
  const int64_t nd = (int64_t)rows.size();
  const Tensor* depths = ints(PyTuple_GET_ITEM(args[3], 1), at::kInt, rows, nd - 1, c.device);
  const Tensor* ancestors = given(PyTuple_GET_ITEM(args[3], 2));
  if (!depths || !ancestors || ancestors->dim() != nd + 1) Py_RETURN_NONE;
  const int64_t words = ancestors->size(-1);
  auto sizes = rows.vec();
  sizes.push_back(words);
  if (!ints(PyTuple_GET_ITEM(args[3], 2), at::kLong, sizes, nd - 1, c.device)) Py_RETURN_NONE;
  if (words < 1 || words > 16 || (!c.packed && rows[1] > 64 * words)) Py_RETURN_NONE;
  c10::DeviceGuard guard(c.device);
  Tensor lse, workspace, out = c.results(*q, args[11] == Py_True, lse);
  rswa_draft_params p{};
  p.cache = c.p;
  p.depths = (const int32_t*)depths->data_ptr();
  p.ancestors = (const int64_t*)ancestors->data_ptr();
  if (!c.packed) {
    p.depths_stride = depths->stride(0);
    p.ancestors_stride = ancestors->stride(0);
  }
  p.words = (int32_t)words;
  if (const uint64_t bytes = cache_lib.tree_attn_bytes(&p)) {
    workspace = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
    p.cache.workspace = workspace.data_ptr();
    p.cache.workspace_bytes = bytes;
  }
  if (launch_call(cache_lib.tree_attn, p, c.device) != RSWA_OK) Py_RETURN_NONE;
  if (!lse.defined()) return THPVariable_Wrap(std::move(out));
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
  END_HANDLE_TH_ERRORS
}

// cache_accept(cache, k, v, path, page_table, seqlens, cu_seqlens or None) -> True, or None: not taken
PyObject* cache_accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CacheCall c;
  if (n != 7 || !cache_lib.accept || observed()) Py_RETURN_NONE;
  const Tensor *k = given(args[1]), *v = given(args[2]), *path = given(args[3]);
  if (!k || !v || !path || path->dim() != 2 || path->size(1) >= (1 << 28)) Py_RETURN_NONE;
  if (!c.set(args[0], args[4], args[5]) || !c.rows(*k, args[6]) || !c.new_rows(k, v, *k)) Py_RETURN_NONE;
  if (!ints(args[3], at::kInt, {c.p.batch, path->size(1)}, 1, c.device)) Py_RETURN_NONE;
  rswa_draft_params p{};
  p.cache = c.p;
  p.path = (const int32_t*)path->data_ptr();
  p.path_stride = path->stride(0);
  p.path_len = (int32_t)path->size(1);
  c10::DeviceGuard guard(c.device);
  if (launch_call(cache_lib.accept, p, c.device) != RSWA_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// verify_drafts(tree, tokens, target, draft or None, uniforms, cu_seqlens or None) -> (path, accepted, next), or None: not taken
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !cache_lib.verify || observed()) Py_RETURN_NONE;
  if (!PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != 3) Py_RETURN_NONE;
  const Tensor *target = given(args[2]), *draft = args[3] == Py_None ? nullptr : given(args[3]), *cu;
  const Tensor *tokens = given(args[1]), *ancestors = given(PyTuple_GET_ITEM(args[0], 2));
  if (!target || !tokens || !ancestors || (!draft && args[3] != Py_None)) Py_RETURN_NONE;
  const c10::Device device = target->device();
  if (!pack_of(args[5], device, cu) || target->dim() != (cu ? 2 : 3) || ancestors->dim() != target->dim()) Py_RETURN_NONE;
  const auto type = target->scalar_type(), token_type = tokens->scalar_type();
  if ((type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) ||
      (token_type != at::kInt && token_type != at::kLong))
    Py_RETURN_NONE;
  for (const Tensor* t : {target, draft})
    if (t && (t->sizes() != target->sizes() || t->scalar_type() != type || t->device() != device || needs_grad(*t) ||
              (t->stride(-1) != 1 && t->size(-1) != 1)))
      Py_RETURN_NONE;
  for (int64_t d = 0; d < target->dim(); d++)
    if (target->size(d) >= (1 << 28)) Py_RETURN_NONE;
  const auto rows = target->sizes().slice(0, target->dim() - 1);
  const int64_t nd = (int64_t)rows.size();
  const Tensor* parents = ints(PyTuple_GET_ITEM(args[0], 0), at::kInt, rows, nd - 1, device);
  const Tensor* uniforms = ints(args[4], at::kFloat, rows, nd - 1, device);
  if (!parents || !uniforms || needs_grad(*uniforms) || !ints(args[1], token_type, rows, nd - 1, device)) Py_RETURN_NONE;
  rswa_verify_params p{};
  p.dtype = type == at::kFloat ? RSWA_F32 : type == at::kBFloat16 ? RSWA_BF16 : RSWA_F16;
  p.token_bytes = token_type == at::kInt ? 4 : 8;
  p.vocab = (int32_t)target->size(-1);
  p.max_nodes = (int32_t)std::min<int64_t>(64 * ancestors->size(-1), INT32_MAX);
  const auto strides = [&](int64_t(&to)[2], const Tensor& t) {
    to[0] = cu ? 0 : t.stride(0);
    to[1] = t.stride(cu ? 0 : 1);
  };
  if (cu) {
    p.batch = (int32_t)(cu->size(0) - 1);
    p.total = rows[0];
    p.cu_seqlens = (const int32_t*)cu->data_ptr();
  } else {
    p.batch = (int32_t)rows[0];
    p.nodes = (int32_t)rows[1];
    p.parents_stride = parents->stride(0);
    p.tokens_stride = tokens->stride(0);
    p.uniforms_stride = uniforms->stride(0);
  }
  p.parents = (const int32_t*)parents->data_ptr();
  p.tokens = tokens->data_ptr();
  p.uniforms = (const float*)uniforms->data_ptr();
  p.target = target->data_ptr();
  strides(p.target_stride, *target);
  if (draft) {
    p.draft = draft->data_ptr();
    strides(p.draft_stride, *draft);
  }
  c10::DeviceGuard guard(device);
  p.path_len = cu ? p.max_nodes : p.nodes;
  if (p.max_nodes < 1 || p.max_nodes > 1024) Py_RETURN_NONE;
  Tensor path = at::empty({p.batch, p.path_len}, parents->options()), accepted = at::empty({p.batch}, parents->options());
  Tensor next = at::empty({p.batch}, tokens->options());
  p.path = (int32_t*)path.data_ptr();
  p.accepted = (int32_t*)accepted.data_ptr();
  p.next_token = next.data_ptr();
  const uint64_t bytes = cache_lib.verify_bytes(&p);
  Tensor workspace = at::empty({(int64_t)bytes}, target->options().dtype(at::kByte));
  p.workspace = workspace.data_ptr();
  p.workspace_bytes = bytes;
  if (launch_call(cache_lib.verify, p, device) != RSWA_OK) Py_RETURN_NONE;
  return Py_BuildValue("NNN", THPVariable_Wrap(std::move(path)), THPVariable_Wrap(std::move(accepted)),
                       THPVariable_Wrap(std::move(next)));
  END_HANDLE_TH_ERRORS
}

// bind_cache(rswa_cache_append, .._attn, .._weights, .._evict, .._attn_workspace_bytes, .._read, rswa_draft_tree,
//   rswa_cache_tree_attn, .._tree_attn_workspace_bytes, .._accept, rswa_verify_drafts, .._workspace_bytes): addresses
PyObject* bind_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 12) {
    PyErr_SetString(PyExc_TypeError, "bind_cache takes twelve addresses");
    return nullptr;
  }
  void* at[12];
  for (int i = 0; i < 12; i++) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  cache_lib.read = reinterpret_cast<decltype(cache_lib.read)>(at[5]);
  cache_lib.draft_tree = reinterpret_cast<decltype(cache_lib.draft_tree)>(at[6]);
  cache_lib.tree_attn_bytes = reinterpret_cast<decltype(cache_lib.tree_attn_bytes)>(at[8]);
  cache_lib.tree_attn = reinterpret_cast<decltype(cache_lib.tree_attn)>(at[7]);
  cache_lib.accept = reinterpret_cast<decltype(cache_lib.accept)>(at[9]);
  cache_lib.verify_bytes = reinterpret_cast<decltype(cache_lib.verify_bytes)>(at[11]);
  cache_lib.verify = reinterpret_cast<decltype(cache_lib.verify)>(at[10]);
  cache_lib.attn_bytes = reinterpret_cast<decltype(cache_lib.attn_bytes)>(at[4]);
  cache_lib.append = reinterpret_cast<decltype(cache_lib.append)>(at[0]);
  cache_lib.attn = reinterpret_cast<decltype(cache_lib.attn)>(at[1]);
  cache_lib.weights = reinterpret_cast<decltype(cache_lib.weights)>(at[2]);
  cache_lib.evict = reinterpret_cast<decltype(cache_lib.evict)>(at[3]);
  Py_RETURN_NONE;
}

// bind(rswa_attn_fwd, rswa_attn_bwd, rswa_attn_bwd_workspace_bytes, raise, python_bwd): addresses and callables
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes three addresses and two callables");
    return nullptr;
  }
  void* at[3];
  for (int i = 0; i < 3; i++) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib.bwd = reinterpret_cast<decltype(lib.bwd)>(at[1]);
  lib.bwd_bytes = reinterpret_cast<decltype(lib.bwd_bytes)>(at[2]);
  Py_INCREF(args[3]);
  Py_INCREF(args[4]);
  lib.raise = args[3];
  lib.python_bwd = args[4];
  lib.fwd = reinterpret_cast<decltype(lib.fwd)>(at[0]);
  Py_RETURN_NONE;
}

// The PyTorch whose headers this was compiled with (ring_swa._lib.torch_build): their inlined accessors read
// tensors at its layout, so that another must not be handed any
PyObject* torch_build(PyObject*, PyObject*) { return PyUnicode_FromString(RSWA_TORCH_BUILD); }

PyObject* params_bytes(PyObject*, PyObject*) { return PyLong_FromSize_t(sizeof(rswa_attn_params)); }

PyObject* cache_params_bytes(PyObject*, PyObject*) { return PyLong_FromSize_t(sizeof(rswa_cache_params)); }

// of the trees, the calls that take one, and the verification
PyObject* draft_params_bytes(PyObject*, PyObject*) {
  return Py_BuildValue("nnn", (Py_ssize_t)sizeof(rswa_tree_params), (Py_ssize_t)sizeof(rswa_draft_params),
                       (Py_ssize_t)sizeof(rswa_verify_params));
}

PyMethodDef methods[] = {
    {"band_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&band_attn)), METH_FASTCALL, nullptr},
    {"cache_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_append)), METH_FASTCALL, nullptr},
    {"cache_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_attn)), METH_FASTCALL, nullptr},
    {"cache_weights", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_weights)), METH_FASTCALL, nullptr},
    {"cache_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_evict)), METH_FASTCALL, nullptr},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_read)), METH_FASTCALL, nullptr},
    {"draft_tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&draft_tree)), METH_FASTCALL, nullptr},
    {"cache_tree_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_tree_attn)), METH_FASTCALL, nullptr},
    {"cache_accept", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_accept)), METH_FASTCALL, nullptr},
    {"verify_drafts", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&verify_drafts)), METH_FASTCALL, nullptr},
    {"bind_cache", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&bind_cache)), METH_FASTCALL, nullptr},
    {"cache_params_bytes", &cache_params_bytes, METH_NOARGS, nullptr},
    {"draft_params_bytes", &draft_params_bytes, METH_NOARGS, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&bind)), METH_FASTCALL, nullptr},
    {"params_bytes", &params_bytes, METH_NOARGS, nullptr},
    {"torch_build", &torch_build, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "rswa_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_rswa_torch() { return PyModule_Create(&module); }
