// Python functions of the decoder-serving operators: the checks of their tensors, the
// outputs and workspaces, and one C-ABI call (include/b2msl.h) on the tensors' device
// and current stream.
//
// A decode step calls these on a few tokens, where the call's cost is the host's: in
// Python (ctypes, torch.empty, tensor attributes) a call took 12 to 22 us, of which the
// launches are 4 to 7. The C entry points come as addresses from the loaded libb2msl.so
// (bind), so both bindings use one copy of the library.
//
// Each operator has two names: its own makes the call, for the kernel that is registered
// with torch; direct_... does so only where torch's dispatcher would come to that kernel
// at once, and otherwise returns NotImplemented, upon which the caller goes through it.
#include <Python.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <optional>
#include <string>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b2msl.h"

namespace {

struct Entries {
  decltype(&b2_qk_norm_rope) qk_norm_rope;
  decltype(&b2_kv_cache_write) kv_cache_write;
  decltype(&b2_kv_cache_read) kv_cache_read;
  decltype(&b2_kv_cache_attn) kv_cache_attn;
  decltype(&b2_fa_packed) fa_packed;
  decltype(&b2_query_workspace) query_workspace;
} entries = {};

// A Python exception on its way to the boundary; type null: already set.
struct Raise {
  PyObject* type;
  char text[400];
};
[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
  Raise r;
  r.type = type;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(r.text, sizeof(r.text), fmt, ap);
  va_end(ap);
  throw r;
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
const char* dtype_of(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

struct GilReleased {
  PyThreadState* const state = PyEval_SaveThread();
  ~GilReleased() { PyEval_RestoreThread(state); }
};

// The tensors of one call: all on one CUDA device.
class Call {
 public:
  Call(const char* what, PyObject* const* args, Py_ssize_t given, Py_ssize_t wanted) : what_(what), args_(args) {
    if (given != wanted) raise(PyExc_TypeError, "%s: %zd arguments given, %zd wanted", what, given, wanted);
    if (!entries.query_workspace) raise(PyExc_RuntimeError, "%s: the kernel library is not bound", what);
  }
  const at::Tensor& tensor(int i) {
    if (!THPVariable_Check(args_[i])) raise(PyExc_TypeError, "%s: argument %d must be a tensor", what_, i + 1);
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (!t.is_cuda())
      raise(PyExc_RuntimeError, "%s: tensors must be on a CUDA device (got %s); b2msl has no CPU path", what_,
            t.device().str().c_str());
    if (device_ < 0) device_ = t.device().index();
    else if (device_ != t.device().index())
      raise(PyExc_RuntimeError, "%s: tensors on different devices (cuda:%d vs %s)", what_, device_,
            t.device().str().c_str());
    return t;
  }
  const at::Tensor* maybe(int i) { return args_[i] == Py_None ? nullptr : &tensor(i); }
  double number(int i) const {
    const double x = PyFloat_AsDouble(args_[i]);
    if (x == -1.0 && PyErr_Occurred()) raise(nullptr, "");
    return x;
  }
  bool truth(int i) const {
    const int x = PyObject_IsTrue(args_[i]);
    if (x < 0) raise(nullptr, "");
    return x != 0;
  }
  int float_code(const at::Tensor& t) const {
    switch (t.scalar_type()) {
      case at::kFloat: return B2_F32;
      case at::kHalf: return B2_F16;
      case at::kBFloat16: return B2_BF16;
      default: raise(PyExc_TypeError, "%s: unsupported dtype %s (float32/float16/bfloat16)", what_, dtype_of(t));
    }
  }
  // A contiguous index vector of `size` entries.
  int index_code(const at::Tensor& t, const char* name, int64_t size, bool wide) const {
    const bool is64 = t.scalar_type() == at::kLong;
    if (!(t.scalar_type() == at::kInt || (wide && is64)))
      raise(PyExc_TypeError, "%s: %s must be int32%s, got %s", what_, name, wide ? " or int64" : "", dtype_of(t));
    if (t.dim() != 1 || t.size(0) != size)
      raise(PyExc_ValueError, "%s: %s must have shape (%lld,), got %s", what_, name, (long long)size, shape_of(t).c_str());
    if (size > 1 && t.stride(0) != 1) raise(PyExc_ValueError, "%s: %s must be contiguous", what_, name);
    return is64 ? B2_I64 : B2_I32;
  }
  // t itself, or a copy where the channels do not lie next to one another
  static at::Tensor unit(const at::Tensor& t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
  }
  at::Tensor empty(c10::IntArrayRef size, at::ScalarType type) const {
    return at::Tensor(at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device_), std::nullopt));
  }
  // Runs f(stream) with the device current and the GIL released; a status other than
  // B2_OK raises. f makes the C call and nothing else: a tensor without storage throws
  // when its pointer is asked for, so the pointers are taken before.
  template <typename F>
  void run(const char* fn, F&& f) const {
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != device_) guard.set_index((c10::DeviceIndex)device_);
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device_).stream();
    int status;
    {
      const GilReleased released;  // taken back also where f throws
      status = f(stream);
    }
    if (status == B2_OK) return;
    // the package's own exception, with the library's message
    PyObject* lib = PyImport_ImportModule("triton_msl_b200._lib");
    PyObject* done = lib ? PyObject_CallMethod(lib, "check", "si", fn, status) : nullptr;
    Py_XDECREF(done);
    Py_XDECREF(lib);
    if (!PyErr_Occurred()) raise(PyExc_RuntimeError, "%s failed (status %d)", fn, status);
    raise(nullptr, "");
  }
  const char* what() const { return what_; }

 private:
  const char* what_;
  PyObject* const* args_;
  int device_ = -1;
};

// Every exception ends here: nothing passes into the interpreter's C code.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Raise& r) {
    if (r.type) PyErr_SetString(r.type, r.text);
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = x ? THPVariable_Wrap(std::move(b)) : nullptr;
  PyObject* out = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return out;
}

// (q, k, table, positions, q_weight, k_weight, eps, interleaved) -> (q, k)
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&] {
    Call c("qk_norm_rope", args, nargs, 8);
    const at::Tensor &q0 = c.tensor(0), &k0 = c.tensor(1), &table = c.tensor(2), &positions = c.tensor(3);
    const at::Tensor* weights[2] = {c.maybe(4), c.maybe(5)};
    const float eps = (float)c.number(6);
    const int interleaved = c.truth(7);
    const int dt = c.float_code(q0);
    if (q0.dim() != 3 || k0.dim() != 3 || q0.size(0) != k0.size(0) || q0.size(2) != k0.size(2))
      raise(PyExc_ValueError, "%s: need q [T, Hq, D] and k [T, Hk, D]; got %s, %s", c.what(), shape_of(q0).c_str(),
            shape_of(k0).c_str());
    if (k0.scalar_type() != q0.scalar_type())
      raise(PyExc_TypeError, "%s: q and k must share a dtype (%s vs %s)", c.what(), dtype_of(q0), dtype_of(k0));
    const int64_t T = q0.size(0), Hq = q0.size(1), Hk = k0.size(1), D = q0.size(2);
    if (table.dim() != 2 || table.scalar_type() != at::kFloat || !table.is_contiguous())
      raise(PyExc_ValueError, "%s: table must be contiguous float32 [positions, rot_dim]", c.what());
    const int64_t P = table.size(0), R = table.size(1);
    if (R % 2 || R > D || D % 2)
      raise(PyExc_ValueError, "%s: rot_dim %lld must be even and at most head_dim %lld (even)", c.what(), (long long)R,
            (long long)D);
    const int pos = c.index_code(positions, "positions", T, true);
    for (int i = 0; i < 2; ++i) {
      const at::Tensor* w = weights[i];
      if (w && (w->scalar_type() != q0.scalar_type() || w->dim() != 1 || w->size(0) != D || !w->is_contiguous()))
        raise(PyExc_ValueError, "%s: %s must be contiguous [%lld] of dtype %s", c.what(), i ? "k_weight" : "q_weight",
              (long long)D, dtype_of(q0));
    }
    const at::Tensor q = Call::unit(q0), k = Call::unit(k0);
    at::Tensor qo = c.empty({T, Hq, D}, q.scalar_type()), ko = c.empty({T, Hk, D}, q.scalar_type());
    const int64_t strides[8] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), Hq * D, D, Hk * D, D};
    const void* in[4] = {q.const_data_ptr(), k.const_data_ptr(), weights[0] ? weights[0]->const_data_ptr() : nullptr,
                         weights[1] ? weights[1]->const_data_ptr() : nullptr};
    void* out[2] = {qo.mutable_data_ptr(), ko.mutable_data_ptr()};
    const float* angles = static_cast<const float*>(table.const_data_ptr());
    const void* at = positions.const_data_ptr();
    c.run("b2_qk_norm_rope", [&](void* stream) {
      return entries.qk_norm_rope(in[0], in[1], out[0], out[1], in[2], in[3], angles, at, pos, T, Hq, Hk, D, R, P, strides,
                                  eps, interleaved, dt, stream);
    });
    return pair(std::move(qo), std::move(ko));
  });
}

// The four arrays of a KVCache at args[i ..]: {pages, H, page_size, D, group}.
struct Cache {
  const at::Tensor &kc, &ks, &vc, &vs;
  int64_t shape[5];
  Cache(Call& c, int i) : kc(c.tensor(i)), ks(c.tensor(i + 1)), vc(c.tensor(i + 2)), vs(c.tensor(i + 3)) {
    if (kc.dim() != 4 || ks.dim() != 5 || vc.sizes() != kc.sizes() || vs.sizes() != ks.sizes() || ks.size(0) != kc.size(0) ||
        ks.size(1) != kc.size(1) || ks.size(2) != kc.size(2) || ks.size(3) == 0 || ks.size(4) != 2)
      raise(PyExc_ValueError, "%s: not a KVCache: codes %s, %s, scales %s, %s", c.what(), shape_of(kc).c_str(),
            shape_of(vc).c_str(), shape_of(ks).c_str(), shape_of(vs).c_str());
    if (kc.scalar_type() != at::kByte || vc.scalar_type() != at::kByte || ks.scalar_type() != at::kBFloat16 ||
        vs.scalar_type() != at::kBFloat16)
      raise(PyExc_TypeError, "%s: the cache holds uint8 codes and bfloat16 scales", c.what());
    if (!kc.is_contiguous() || !ks.is_contiguous() || !vc.is_contiguous() || !vs.is_contiguous())
      raise(PyExc_ValueError, "%s: the cache's tensors must be contiguous", c.what());
    shape[0] = kc.size(0);
    shape[1] = kc.size(1);
    shape[2] = kc.size(2);
    shape[3] = 2 * kc.size(3);
    shape[4] = shape[3] / ks.size(3);
  }
  int64_t H() const { return shape[1]; }
  int64_t D() const { return shape[3]; }
  // The four arrays, to be read.
  struct Arrays {
    const void *kc, *ks, *vc, *vs;
  };
  Arrays arrays() const { return {kc.const_data_ptr(), ks.const_data_ptr(), vc.const_data_ptr(), vs.const_data_ptr()}; }
};

// (k_codes, k_scales, v_codes, v_scales, k, v, slots) -> None
PyObject* kv_cache_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Call c("kv_cache_write", args, nargs, 7);
    const Cache cache(c, 0);
    const at::Tensor &k0 = c.tensor(4), &v0 = c.tensor(5), &slots = c.tensor(6);
    if (k0.dim() != 3 || v0.sizes() != k0.sizes() || k0.size(1) != cache.H() || k0.size(2) != cache.D())
      raise(PyExc_ValueError, "%s: k and v must be [T, %lld, %lld]; got %s, %s", c.what(), (long long)cache.H(),
            (long long)cache.D(), shape_of(k0).c_str(), shape_of(v0).c_str());
    if (v0.scalar_type() != k0.scalar_type())
      raise(PyExc_TypeError, "%s: k and v must share a dtype (%s vs %s)", c.what(), dtype_of(k0), dtype_of(v0));
    const int dt = c.float_code(k0);
    const int64_t T = k0.size(0);
    const int sdt = c.index_code(slots, "slots", T, true);
    const at::Tensor k = Call::unit(k0), v = Call::unit(v0);
    const int64_t strides[4] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
    const void *kp = k.const_data_ptr(), *vp = v.const_data_ptr(), *at = slots.const_data_ptr();
    void* to[4] = {cache.kc.mutable_data_ptr(), cache.ks.mutable_data_ptr(), cache.vc.mutable_data_ptr(),
                   cache.vs.mutable_data_ptr()};
    c.run("b2_kv_cache_write", [&](void* stream) {
      return entries.kv_cache_write(kp, vp, to[0], to[1], to[2], to[3], at, sdt, T, cache.shape, strides, dt, stream);
    });
    // the cache was written in place: views that autograd or a tracer holds see a new version
    for (const at::Tensor* t : {&cache.kc, &cache.ks, &cache.vc, &cache.vs})
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
  });
}

// (k_codes, k_scales, v_codes, v_scales, slots, dtype) -> (k, v)
PyObject* kv_cache_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&] {
    Call c("kv_cache_read", args, nargs, 6);
    const Cache cache(c, 0);
    const at::Tensor& slots = c.tensor(4);
    if (slots.dim() != 1) raise(PyExc_ValueError, "%s: slots must be [T], got %s", c.what(), shape_of(slots).c_str());
    if (!THPDtype_Check(args[5])) raise(PyExc_TypeError, "%s: dtype must be a torch.dtype", c.what());
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    int dt = -1;
    if (type == at::kFloat) dt = B2_F32;
    if (type == at::kHalf) dt = B2_F16;
    if (type == at::kBFloat16) dt = B2_BF16;
    if (dt < 0) raise(PyExc_TypeError, "%s: unsupported dtype %s (float32/float16/bfloat16)", c.what(), c10::toString(type));
    const int64_t T = slots.size(0), H = cache.H(), D = cache.D();
    const int sdt = c.index_code(slots, "slots", T, true);
    at::Tensor k = c.empty({T, H, D}, type), v = c.empty({T, H, D}, type);
    const int64_t strides[4] = {H * D, D, H * D, D};
    void *kp = k.mutable_data_ptr(), *vp = v.mutable_data_ptr();
    const Cache::Arrays from = cache.arrays();
    const void* at = slots.const_data_ptr();
    c.run("b2_kv_cache_read", [&](void* stream) {
      return entries.kv_cache_read(kp, vp, from.kc, from.ks, from.vc, from.vs, at, sdt, T, cache.shape, strides, dt, stream);
    });
    return pair(std::move(k), std::move(v));
  });
}

// (q, k_codes, k_scales, v_codes, v_scales, page_table, lengths, sm_scale) -> o
PyObject* kv_cache_attn(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&] {
    Call c("kv_cache_attn", args, nargs, 8);
    const at::Tensor& q0 = c.tensor(0);
    const Cache cache(c, 1);
    const at::Tensor &pages = c.tensor(5), &lengths = c.tensor(6);
    const float scale = (float)c.number(7);
    const int dt = c.float_code(q0);
    const int64_t H = cache.H(), D = cache.D();
    if (q0.dim() != 4 || q0.size(3) != D || H == 0 || q0.size(2) % H)
      raise(PyExc_ValueError, "%s: q must be [B, N, Hq, %lld] with Hq a multiple of %lld; got %s", c.what(), (long long)D,
            (long long)H, shape_of(q0).c_str());
    const int64_t B = q0.size(0), N = q0.size(1), Hq = q0.size(2);
    if (pages.dim() != 2 || pages.size(0) != B || pages.scalar_type() != at::kInt ||
        (pages.size(1) > 1 && pages.stride(1) != 1))
      raise(PyExc_ValueError, "%s: page_table must be int32 [%lld, max_pages] with unit stride along a row", c.what(),
            (long long)B);
    c.index_code(lengths, "lengths", B, false);
    const at::Tensor q = Call::unit(q0);
    at::Tensor o = c.empty({B, N, Hq, D}, q.scalar_type());
    const int64_t strides[6] = {q.stride(0), q.stride(1), q.stride(2), N * Hq * D, Hq * D, D};
    const size_t ws_bytes = entries.query_workspace(4, B, N * (Hq / H), H, D);
    const at::Tensor ws = ws_bytes ? c.empty({(int64_t)ws_bytes}, at::kByte) : at::Tensor();
    const void* qp = q.const_data_ptr();
    void *op = o.mutable_data_ptr(), *wp = ws_bytes ? ws.mutable_data_ptr() : nullptr;
    const Cache::Arrays from = cache.arrays();
    const int32_t *pp = static_cast<const int32_t*>(pages.const_data_ptr()),
                  *lp = static_cast<const int32_t*>(lengths.const_data_ptr());
    const int64_t max_pages = pages.size(1), table_stride = pages.stride(0);
    c.run("b2_kv_cache_attn", [&](void* stream) {
      return entries.kv_cache_attn(qp, op, from.kc, from.ks, from.vc, from.vs, pp, lp, B, N, Hq, max_pages, table_stride,
                                   cache.shape, strides, scale, dt, wp, ws_bytes, stream);
    });
    return THPVariable_Wrap(std::move(o));
  });
}

// (q, k, v, cu_q, cu_k, causal, sm_scale) -> o
PyObject* flash_attn_packed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&] {
    Call c("flash_attn_packed", args, nargs, 7);
    const at::Tensor &q = c.tensor(0), &k = c.tensor(1), &v = c.tensor(2), &cu_q = c.tensor(3), &cu_k = c.tensor(4);
    const int causal = c.truth(5);
    const float scale = (float)c.number(6);
    const int dt = c.float_code(q);
    if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || q.size(2) != k.size(2) || k.size(1) == 0 ||
        q.size(1) % k.size(1))
      raise(PyExc_ValueError, "%s: need q [Tq, Hq, D] and k, v [Tk, Hk, D] with Hq a multiple of Hk; got %s, %s, %s",
            c.what(), shape_of(q).c_str(), shape_of(k).c_str(), shape_of(v).c_str());
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
      raise(PyExc_TypeError, "%s: q, k, v must share a dtype (%s, %s, %s)", c.what(), dtype_of(q), dtype_of(k), dtype_of(v));
    if (cu_q.dim() != 1 || cu_q.size(0) < 1)
      raise(PyExc_ValueError, "%s: cu_q must hold the B + 1 offsets of B sequences", c.what());
    const int64_t B = cu_q.size(0) - 1, Tq = q.size(0), Tk = k.size(0), Hq = q.size(1), Hk = k.size(1), D = q.size(2);
    c.index_code(cu_q, "cu_q", B + 1, false);
    c.index_code(cu_k, "cu_k", B + 1, false);
    at::Tensor o = c.empty({Tq, Hq, D}, q.scalar_type());
    const int64_t strides[12] = {q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
                                 v.stride(0), v.stride(1), v.stride(2), Hq * D,      D,           1};
    const size_t ws_bytes = entries.query_workspace(5, B, Tq, Hq / Hk, 0);
    const at::Tensor ws = ws_bytes ? c.empty({(int64_t)ws_bytes}, at::kByte) : at::Tensor();
    const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
    void *op = o.mutable_data_ptr(), *wp = ws_bytes ? ws.mutable_data_ptr() : nullptr;
    const int32_t *cq = static_cast<const int32_t*>(cu_q.const_data_ptr()),
                  *ck = static_cast<const int32_t*>(cu_k.const_data_ptr());
    c.run("b2_fa_packed", [&](void* stream) {
      return entries.fa_packed(qp, kp, vp, op, cq, ck, B, Tq, Tk, Hq, Hk, D, strides, scale, causal, dt, wp, ws_bytes,
                               stream);
    });
    return THPVariable_Wrap(std::move(o));
  });
}

// torch's mode of a default device, which changes the factories of tensors and nothing here.
PyObject* device_context = nullptr;

// Whether the dispatcher would bring a call with these arguments to the CUDA kernel and
// do nothing else on the way: no mode or tracer is on, no transform is at work, and the
// tensors are what they seem. Everything that would see the call has a key that is
// included for the thread or is the tensor's own, so nothing has to be named.
// `grads`: nor does a result need a gradient.
bool plain(bool grads, PyObject* const* args, Py_ssize_t nargs) {
  using c10::DispatchKey;
  using c10::DispatchKeySet;
  using Modes = at::impl::PythonTorchFunctionTLS;
  if (at::impl::torch_function_mode_enabled())
    for (int64_t i = 0; i < Modes::stack_len(); ++i)
      if ((PyObject*)Py_TYPE(Modes::get_stack_at(i)->ptr(getPyInterpreter())) != device_context) return false;
  constexpr DispatchKeySet always({DispatchKey::BackendSelect, DispatchKey::ADInplaceOrView});
  if (!(c10::impl::tls_local_dispatch_key_set().included_ - always).empty()) return false;
  constexpr DispatchKeySet usual(
      {DispatchKey::CUDA, DispatchKey::ADInplaceOrView, DispatchKey::AutogradCUDA, DispatchKey::AutocastCUDA});
  constexpr DispatchKeySet on_cuda(c10::BackendComponent::CUDABit);
  for (Py_ssize_t i = 0; i < nargs; ++i) {
    PyObject* const a = args[i];
    if (a == Py_None || PyFloat_Check(a) || PyLong_Check(a)) continue;
    if (!THPVariable_CheckExact(a)) {
      if (THPVariable_Check(a)) return false;  // a subclass
      continue;
    }
    const at::Tensor& t = THPVariable_Unpack(a);
    if (t.key_set() - usual != on_cuda) return false;
    if (grads && t.requires_grad() && c10::GradMode::is_enabled()) return false;
  }
  return true;
}
// F where the dispatcher has nothing to do, else NotImplemented. GRADS: F has results of
// its tensors' values (a write into the cache has none).
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), bool GRADS>
PyObject* direct(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  const int is = [&] {
    PyObject* done = guarded([&]() -> PyObject* { return plain(GRADS, args, nargs) ? Py_True : Py_False; });
    return done ? done == Py_True : -1;
  }();
  if (is < 0) return nullptr;
  if (!is) Py_RETURN_NOTIMPLEMENTED;
  return F(self, args, nargs);
}

// The addresses of the C entry points, in the order of Entries, and the class of torch's
// default-device mode.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    void* at[6];
    if (nargs != 7) raise(PyExc_TypeError, "bind: 6 addresses and a class wanted");
    for (int i = 0; i < 6; ++i) {
      at[i] = PyLong_AsVoidPtr(args[i]);
      if (!at[i]) raise(PyErr_Occurred() ? nullptr : PyExc_ValueError, "bind: null address");
    }
    Py_XSETREF(device_context, Py_NewRef(args[6]));
    entries.qk_norm_rope = reinterpret_cast<decltype(entries.qk_norm_rope)>(at[0]);
    entries.kv_cache_write = reinterpret_cast<decltype(entries.kv_cache_write)>(at[1]);
    entries.kv_cache_read = reinterpret_cast<decltype(entries.kv_cache_read)>(at[2]);
    entries.kv_cache_attn = reinterpret_cast<decltype(entries.kv_cache_attn)>(at[3]);
    entries.fa_packed = reinterpret_cast<decltype(entries.fa_packed)>(at[4]);
    entries.query_workspace = reinterpret_cast<decltype(entries.query_workspace)>(at[5]);
    Py_RETURN_NONE;
  });
}

#define B2_METHOD(NAME, F) \
  { NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr }
#define B2_OPERATOR(NAME, GRADS) B2_METHOD(#NAME, NAME), B2_METHOD("direct_" #NAME, (direct<NAME, GRADS>))
PyMethodDef methods[] = {B2_METHOD("bind", bind),           B2_OPERATOR(qk_norm_rope, true),
                         B2_OPERATOR(kv_cache_write, false), B2_OPERATOR(kv_cache_read, true),
                         B2_OPERATOR(kv_cache_attn, true),   B2_OPERATOR(flash_attn_packed, true),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder(void) { return PyModule_Create(&module); }
