// Host path of one layer call (`DualLinear.__call__`, `DualLinear.silu_linear`, `DualLinear.linear`), and of the calls between layers
// (`producer.norm_pack`, `PagedCache.write`, `PagedCache.attention` and the like), as a CPython extension.
//
// A call at decode sizes is bounded by the host: 3.4 us of GPU time at 8 tokens of 896 -> 4864.  Through ctypes and
// torch's Python bindings the host needed 7.3 us a call, of which 2.4 us are the launch itself; the rest was the output
// allocation (1.9 us), the foreign call (0.9 us) and Python bytecode.  Here one C call checks the argument, finds the
// prepared state of the token count, allocates and launches: 4.4 us.
//
// The module holds no state of its own but the addresses of the library's entry points.  It is built against the torch
// that loads it and knows nothing of CUDA beyond the current stream.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <initializer_list>
#include <iterator>
#include <type_traits>

#include "../../include/hygemm.h"

namespace {

decltype(&hg_linear) run_linear = nullptr;
decltype(&hg_linear_silu) run_linear_silu = nullptr;
decltype(&hg_last_error) last_error = nullptr;
decltype(&hg_linear_epilogue) run_linear_epilogue = nullptr;
decltype(&hg_norm) run_norm = nullptr;
decltype(&hg_cache_write) run_cache_write = nullptr;
decltype(&hg_cache_read) run_cache_read = nullptr;
decltype(&hg_attention) run_attention = nullptr;
decltype(&hg_attention_workspace) attention_workspace = nullptr;

PyObject *s_ready, *s_w4, *s_sf4, *s_lo, *s_w8, *s_sf8, *s_hi, *s_low_id, *s_high_id, *s_concurrent, *s_plans, *s_calls;

const char kName[] = "hygemm.ready";

// What calls of one layer with one token count share.  Valid while the layer's six operand tensors still lie where the
// structs say (an attribute may be replaced, and so may the storage behind one) and the schedule ids are the same.
struct Ready {
  PyObject *low_id, *high_id, *problems;              // owned
  void* handle;
  const hg_problem *low, *high;                       // inside `problems`
  int64_t tokens, k, outputs, packed;                 // packed: bytes of the quantised activations
  int fused;                                          // calls quantise inside the GEMM launch: 0 none, 1 all, 2 eager ones
  bool explicit_schedule;                             // no epilogue then
  at::TensorOptions output;
  c10::Device device = c10::Device(c10::kCPU);
};

Ready* ready_of(PyObject* capsule) { return static_cast<Ready*>(PyCapsule_GetPointer(capsule, kName)); }

void destroy(PyObject* capsule) {
  Ready* r = ready_of(capsule);
  if (!r) return;
  for (PyObject* o : {r->low_id, r->high_id, r->problems}) Py_XDECREF(o);
  delete r;
}

// The attributes of a layer.  A call asks for eleven, so they are looked up in the instance's dict directly; one that is
// not there is asked for in the ordinary way.
struct Attributes {
  PyObject *layer, *dict;
  explicit Attributes(PyObject* of) : layer(of), dict(PyObject_GenericGetDict(of, nullptr)) {
    if (!dict) PyErr_Clear();
  }
  ~Attributes() { Py_XDECREF(dict); }
  Attributes(const Attributes&) = delete;
  // A new reference, or null with an error set.
  PyObject* get(PyObject* name) const {
    if (dict) {
      if (PyObject* found = PyDict_GetItemWithError(dict, name)) return Py_NewRef(found);
      if (PyErr_Occurred()) return nullptr;
    }
    return PyObject_GetAttr(layer, name);
  }
};

// True when attribute `name` is `wanted` (the same object, or an equal int).
bool unchanged(const Attributes& layer, PyObject* name, PyObject* wanted) {
  PyObject* now = layer.get(name);
  if (!now) { PyErr_Clear(); return false; }
  bool same = now == wanted;
  if (!same && PyLong_Check(now)) {
    const int equal = PyObject_RichCompareBool(now, wanted, Py_EQ);
    if (equal < 0) PyErr_Clear();
    same = equal == 1;
  }
  Py_DECREF(now);
  return same;
}

// True when attribute `name` is a tensor whose elements start at `data`, `elements` of them (-1: any number).
bool still_at(const Attributes& layer, PyObject* name, const void* data, int64_t elements = -1) {
  PyObject* now = layer.get(name);
  if (!now) { PyErr_Clear(); return false; }
  struct Release { PyObject* o; ~Release() { Py_DECREF(o); } } release{now};   // the tensor's accessors may throw
  if (!THPVariable_Check(now)) return false;
  const at::Tensor& t = THPVariable_Unpack(now);
  return t.const_data_ptr() == data && (elements < 0 || t.numel() == elements);
}

// True for the launch policies that all enqueue the tensor-core launch: False and True, 0 to 3.
bool tensor_core_policy(const Attributes& layer) {
  PyObject* now = layer.get(s_concurrent);
  if (!now) { PyErr_Clear(); return false; }
  bool plain = now == Py_True || now == Py_False;
  if (!plain) {
    PyObject* number = PyNumber_Long(now);
    const long policy = number ? PyLong_AsLong(number) : -1;
    PyErr_Clear();
    Py_XDECREF(number);
    plain = policy >= HG_POLICY_SERIAL && policy < HG_POLICY_GEMV_PAIR1;
  }
  Py_DECREF(now);
  return plain;
}

bool operands_unchanged(const Attributes& layer, const hg_problem& low, const hg_problem& high) {
  return still_at(layer, s_w4, low.weight) && still_at(layer, s_sf4, low.weight_scales) && still_at(layer, s_lo, low.ids, low.rows) &&
         still_at(layer, s_w8, high.weight) && still_at(layer, s_sf8, high.weight_scales) && still_at(layer, s_hi, high.ids, high.rows);
}

// The prepared state of a call, a new reference; null without an error when the call is not a prepared, ordinary one.
PyObject* find(const Attributes& layer, int64_t tokens) {
  PyObject* plans = layer.get(s_plans);
  if (!plans) return nullptr;
  const int planned = PyObject_IsTrue(plans);
  Py_DECREF(plans);
  if (planned) return nullptr;
  PyObject* all = layer.get(s_ready);
  if (!all) return nullptr;
  PyObject* capsule = nullptr;
  PyObject* key = PyLong_FromLongLong(tokens);
  if (key && PyDict_Check(all)) {
    capsule = PyDict_GetItemWithError(all, key);
    Py_XINCREF(capsule);
  }
  Py_XDECREF(key);
  Py_DECREF(all);
  return capsule;
}

bool count_call(const Attributes& layer, int64_t tokens) {
  PyObject* calls = layer.get(s_calls);
  if (!calls) return false;
  bool ok = false;
  PyObject* key = PyLong_FromLongLong(tokens);
  if (key && PyDict_Check(calls)) {
    PyObject* old = PyDict_GetItemWithError(calls, key);
    if (old || !PyErr_Occurred()) {
      PyObject* sum = PyLong_FromLongLong((old ? PyLong_AsLongLong(old) : 0) + 1);
      ok = sum && !PyErr_Occurred() && PyDict_SetItem(calls, key, sum) == 0;
      Py_XDECREF(sum);
    }
  }
  Py_XDECREF(key);
  Py_DECREF(calls);
  return ok;
}

// The interpreter lock given up for a scope, also when it is left by an exception.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// Operands of `DualLinear.linear`: null, or what an epilogue takes.
struct Added { const at::Tensor *bias, *residual; int activation; };

// A gradient would be asked of it, or it carries a tangent of forward mode: the calls have neither, and Python says so.
bool differentiated(const at::Tensor& t) {
  return (c10::GradMode::is_enabled() && t.requires_grad()) || (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}
bool sixteen_bits(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
// A tensor without memory (under tracing, say) would be taken for an operand that is not there.
bool held(const at::Tensor& t) { return t.const_data_ptr() || !t.numel(); }
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && held(t); }
int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? HG_DTYPE_BF16 : HG_DTYPE_F16; }

PyObject* forward_checked(PyObject* self, const at::Tensor& x, long math, const Added* added = nullptr) {
  const Attributes layer(self);
  const bool swiglu = math >= 0;
  if (x.dim() != 2) Py_RETURN_NONE;
  const auto type = x.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
  const int64_t tokens = x.size(0);
  PyObject* capsule = find(layer, tokens);
  if (!capsule) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  struct Release { PyObject* o; ~Release() { Py_DECREF(o); } } release{capsule};
  const Ready* r = ready_of(capsule);
  if (!r) return nullptr;
  if (x.size(1) != (swiglu ? 2 * r->k : r->k) || x.device() != r->device || !x.is_contiguous() ||
      !unchanged(layer, s_low_id, r->low_id) || !unchanged(layer, s_high_id, r->high_id) || !tensor_core_policy(layer) ||
      !operands_unchanged(layer, *r->low, *r->high))
    Py_RETURN_NONE;
  hg_epilogue epilogue{};
  if (added) {
    const auto type = r->output.dtype().toScalarType();
    if (r->explicit_schedule || differentiated(x)) Py_RETURN_NONE;
    if (const at::Tensor* bias = added->bias) {
      if (bias->device() != r->device || bias->scalar_type() != type || bias->dim() != 1 || bias->size(0) != r->outputs || !bias->is_contiguous() || !held(*bias) || differentiated(*bias))
        Py_RETURN_NONE;
      epilogue.bias = bias->const_data_ptr();
    }
    if (const at::Tensor* residual = added->residual) {
      if (residual->device() != r->device || residual->scalar_type() != type || residual->dim() != 2 || residual->size(0) != r->tokens ||
          residual->size(1) != r->outputs || residual->stride(1) != 1 || !held(*residual) || differentiated(*residual))
        Py_RETURN_NONE;
      epilogue.residual = residual->const_data_ptr();
      epilogue.residual_stride = residual->stride(0);
    }
    epilogue.activation = added->activation;
  }
  const int dtype = type == at::kBFloat16 ? HG_DTYPE_BF16 : HG_DTYPE_F16;
  at::Tensor y;
  int status;
  // A layer on another device than the current one; plain calls leave that to their caller.
  c10::cuda::OptionalCUDAGuard elsewhere;
  if (added) elsewhere.set_device(r->device);
  {
    // Without the interpreter lock, as torch's own bindings: an allocator may wait for a thread that wants it (one whose
    // callbacks are Python functions, as of a pool that a serving engine puts to sleep), or for the device.
    const Unlocked unlocked;
    // Fresh tensors per call: under CUDA-graph capture the graph's pool owns them.
    y = at::empty({r->tokens, r->outputs}, r->output);
    const bool in_gemm = !swiglu && (r->fused == 1 || (r->fused == 2 && c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None));
    const int64_t bytes = in_gemm ? 0 : r->packed;
    // Scratch that nobody else sees: the allocator itself, for the same stream and with the same lifetime, without a tensor round it
    // (0.3 us of a call of two launches, of which the host then needs 7.3 to 7.8 us).
    c10::DataPtr workspace;
    if (bytes) {
      const c10::cuda::CUDAGuard guard(r->device);
      workspace = c10::cuda::CUDACachingAllocator::get()->allocate(size_t(bytes));
    }
    const void* in = x.const_data_ptr();
    void* out = y.mutable_data_ptr();
    void* scratch = workspace.get();
    void* stream = c10::cuda::getCurrentCUDAStream(r->device.index()).stream();
    status = added ? run_linear_epilogue(r->handle, r->low, r->high, in, dtype, scratch, out, &epilogue, stream)
             : swiglu ? run_linear_silu(r->handle, r->low, r->high, in, dtype, int(math), scratch, out, stream)
                    : run_linear(r->handle, r->low, r->high, in, dtype, scratch, out, stream);
  }
  if (status) return PyErr_SetString(PyExc_RuntimeError, last_error()), nullptr;
  if (!count_call(layer, tokens)) return nullptr;
  return THPVariable_Wrap(std::move(y));
}

// Runs `body`, an exception of C++ becomes one of Python.
template <typename Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* type = PyObject_GetAttrString(PyImport_AddModule("torch"), "OutOfMemoryError");
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// forward(layer, x, math): the layer on `x`, of SwiGLU of `x` when math >= 0.  None: not an ordinary call, or the first one.
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) return PyErr_SetString(PyExc_TypeError, "forward(layer, x, math)"), nullptr;
  if (!run_linear || !THPVariable_Check(args[1])) Py_RETURN_NONE;
  const long math = PyLong_AsLong(args[2]);
  if (math == -1 && PyErr_Occurred()) return nullptr;
  return guarded([&] { return forward_checked(args[0], THPVariable_Unpack(args[1]), math); });
}

// A tensor or None; false: something else.
bool optional_tensor(PyObject* o, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = &THPVariable_Unpack(o);
  return true;
}

// forward_epilogue(layer, x, bias, activation, residual): as forward, with what is added (`activation` a number).
PyObject* forward_epilogue(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) return PyErr_SetString(PyExc_TypeError, "forward_epilogue(layer, x, bias, activation, residual)"), nullptr;
  Added added{};
  if (!run_linear_epilogue || !THPVariable_Check(args[1]) || !optional_tensor(args[2], &added.bias) || !optional_tensor(args[4], &added.residual)) Py_RETURN_NONE;
  const long activation = PyLong_AsLong(args[3]);
  if (activation == -1 && PyErr_Occurred()) return nullptr;
  added.activation = int(activation);
  return guarded([&] { return forward_checked(args[0], THPVariable_Unpack(args[1]), -1, &added); });
}

// ---- calls between layers: None where an argument is not an ordinary one; Python then says what is wrong, or makes the call ----

int64_t scale_bytes(int64_t rows, int64_t k) { return (rows + 127) / 128 * (k / 128) * 512; }
// A result on t's device, which is the current one.  Past the dispatcher a tensor costs 0.3 us less (a norm call with three 5.6 -> 4.9 us).
at::Tensor result(at::IntArrayRef size, at::ScalarType type, const at::Tensor& t) { return at::Tensor(at::detail::empty_cuda(size, type, t.device(), std::nullopt)); }
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
bool failed(int status) {
  if (status) PyErr_SetString(PyExc_RuntimeError, last_error());
  return status != 0;
}
// New references of the tuple's items.
PyObject* tuple_of(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New(Py_ssize_t(items.size()));
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    if (!t || !o) {
      Py_XDECREF(o);
      if (t && !o) Py_CLEAR(t);
    } else {
      PyTuple_SET_ITEM(t, i, o);
    }
    ++i;
  }
  return t;
}

// A 16-bit matrix like x: contiguous rows aligned to 16 bytes.
bool rows_like(const at::Tensor& t, const at::Tensor& x) {
  return t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.dim() == 2 && t.size(0) == x.size(0) && t.size(1) == x.size(1) &&
         t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) % 8 == 0) && aligned(t) && !differentiated(t);
}
bool vector_like(const at::Tensor& t, const at::Tensor& x) {
  return t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.dim() == 1 && t.size(0) == x.size(1) && t.is_contiguous() && aligned(t) && !differentiated(t);
}

// norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, packed)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return PyErr_SetString(PyExc_TypeError, "norm takes nine arguments"), nullptr;
  const at::Tensor *residual, *gate, *post;
  if (!run_norm || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !optional_tensor(args[3], &residual) || !optional_tensor(args[4], &gate) ||
      !optional_tensor(args[6], &post))
    Py_RETURN_NONE;
  hg_norm_call call{};
  call.eps = float(PyFloat_AsDouble(args[2]));
  call.scale = float(PyFloat_AsDouble(args[5]));
  call.post_eps = args[7] == Py_None ? call.eps : float(PyFloat_AsDouble(args[7]));
  if (PyErr_Occurred()) return nullptr;
  const bool packed = args[8] == Py_True;
  return guarded([&]() -> PyObject* {
    const at::Tensor &x = THPVariable_Unpack(args[0]), &weight = THPVariable_Unpack(args[1]);
    if (!x.is_cuda() || !sixteen_bits(x) || x.dim() != 2) Py_RETURN_NONE;
    const int64_t rows = x.size(0), k = x.size(1);
    if (!rows || rows > 0x7fffff00 || !k || k > 32768 || k % (packed ? 128 : 8) || !rows_like(x, x) || !vector_like(weight, x) || (residual && !rows_like(*residual, x)) ||
        (post && !vector_like(*post, x)))
      Py_RETURN_NONE;
    if (gate) {
      if (gate->dim() == 1 ? !vector_like(*gate, x) : !rows_like(*gate, x)) Py_RETURN_NONE;   // [rows,1]: by way of Python
      call.gate = gate->const_data_ptr();
      call.gate_stride = gate->dim() == 2 ? gate->stride(0) : 0;
    }
    const bool changed = residual || gate || post || call.scale != 1.f;
    at::Tensor codes, scales, stream;
    int status;
    {
      const Unlocked unlocked;
      const c10::cuda::CUDAGuard guard(x.device());
      if (changed) stream = result({rows, k}, x.scalar_type(), x);
      codes = result({rows, k}, packed ? at::kByte : x.scalar_type(), x);
      if (packed) {
        scales = result({scale_bytes(rows, k)}, at::kByte, x);
        call.codes = codes.mutable_data_ptr();
        call.scales = scales.mutable_data_ptr();
      } else {
        call.normed = codes.mutable_data_ptr();
      }
      call.x = x.const_data_ptr();
      call.x_stride = rows > 1 ? x.stride(0) : 0;
      call.weight = weight.const_data_ptr();
      if (residual) {
        call.residual = residual->const_data_ptr();
        call.residual_stride = rows > 1 ? residual->stride(0) : 0;
      }
      if (rows == 1) call.gate_stride = 0;
      if (post) call.post_weight = post->const_data_ptr();
      if (changed) call.stream_out = stream.mutable_data_ptr();
      call.rows = int(rows);
      call.k = int(k);
      status = run_norm(&call, dtype_of(x), stream_of(x));
    }
    if (failed(status)) return nullptr;
    PyObject* const h = changed ? THPVariable_Wrap(std::move(stream)) : Py_NewRef(args[0]);
    return packed ? tuple_of({THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)), h}) : tuple_of({THPVariable_Wrap(std::move(codes)), h});
  });
}

// A cache as the library takes it; false: `data` is not one.
bool cache_of(const at::Tensor& data, long page_size, long head_dim, hg_cache* cache) {
  if (!data.is_cuda() || data.scalar_type() != at::kByte || data.dim() != 3 || !data.is_contiguous() || !held(data) || data.size(0) > 0x7fffffff || data.size(1) > 0x7fffffff ||
      page_size <= 0 || page_size > 1024 || (head_dim != 64 && head_dim != 128) || data.size(2) != page_size * (2 * head_dim + head_dim / 16))
    return false;
  *cache = hg_cache{data.data_ptr(), int(data.size(0)), int(data.size(1)), int(page_size), int(head_dim)};
  return true;
}
bool slots_of(const at::Tensor& slots, const at::Tensor& data) {
  return slots.device() == data.device() && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous() && held(slots) && slots.size(0) > 0 && slots.size(0) <= 0x7fffffff;
}

// cache_write(data, page_size, head_dim, k, v, slots): True when done
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) return PyErr_SetString(PyExc_TypeError, "cache_write takes six arguments"), nullptr;
  for (int i : {0, 3, 4, 5})
    if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
  const long page_size = PyLong_AsLong(args[1]), head_dim = PyLong_AsLong(args[2]);
  if (!run_cache_write || PyErr_Occurred()) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  return guarded([&]() -> PyObject* {
    const at::Tensor &data = THPVariable_Unpack(args[0]), &k = THPVariable_Unpack(args[3]), &v = THPVariable_Unpack(args[4]), &slots = THPVariable_Unpack(args[5]);
    hg_cache cache;
    if (!cache_of(data, page_size, head_dim, &cache) || !slots_of(slots, data)) Py_RETURN_NONE;
    int64_t strides[4];
    for (int i : {0, 1}) {
      const at::Tensor& t = i ? v : k;
      if (t.device() != data.device() || !sixteen_bits(t) || t.scalar_type() != k.scalar_type() || t.dim() != 3 || t.size(0) != slots.size(0) ||
          t.size(1) != cache.kv_heads || t.size(2) != head_dim || t.stride(2) != 1 || t.stride(0) % 4 || t.stride(1) % 4 ||
          reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 8 || !held(t) || differentiated(t))
        Py_RETURN_NONE;
      strides[2 * i] = t.stride(0);
      strides[2 * i + 1] = t.stride(1);
    }
    int status;
    {
      const Unlocked unlocked;
      const c10::cuda::CUDAGuard guard(data.device());
      status = run_cache_write(&cache, k.const_data_ptr(), v.const_data_ptr(), strides, static_cast<const int64_t*>(slots.const_data_ptr()), int(slots.size(0)),
                               dtype_of(k), stream_of(data));
    }
    return failed(status) ? nullptr : Py_NewRef(Py_True);
  });
}

// cache_read(data, page_size, head_dim, slots, bf16): (k, v)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) return PyErr_SetString(PyExc_TypeError, "cache_read takes five arguments"), nullptr;
  if (!run_cache_read || !THPVariable_Check(args[0]) || !THPVariable_Check(args[3])) Py_RETURN_NONE;
  const long page_size = PyLong_AsLong(args[1]), head_dim = PyLong_AsLong(args[2]), bf16 = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &data = THPVariable_Unpack(args[0]), &slots = THPVariable_Unpack(args[3]);
    hg_cache cache;
    if (!cache_of(data, page_size, head_dim, &cache) || !slots_of(slots, data)) Py_RETURN_NONE;
    at::Tensor k, v;
    int status;
    {
      const Unlocked unlocked;
      const c10::cuda::CUDAGuard guard(data.device());
      const auto type = bf16 ? at::kBFloat16 : at::kHalf;
      k = result({slots.size(0), cache.kv_heads, head_dim}, type, data);
      v = result({slots.size(0), cache.kv_heads, head_dim}, type, data);
      status = run_cache_read(&cache, k.mutable_data_ptr(), v.mutable_data_ptr(), static_cast<const int64_t*>(slots.const_data_ptr()), int(slots.size(0)),
                              bf16 ? HG_DTYPE_BF16 : HG_DTYPE_F16, stream_of(data));
    }
    return failed(status) ? nullptr : tuple_of({THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v))});
  });
}

// attention(data, page_size, head_dim, q, table, lengths, scale, window, lse, packed): out, (out, lse), (codes, scales) or (codes, scales, lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 10) return PyErr_SetString(PyExc_TypeError, "attention takes ten arguments"), nullptr;
  for (int i : {0, 3, 4, 5})
    if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
  if (!run_attention || !attention_workspace) Py_RETURN_NONE;
  const long page_size = PyLong_AsLong(args[1]), head_dim = PyLong_AsLong(args[2]);
  hg_attention_call call{};
  const double scale = args[6] == Py_None ? 0 : PyFloat_AsDouble(args[6]);
  const long long window = PyLong_AsLongLong(args[7]);
  const int with_lse = PyObject_IsTrue(args[8]);
  const bool packed = args[9] == Py_True;
  if (PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &data = THPVariable_Unpack(args[0]), &q = THPVariable_Unpack(args[3]), &table = THPVariable_Unpack(args[4]), &lengths = THPVariable_Unpack(args[5]);
    hg_cache cache;
    if (!cache_of(data, page_size, head_dim, &cache) || q.device() != data.device() || !sixteen_bits(q) || q.dim() != 3 || q.size(2) != head_dim || !q.size(0) ||
        !q.size(1) || q.size(1) % cache.kv_heads || q.stride(2) != 1 || (q.size(1) > 1 && q.stride(1) != head_dim) || (q.size(0) > 1 && q.stride(0) % 8) ||
        !aligned(q) || differentiated(q) || (packed && q.size(1) * head_dim % 128) || q.size(0) > 0x7fffffff || q.size(1) > 0x7fffff)
      Py_RETURN_NONE;
    const int64_t seqs = q.size(0), heads = q.size(1);
    if (table.device() != data.device() || table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != seqs || (table.size(1) > 1 && table.stride(1) != 1) ||
        lengths.device() != data.device() || lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != seqs || !lengths.is_contiguous() || !held(table) || !held(lengths))
      Py_RETURN_NONE;
    const int64_t positions = table.size(1) * page_size;
    if (positions > (1 << 30) || window < 0) Py_RETURN_NONE;
    at::Tensor out, scales, lse;
    int status;
    {
      const Unlocked unlocked;
      const c10::cuda::CUDAGuard guard(data.device());
      call.q = q.const_data_ptr();
      call.q_stride = seqs > 1 ? q.stride(0) : 0;
      call.table = static_cast<const int*>(table.const_data_ptr());
      call.table_stride = table.stride(0);
      call.lengths = static_cast<const int*>(lengths.const_data_ptr());
      call.seqs = int(seqs);
      call.heads = int(heads);
      call.table_width = int(table.size(1));
      call.window = window >= positions ? 0 : int(window);
      call.scale = args[6] == Py_None ? float(head_dim == 64 ? 0.125 : 0.08838834764831845) : float(scale);
      const int64_t bytes = attention_workspace(&cache, call.seqs, call.heads, call.table_width, call.window);
      c10::DataPtr workspace;
      status = bytes < 0 ? -1 : 0;
      if (!status) {
        if (packed) {
          out = result({seqs, heads * head_dim}, at::kByte, q);
          scales = result({scale_bytes(seqs, heads * head_dim)}, at::kByte, q);
          call.codes = out.mutable_data_ptr();
          call.scales = scales.mutable_data_ptr();
        } else {
          out = result({seqs, heads, head_dim}, q.scalar_type(), q);
          call.out = out.mutable_data_ptr();
        }
        if (with_lse) {
          lse = result({seqs, heads}, at::kFloat, q);
          call.lse = static_cast<float*>(lse.mutable_data_ptr());
        }
        if (bytes) workspace = c10::cuda::CUDACachingAllocator::get()->allocate(size_t(bytes));
        call.workspace = workspace.get();
        status = run_attention(&cache, &call, dtype_of(q), stream_of(data));
      }
    }
    if (failed(status)) return nullptr;
    PyObject* const first = THPVariable_Wrap(std::move(out));
    if (!packed && !with_lse) return first;
    if (!packed) return tuple_of({first, THPVariable_Wrap(std::move(lse))});
    if (!with_lse) return tuple_of({first, THPVariable_Wrap(std::move(scales))});
    return tuple_of({first, THPVariable_Wrap(std::move(scales)), THPVariable_Wrap(std::move(lse))});
  });
}

// prepare(layer, tokens, handle, low, high, problems, y, packed, fused): the state `forward` looks up.
// `low` and `high` are addresses of the two structs that `problems` keeps alive, `y` is a tensor like the output.
PyObject* prepare(PyObject*, PyObject* args) {
  PyObject *layer, *problems, *y;
  long long tokens, packed;
  int fused;
  unsigned long long handle, low, high;
  if (!PyArg_ParseTuple(args, "OLKKKOOLi", &layer, &tokens, &handle, &low, &high, &problems, &y, &packed, &fused)) return nullptr;
  if (!THPVariable_Check(y)) return PyErr_SetString(PyExc_TypeError, "prepare: y must be a tensor"), nullptr;
  auto* r = new Ready{};
  r->problems = Py_NewRef(problems);
  PyObject* capsule = PyCapsule_New(r, kName, destroy);
  if (!capsule) return nullptr;
  if (!(r->low_id = PyObject_GetAttr(layer, s_low_id)) || !(r->high_id = PyObject_GetAttr(layer, s_high_id))) return Py_DECREF(capsule), nullptr;
  const at::Tensor& like = THPVariable_Unpack(y);
  r->handle = reinterpret_cast<void*>(uintptr_t(handle));
  r->low = reinterpret_cast<const hg_problem*>(uintptr_t(low));
  r->high = reinterpret_cast<const hg_problem*>(uintptr_t(high));
  r->tokens = tokens;
  r->outputs = like.size(1);
  r->k = r->low->k;
  r->packed = packed;
  r->fused = fused;
  const auto is_zero = [](PyObject* id) { return PyObject_IsTrue(id) == 0; };
  r->explicit_schedule = !is_zero(r->low_id) || !is_zero(r->high_id);
  PyErr_Clear();
  r->device = like.device();
  r->output = at::TensorOptions().dtype(like.scalar_type()).device(like.device());
  return capsule;
}

// bind(hg_linear, hg_linear_silu, hg_last_error, ...): addresses in the loaded library.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long at[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", &at[0], &at[1], &at[2], &at[3], &at[4], &at[5], &at[6], &at[7], &at[8])) return nullptr;
  const auto set = [](auto& function, unsigned long long address) { function = reinterpret_cast<std::decay_t<decltype(function)>>(uintptr_t(address)); };
  set(run_linear, at[0]);
  set(run_linear_silu, at[1]);
  set(last_error, at[2]);
  set(run_linear_epilogue, at[3]);
  set(run_norm, at[4]);
  set(run_cache_write, at[5]);
  set(run_cache_read, at[6]);
  set(run_attention, at[7]);
  set(attention_workspace, at[8]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"forward_epilogue", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward_epilogue)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm)), METH_FASTCALL, nullptr},
    {"cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_write)), METH_FASTCALL, nullptr},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_read)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"prepare", prepare, METH_VARARGS, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hygemm_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hygemm_host() {
  PyObject** names[] = {&s_ready, &s_w4, &s_sf4, &s_lo, &s_w8, &s_sf8, &s_hi, &s_low_id, &s_high_id, &s_concurrent, &s_plans, &s_calls};
  const char* text[] = {"_ready", "w4", "sf4", "lo", "w8", "sf8", "hi", "low_id", "high_id", "concurrent", "plans", "calls"};
  for (size_t i = 0; i < std::size(names); ++i)
    if (!(*names[i] = PyUnicode_InternFromString(text[i]))) return nullptr;
  return PyModule_Create(&module);
}
