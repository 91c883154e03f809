// Host path of QuantizedLinear, and of the 8-bit integer operators and block norms, as a CPython extension (tilus_b200._native): argument checks, output and
// workspace tensors, stream lookup and the call into libb200q, in one native function per call.
//
// A decode call occupies the GPU for 5..15 us, so a program that calls its layers one by one is bound by
// whatever the host spends per call.  The same steps written in Python around ctypes took 14 us (measured
// on M = 1, K = N = 8192, where the kernel takes 10.6 us); here they take about a third of that.
// The functions are entered through METH_FASTCALL and touch tensors through the C++ API; the library is
// called through addresses handed over by `bind`, so that whichever build _lib.load() opened is used.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/b200q.h"

namespace {

typedef decltype(&b200q_gemm) GemmFn;
typedef decltype(&b200q_gemm_host) GemmHostFn;
typedef decltype(&b200q_gemm_swiglu_cast) GemmCastFn;
typedef decltype(&b200q_workspace_bytes) WorkspaceFn;

GemmFn g_gemm = nullptr;
GemmHostFn g_gemm_host = nullptr;
GemmCastFn g_gemm_cast = nullptr;
WorkspaceFn g_workspace_bytes = nullptr;
PyObject* g_raise_status = nullptr;       // _lib.check
PyObject* g_raise_unsupported = nullptr;  // callable(M, N, K)

// what a layer's calls have in common: (dtype code, zero point, group size, in_features, out_features)
struct Layer { int code, zero_point, group, K, N; };

bool parse_layer(PyObject* t, Layer* l) {
  if (!PyTuple_CheckExact(t) || PyTuple_GET_SIZE(t) != 5) {
    PyErr_SetString(PyExc_TypeError, "layer constants are a tuple of five integers");
    return false;
  }
  int* dst[5] = {&l->code, &l->zero_point, &l->group, &l->K, &l->N};
  for (int i = 0; i < 5; ++i) *dst[i] = (int)PyLong_AsLong(PyTuple_GET_ITEM(t, i));
  return !PyErr_Occurred();
}

const at::Tensor* as_tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a torch.Tensor", what);
    return nullptr;
  }
  return &THPVariable_Unpack(o);
}

// activation dtype tag of the C ABI, -1 when it is neither float16 nor bfloat16
int act_code(at::ScalarType t) { return t == at::kHalf ? 0 : (t == at::kBFloat16 ? 1 : -1); }

bool check_weights(const at::Tensor& qw, const at::Tensor& scales, const c10::Device& dev) {
  if (qw.device() == dev && scales.device() == dev) return true;
  PyErr_SetString(PyExc_ValueError, "the layer's weights and the activations must be on one CUDA device");
  return false;
}

// Per (device, stream) buffers, grown on demand.  The kernels leave a workspace zeroed, so it is cleared
// only when it is (re)allocated; one stream's calls run one after the other, so they share one.  The
// staging pair holds the activations and results of host calls: decode batches (whose kernel fetches
// its own activations, so that consecutive calls overlap) have a pair of their own, so that a larger
// batch in between does not make the next decode call wait for it.
// A buffer that has become too small is replaced by one of at least twice its size, and kept: a captured graph may
// name its address, and b200q_gemm_host remembers staging buffers by theirs.  What is kept is less than what replaced it.
struct StreamBuffers {
  int device;
  cudaStream_t stream;
  at::Tensor workspace;
  at::Tensor staging[2][2];
  std::vector<at::Tensor> superseded;
  std::mutex host_call;  // a host call is several operations on one staging pair: one thread's at a time
};
std::mutex g_mutex;
std::vector<std::unique_ptr<StreamBuffers>>& pool() {
  static auto* p = new std::vector<std::unique_ptr<StreamBuffers>>();  // outlives the interpreter's teardown
  return *p;
}
StreamBuffers& buffers_of(int device, cudaStream_t stream) {  // g_mutex held; the entry stays where it is
  for (const auto& b : pool())
    if (b->device == device && b->stream == stream) return *b;
  pool().push_back(std::make_unique<StreamBuffers>());
  pool().back()->device = device;
  pool().back()->stream = stream;
  return *pool().back();
}
// Device memory for b's stream, which is b's device's current stream, zeroed if asked for.  While the stream is being
// captured the allocation and the zeroing are not part of the capture: memory of the graph's own pool would be cleared by that
// graph's replays only, and not before the first of them.  They take place on a stream of their own then, at once.
at::Tensor allocate(const StreamBuffers& b, int64_t size, bool zero) {
  const c10::Device dev(at::kCUDA, (c10::DeviceIndex)b.device);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(b.stream, &capture) != cudaSuccess) (void)cudaGetLastError();  // (the launch will say what is wrong)
  if (capture == cudaStreamCaptureStatusNone) {
    at::Tensor t = at::detail::empty_cuda({size}, at::kByte, dev, std::nullopt);
    if (zero) C10_CUDA_CHECK(cudaMemsetAsync(t.mutable_data_ptr(), 0, (size_t)size, b.stream));
    return t;
  }
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  static auto* sides = new std::vector<std::pair<int, cudaStream_t>>();  // per device; g_mutex held
  cudaStream_t side = nullptr;
  for (const auto& s : *sides)
    if (s.first == b.device) side = s.second;
  if (side == nullptr) {
    C10_CUDA_CHECK(cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking));
    sides->emplace_back(b.device, side);
  }
  const c10::cuda::CUDAStreamGuard guard(c10::cuda::getStreamFromExternal(side, dev.index()));
  at::Tensor t = at::detail::empty_cuda({size}, at::kByte, dev, std::nullopt);
  if (zero) C10_CUDA_CHECK(cudaMemsetAsync(t.mutable_data_ptr(), 0, (size_t)size, side));
  C10_CUDA_CHECK(cudaStreamSynchronize(side));
  return t;
}
// One of b's buffers with room for `need` bytes; g_mutex held, b's device current and b's stream its current stream.
at::Tensor with_room(StreamBuffers& b, at::Tensor& buffer, size_t need, bool zero) {
  const size_t have = buffer.defined() ? (size_t)buffer.numel() : 0;
  if (have < need || !buffer.defined()) {
    at::Tensor larger = allocate(b, (int64_t)std::max(need, 2 * have), zero);
    if (buffer.defined()) b.superseded.push_back(std::move(buffer));
    buffer = std::move(larger);
  }
  return buffer;
}
// `device` is current and `stream` its current stream
at::Tensor workspace_of(int device, cudaStream_t stream, size_t need) {
  std::lock_guard<std::mutex> lock(g_mutex);
  StreamBuffers& b = buffers_of(device, stream);
  return with_room(b, b.workspace, std::max(need, (size_t)1 << 20), true);
}

// Library calls run without the interpreter lock (as through ctypes): a launch into a full queue blocks, and a copy to
// pageable memory waits for everything queued before it.
class NoGil {
 public:
  NoGil() : state_(PyEval_SaveThread()) {}
  ~NoGil() { PyEval_RestoreThread(state_); }
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;

 private:
  PyThreadState* state_;
};

PyObject* raise_status(int st) {
  PyObject* r = PyObject_CallFunction(g_raise_status, "i", st);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "b200q call failed");
  return nullptr;
}
PyObject* raise_unsupported(int M, int N, int K) {
  PyObject* r = PyObject_CallFunction(g_raise_unsupported, "iii", M, N, K);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "no kernel for this shape");
  return nullptr;
}

// activations as rows of K values: the tensor itself, or reshaped to two dimensions
bool as_rows(const at::Tensor& x, int K, at::Tensor* rows) {
  if (x.dim() == 0 || x.size(-1) != K) {
    PyErr_Format(PyExc_ValueError, "expected %d input features, got %lld", K,
                 x.dim() ? (long long)x.size(-1) : 1LL);
    return false;
  }
  *rows = x.dim() == 2 ? x : x.reshape({-1, (int64_t)K});
  return true;
}

// linear(x, quantized_weight, scales, layer) -> [..., out_features]
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4) { PyErr_SetString(PyExc_TypeError, "linear takes 4 arguments"); return nullptr; }
  const at::Tensor* x = as_tensor(args[0], "activations");
  const at::Tensor* qw = as_tensor(args[1], "quantized_weight");
  const at::Tensor* scales = as_tensor(args[2], "scales");
  Layer l;
  if (!x || !qw || !scales || !parse_layer(args[3], &l)) return nullptr;
  at::Tensor rows;
  if (!as_rows(*x, l.K, &rows)) return nullptr;
  if (!rows.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "QuantizedLinear needs CUDA tensors (there is no CPU path)");
    return nullptr;
  }
  const at::ScalarType dtype = scales->scalar_type();
  const int act = act_code(dtype);
  if (rows.scalar_type() != dtype || act < 0 || rows.stride(1) != 1) {
    PyErr_Format(PyExc_TypeError, "activations must be %s with unit inner stride", c10::toString(dtype));
    return nullptr;
  }
  const c10::Device dev = rows.device();
  if (!check_weights(*qw, *scales, dev)) return nullptr;
  const int M = (int)rows.size(0);
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor out = at::detail::empty_cuda({(int64_t)M, (int64_t)l.N}, dtype, dev, std::nullopt);
  if (M > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const size_t need = g_workspace_bytes(M, l.N, l.K, l.code, l.zero_point, l.group);
    if (need == 0) return raise_unsupported(M, l.N, l.K);
    const at::Tensor ws = workspace_of(dev.index(), stream, need);
    const void *a = rows.const_data_ptr(), *bq = qw->const_data_ptr(), *sc = scales->const_data_ptr();
    void *c = out.mutable_data_ptr(), *w = ws.mutable_data_ptr();
    const int lda = (int)rows.stride(0);
    int st;
    {
      const NoGil unlocked;
      st = g_gemm(a, lda, bq, sc, c, l.N, M, l.N, l.K, l.code, l.zero_point, l.group, act, w, (size_t)ws.numel(), stream);
    }
    if (st != 0) return raise_status(st);
  }
  if (x->dim() != 2) {
    std::vector<int64_t> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = l.N;
    out = out.reshape(shape);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// linear_host(x_host, out_host, quantized_weight, scales, layer) -> out_host
PyObject* linear_host(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) { PyErr_SetString(PyExc_TypeError, "linear_host takes 5 arguments"); return nullptr; }
  const at::Tensor* x = as_tensor(args[0], "x_host");
  const at::Tensor* out = as_tensor(args[1], "out_host");
  const at::Tensor* qw = as_tensor(args[2], "quantized_weight");
  const at::Tensor* scales = as_tensor(args[3], "scales");
  Layer l;
  if (!x || !out || !qw || !scales || !parse_layer(args[4], &l)) return nullptr;
  if (x->is_cuda() || out->is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "forward_host takes host tensors (use forward for device tensors)");
    return nullptr;
  }
  const at::ScalarType dtype = scales->scalar_type();
  const int act = act_code(dtype);
  if (x->scalar_type() != dtype || out->scalar_type() != dtype || act < 0) {
    PyErr_Format(PyExc_TypeError, "activations and result must be %s", c10::toString(dtype));
    return nullptr;
  }
  if (x->dim() != 2 || x->stride(1) != 1 || x->size(1) != l.K) {
    PyErr_Format(PyExc_ValueError, "x_host must be [M, %d] with unit inner stride", l.K);
    return nullptr;
  }
  const int M = (int)x->size(0);
  if (out->dim() != 2 || out->stride(1) != 1 || out->size(0) != M || out->size(1) != l.N) {
    PyErr_Format(PyExc_ValueError, "out_host must be [%d, %d] with unit inner stride", M, l.N);
    return nullptr;
  }
  const c10::Device dev = qw->device();
  if (!dev.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "QuantizedLinear needs its weights on a CUDA device (there is no CPU path)");
    return nullptr;
  }
  if (!check_weights(*qw, *scales, dev)) return nullptr;
  if (M > 0) {
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const size_t need = g_workspace_bytes(M, l.N, l.K, l.code, l.zero_point, l.group);
    if (need == 0) return raise_unsupported(M, l.N, l.K);
    const at::Tensor ws = workspace_of(dev.index(), stream, need);
    at::Tensor sa, sc;
    StreamBuffers* buffers;
    {
      std::lock_guard<std::mutex> lock(g_mutex);
      buffers = &buffers_of(dev.index(), stream);
      at::Tensor* s = buffers->staging[M <= 16 ? 1 : 0];
      sa = with_room(*buffers, s[0], (size_t)M * l.K * 2, false);
      sc = with_room(*buffers, s[1], (size_t)M * l.N * 2, false);
    }
    const void *a = x->const_data_ptr(), *bq = qw->const_data_ptr(), *scp = scales->const_data_ptr();
    void *c = out->mutable_data_ptr(), *a_stage = sa.mutable_data_ptr(), *c_stage = sc.mutable_data_ptr();
    void* w = ws.mutable_data_ptr();
    const int lda = (int)x->stride(0), ldc = (int)out->stride(0);
    int st;
    {
      const NoGil unlocked;
      std::lock_guard<std::mutex> lock(buffers->host_call);
      st = g_gemm_host(a, lda, bq, scp, c, ldc, M, l.N, l.K, l.code, l.zero_point, l.group, act, a_stage, c_stage, w,
                       (size_t)ws.numel(), stream);
    }
    if (st != 0) return raise_status(st);
  }
  Py_INCREF(args[1]);
  return args[1];
  END_HANDLE_TH_ERRORS
}

// gate_up_cast(x, quantized_weight, scales, layer, channels per scale, clamp value or None)
//   -> (out e4m3 [M, N / 2], out_sf float32 [M, N / 2 / channels], gate_up [M, N])
PyObject* gate_up_cast(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6) { PyErr_SetString(PyExc_TypeError, "gate_up_cast takes 6 arguments"); return nullptr; }
  const at::Tensor* x = as_tensor(args[0], "activations");
  const at::Tensor* qw = as_tensor(args[1], "quantized_weight");
  const at::Tensor* scales = as_tensor(args[2], "scales");
  Layer l;
  if (!x || !qw || !scales || !parse_layer(args[3], &l)) return nullptr;
  const long channels = PyLong_AsLong(args[4]);
  const bool clamp = args[5] != Py_None;
  const double clamp_value = clamp ? PyFloat_AsDouble(args[5]) : 0.0;
  if (PyErr_Occurred()) return nullptr;
  if (channels < 1) { PyErr_SetString(PyExc_ValueError, "channels per scale must be positive"); return nullptr; }
  // rows of K values: any shape whose elements make them up ([tokens, heads, head size] of an attention output), or the
  // first K columns of a wider matrix
  at::Tensor rows;
  if (x->dim() == 2 && x->size(1) >= l.K) {
    rows = *x;
  } else if (x->dim() != 2 && x->numel() % l.K == 0) {
    rows = x->reshape({-1, (int64_t)l.K});
  } else {
    PyErr_Format(PyExc_ValueError, "expected rows of %d input features", l.K);
    return nullptr;
  }
  const at::ScalarType dtype = scales->scalar_type();
  const int act = act_code(dtype);
  if (!rows.is_cuda() || rows.scalar_type() != dtype || act < 0 || rows.stride(1) != 1) {
    PyErr_Format(PyExc_ValueError, "activations must be CUDA %s with unit inner stride", c10::toString(dtype));
    return nullptr;
  }
  const c10::Device dev = rows.device();
  if (!check_weights(*qw, *scales, dev)) return nullptr;
  const int M = (int)rows.size(0), H = l.N / 2;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor gate_up = at::detail::empty_cuda({M, l.N}, dtype, dev, std::nullopt);
  at::Tensor out = at::detail::empty_cuda({M, H}, at::kFloat8_e4m3fn, dev, std::nullopt);
  at::Tensor sf = at::detail::empty_cuda({M, H / channels}, at::kFloat, dev, std::nullopt);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const size_t need = g_workspace_bytes(M, l.N, l.K, l.code, l.zero_point, l.group);
  if (need == 0) return raise_unsupported(M, l.N, l.K);
  const at::Tensor ws = workspace_of(dev.index(), stream, need);
  const void *a = rows.const_data_ptr(), *bq = qw->const_data_ptr(), *sc = scales->const_data_ptr();
  void *g = gate_up.mutable_data_ptr(), *o = out.mutable_data_ptr(), *f = sf.mutable_data_ptr(), *w = ws.mutable_data_ptr();
  const int lda = (int)rows.stride(0);
  int st;
  {
    const NoGil unlocked;
    st = g_gemm_cast(a, lda, bq, sc, g, l.N, o, H, static_cast<float*>(f), M, l.N, l.K, l.code, l.zero_point, l.group, act,
                     (int)channels, clamp ? 1 : 0, (float)clamp_value, w, (size_t)ws.numel(), stream);
  }
  if (st != 0) return raise_status(st);
  return PyTuple_Pack(3, THPObjectPtr(THPVariable_Wrap(std::move(out))).get(),
                      THPObjectPtr(THPVariable_Wrap(std::move(sf))).get(),
                      THPObjectPtr(THPVariable_Wrap(std::move(gate_up))).get());
  END_HANDLE_TH_ERRORS
}

// workspace(device index, bytes) -> the zeroed workspace of the device's current stream
PyObject* workspace(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  int device;
  Py_ssize_t bytes;
  if (!PyArg_ParseTuple(args, "in", &device, &bytes)) return nullptr;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  return THPVariable_Wrap(
      workspace_of(device, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(), (size_t)bytes));
  END_HANDLE_TH_ERRORS
}

// ---- 8-bit integer operators and block norms ------------------------------------------------------------
decltype(&b200q_per_token_cast_int) g_cast_int = nullptr;
decltype(&b200q_igemm) g_igemm = nullptr;
decltype(&b200q_igemm_swiglu) g_igemm_swiglu = nullptr;
decltype(&b200q_block_norm) g_norm = nullptr;
decltype(&b200q_block_norm_scratch_bytes) g_norm_scratch = nullptr;
decltype(&b200q_block_norm_backward) g_norm_backward = nullptr;

bool value_error(const char* what) {
  PyErr_SetString(PyExc_ValueError, what);
  return false;
}
bool type_error(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return false;
}
// rows of an operator: 2-D with unit inner stride, rows that do not share memory, sizes that fit the C ABI's integers
bool check_rows(const at::Tensor& t, const char* name, const c10::Device& dev) {
  if (t.device() != dev) { PyErr_Format(PyExc_ValueError, "%s must be on the device of the other operands", name); return false; }
  if (t.dim() != 2 || (t.stride(1) != 1 && t.size(1) > 1)) {
    PyErr_Format(PyExc_ValueError, "%s must be a 2-D tensor with unit inner stride", name);
    return false;
  }
  if (t.size(0) > INT32_MAX || t.size(1) > INT32_MAX || t.stride(0) > INT32_MAX) {
    PyErr_Format(PyExc_ValueError, "%s is too large", name);
    return false;
  }
  return true;
}
// the row stride; of a single row its length, whatever the tensor says
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// a contiguous vector of `n` values
bool check_vector(const at::Tensor& t, const char* name, int64_t n, at::ScalarType type, const c10::Device& dev) {
  if (t.device() != dev) { PyErr_Format(PyExc_ValueError, "%s must be on the device of the other operands", name); return false; }
  if (t.scalar_type() != type) { PyErr_Format(PyExc_TypeError, "%s must be %s", name, c10::toString(type)); return false; }
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) {
    PyErr_Format(PyExc_ValueError, "%s must be a contiguous tensor of %lld values", name, (long long)n);
    return false;
  }
  return true;
}
bool need_cuda(const at::Tensor& t, const char* op) {
  if (t.is_cuda()) return true;
  PyErr_Format(PyExc_ValueError, "%s needs CUDA tensors (there is no CPU path)", op);
  return false;
}
// an optional tensor argument: *t is null where it is None
bool optional_tensor(PyObject* o, const char* name, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = as_tensor(o, name);
  return *t != nullptr;
}

// cast_int8(x) -> (out int8 [tokens, hidden], out_sf float32 [tokens])
PyObject* cast_int8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 1) { type_error("cast_int8 takes 1 argument"); return nullptr; }
  const at::Tensor* x = as_tensor(args[0], "x");
  if (!x || !need_cuda(*x, "per_token_cast_int8") || !check_rows(*x, "x", x->device())) return nullptr;
  const int act = act_code(x->scalar_type());
  if (act < 0) { type_error("x must be float16 or bfloat16"); return nullptr; }
  const c10::Device dev = x->device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int T = (int)x->size(0), H = (int)x->size(1);
  at::Tensor out = at::detail::empty_cuda({T, H}, at::kChar, dev, std::nullopt);
  at::Tensor sf = at::detail::empty_cuda({T}, at::kFloat, dev, std::nullopt);
  if (T > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const void* xp = x->const_data_ptr();
    void *op = out.mutable_data_ptr(), *fp = sf.mutable_data_ptr();
    const int ldx = (int)row_stride(*x);
    int st;
    {
      const NoGil unlocked;
      st = g_cast_int(xp, ldx, op, H, static_cast<float*>(fp), T, H, act, stream);
    }
    if (st != 0) return raise_status(st);
  }
  return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(std::move(out))).get(), THPObjectPtr(THPVariable_Wrap(std::move(sf))).get());
  END_HANDLE_TH_ERRORS
}

// igemm(a, b, a_sf, b_sf, bias or None, activation type's code, gated, clamp value or None, out or None, early) -> out
// `early`: the caller knows that B has been complete since before the stream's previous kernel.  (Nothing here can know it: kernels of others
// are not seen, and what a kernel has written that lets its successor start under its end counts only after that successor's wait.)
PyObject* igemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10) { type_error("igemm takes 10 arguments"); return nullptr; }
  const at::Tensor *a = as_tensor(args[0], "a"), *b = a ? as_tensor(args[1], "b") : nullptr;
  const at::Tensor *a_sf = b ? as_tensor(args[2], "a_sf") : nullptr, *b_sf = a_sf ? as_tensor(args[3], "b_sf") : nullptr;
  const at::Tensor *bias, *given;
  if (!b_sf || !optional_tensor(args[4], "bias", &bias) || !optional_tensor(args[8], "out", &given)) return nullptr;
  const long act = PyLong_AsLong(args[5]);
  const int gated = PyObject_IsTrue(args[6]), early = PyObject_IsTrue(args[9]);
  const bool clamp = args[7] != Py_None;
  const double clamp_value = clamp ? PyFloat_AsDouble(args[7]) : 0.0;
  if (PyErr_Occurred()) return nullptr;
  if (!need_cuda(*a, gated ? "int8_gate_up" : "int8_matmul")) return nullptr;
  const c10::Device dev = a->device();
  if (!check_rows(*a, "a", dev) || !check_rows(*b, "b", dev)) return nullptr;
  if (a->scalar_type() != at::kChar || b->scalar_type() != at::kChar) { type_error("a and b must be int8"); return nullptr; }
  const int64_t M = a->size(0), K = a->size(1), rows = b->size(0), N = gated ? rows / 2 : rows;
  if (b->size(1) != K) { value_error("a and b must have rows of the same length"); return nullptr; }
  if (gated && rows % 2 != 0) { value_error("b must hold as many rows behind the gate's as the gate has"); return nullptr; }
  if (!check_vector(*a_sf, "a_sf", M, at::kFloat, dev) || !check_vector(*b_sf, "b_sf", rows, at::kFloat, dev)) return nullptr;
  const at::ScalarType type = act == 1 ? at::kBFloat16 : at::kHalf;
  if (bias && !check_vector(*bias, "bias", N, type, dev)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (given) {
    if (!check_rows(*given, "out", dev)) return nullptr;
    if (given->scalar_type() != type) { type_error("out must be of out_dtype"); return nullptr; }
    if (given->size(0) != M || given->size(1) != N) { value_error("out has the wrong shape"); return nullptr; }
    if (c10::GradMode::is_enabled() && given->requires_grad()) { value_error("out must not require a gradient"); return nullptr; }
  }
  at::Tensor out;
  if (given) out = *given;
  else out = at::detail::empty_cuda({M, N}, type, dev, std::nullopt);
  if (M > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspace_of(dev.index(), stream, 256);
    const void *ap = a->const_data_ptr(), *bp = b->const_data_ptr(), *biasp = bias ? bias->const_data_ptr() : nullptr;
    const float *fa = a_sf->const_data_ptr<float>(), *fb = b_sf->const_data_ptr<float>();
    void *c = out.mutable_data_ptr(), *w = ws.mutable_data_ptr();
    const int lda = (int)row_stride(*a), ldb = (int)row_stride(*b), ldc = (int)row_stride(out);
    const size_t ws_bytes = (size_t)ws.numel();
    int st;
    {
      const NoGil unlocked;
      st = gated ? g_igemm_swiglu(ap, lda, bp, ldb, fa, fb, c, ldc, (int)M, (int)N, (int)K, (int)act, clamp ? 1 : 0, (float)clamp_value,
                                  early, w, ws_bytes, stream)
                 : g_igemm(ap, lda, bp, ldb, fa, fb, biasp, c, ldc, (int)M, (int)N, (int)K, (int)act, early, w, ws_bytes, stream);
    }
    if (st != 0) return raise_status(st);
    if (given && !given->is_inference()) given->unsafeGetTensorImpl()->bump_version();  // autograd may have saved it
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The operands that a block norm and its gradient share: (block, residual or None, weight, post weight or None, gate or None,
// residual scale, eps)
struct NormOperands {
  const at::Tensor *block, *residual, *weight, *post, *gate;
  at::ScalarType residual_type;
  b200q_block_norm_t c;
};
bool parse_norm(PyObject* const* args, const char* op, NormOperands* n) {
  if (!(n->block = as_tensor(args[0], "block")) || !optional_tensor(args[1], "residual", &n->residual) ||
      !(n->weight = as_tensor(args[2], "weight")) || !optional_tensor(args[3], "post_weight", &n->post) ||
      !optional_tensor(args[4], "gate", &n->gate) || !need_cuda(*n->block, op))
    return false;
  const double scale = PyFloat_AsDouble(args[5]), eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return false;
  const at::ScalarType type = n->block->scalar_type();
  const c10::Device dev = n->block->device();
  n->c = b200q_block_norm_t();
  n->c.act_dtype = act_code(type);
  if (n->c.act_dtype < 0) return type_error("block must be float16 or bfloat16");
  if (!check_rows(*n->block, "block", dev)) return false;
  const int64_t T = n->block->size(0), D = n->block->size(1);
  n->residual_type = type;
  if (n->residual) {
    if (!check_rows(*n->residual, "residual", dev)) return false;
    n->residual_type = n->residual->scalar_type();
    if (n->residual_type != type && n->residual_type != at::kFloat)
      return type_error("residual must be float32 or of the block's type");
    if (n->residual->size(0) != T || n->residual->size(1) != D) return value_error("residual must have the block's shape");
    n->c.residual = n->residual->const_data_ptr();
    n->c.ldr = row_stride(*n->residual);
  }
  if (!check_vector(*n->weight, "weight", D, type, dev)) return false;
  if (n->post && !check_vector(*n->post, "post_weight", D, type, dev)) return false;
  if (n->gate) {
    if (n->gate->device() != dev || n->gate->scalar_type() != type)
      return type_error("gate must be of the block's type and on its device");
    const int64_t G = n->gate->dim() == 1 ? 1 : n->gate->size(0);
    if (n->gate->dim() < 1 || n->gate->dim() > 2 || n->gate->size(-1) != D || (D > 1 && n->gate->stride(-1) != 1))
      return value_error("gate must be [hidden] or [gates, hidden] with unit inner stride");
    if (G < 1 || T % G != 0) return value_error("gate must have a row for each run of as many tokens");
    n->c.gate = n->gate->const_data_ptr();
    n->c.gates = (int32_t)G;
    n->c.ldg = G > 1 ? n->gate->stride(0) : D;
  }
  n->c.block = n->block->const_data_ptr();
  n->c.weight = n->weight->const_data_ptr();
  n->c.post_weight = n->post ? n->post->const_data_ptr() : nullptr;
  n->c.ldb = row_stride(*n->block);
  n->c.tokens = (int32_t)T;
  n->c.hidden = (int32_t)D;
  n->c.residual_f32 = n->residual_type == at::kFloat;
  n->c.residual_scale = (float)scale;
  n->c.eps = (float)eps;
  return true;
}

// block_norm(the operands, cast) -> (x, new residual), or with the cast (x int8, x_sf float32 [tokens], new residual)
PyObject* block_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8) { type_error("block_norm takes 8 arguments"); return nullptr; }
  const int cast = PyObject_IsTrue(args[7]);
  NormOperands n;
  if (!parse_norm(args, cast ? "block_norm_cast_int8" : "block_norm", &n)) return nullptr;
  const c10::Device dev = n.block->device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int64_t T = n.c.tokens, D = n.c.hidden;
  at::Tensor x = at::detail::empty_cuda({T, D}, cast ? at::kChar : n.block->scalar_type(), dev, std::nullopt);
  at::Tensor fresh = at::detail::empty_cuda({T, D}, n.residual_type, dev, std::nullopt), sf;
  if (cast) sf = at::detail::empty_cuda({T}, at::kFloat, dev, std::nullopt);
  if (T > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    void *xp = x.mutable_data_ptr(), *rp = fresh.mutable_data_ptr(), *fp = cast ? sf.mutable_data_ptr() : nullptr;
    int st;
    {
      const NoGil unlocked;
      st = g_norm(&n.c, cast ? nullptr : xp, D, cast ? xp : nullptr, static_cast<float*>(fp), rp, D, stream);
    }
    if (st != 0) return raise_status(st);
  }
  if (cast)
    return PyTuple_Pack(3, THPObjectPtr(THPVariable_Wrap(std::move(x))).get(), THPObjectPtr(THPVariable_Wrap(std::move(sf))).get(),
                        THPObjectPtr(THPVariable_Wrap(std::move(fresh))).get());
  return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(std::move(x))).get(), THPObjectPtr(THPVariable_Wrap(std::move(fresh))).get());
  END_HANDLE_TH_ERRORS
}

// block_norm_backward(the operands, grad_x, grad of the new residual or None)
//   -> (grad_block, grad_residual or None, grad_weight, grad_post or None, grad_gate or None), the last three float32
PyObject* block_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) { type_error("block_norm_backward takes 9 arguments"); return nullptr; }
  NormOperands n;
  const at::Tensor *dx, *dn;
  if (!parse_norm(args, "block_norm_backward", &n) || !(dx = as_tensor(args[7], "grad_x")) ||
      !optional_tensor(args[8], "grad_new_residual", &dn))
    return nullptr;
  const c10::Device dev = n.block->device();
  const int64_t T = n.c.tokens, D = n.c.hidden;
  if (!check_rows(*dx, "grad_x", dev) || (dn && !check_rows(*dn, "grad_new_residual", dev))) return nullptr;
  if (dx->scalar_type() != n.block->scalar_type()) { type_error("grad_x must be of the block's type"); return nullptr; }
  if (dx->size(0) != T || dx->size(1) != D) { value_error("grad_x must have the block's shape"); return nullptr; }
  if (dn) {
    // (without a residual the new one has the block's type)
    if (dn->scalar_type() != n.residual_type) { type_error("grad_new_residual must be of the new residual's type"); return nullptr; }
    if (dn->size(0) != T || dn->size(1) != D) { value_error("grad_new_residual must have the block's shape"); return nullptr; }
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  at::Tensor gb = at::detail::empty_cuda({T, D}, n.block->scalar_type(), dev, std::nullopt), gr, gp, gg;
  at::Tensor gw = at::detail::empty_cuda({D}, at::kFloat, dev, std::nullopt);
  if (n.residual) gr = at::detail::empty_cuda({T, D}, n.residual_type, dev, std::nullopt);
  if (n.post) gp = at::detail::empty_cuda({D}, at::kFloat, dev, std::nullopt);
  if (n.gate) gg = at::detail::empty_cuda(n.gate->sizes(), at::kFloat, dev, std::nullopt);
  if (T > 0) {
    const size_t need = g_norm_scratch((int)T, (int)D, n.c.gates);
    if (need == 0) return raise_status(B200Q_ERR_UNSUPPORTED);
    const at::Tensor scratch = at::detail::empty_cuda({(int64_t)need}, at::kByte, dev, std::nullopt);
    const at::Tensor ws = workspace_of(dev.index(), stream, 256);
    void* wsp = ws.mutable_data_ptr();
    const size_t ws_bytes = (size_t)ws.numel();
    void *b = gb.mutable_data_ptr(), *r = n.residual ? gr.mutable_data_ptr() : nullptr, *s = scratch.mutable_data_ptr();
    float *w = gw.mutable_data_ptr<float>(), *p = n.post ? gp.mutable_data_ptr<float>() : nullptr;
    float* g = n.gate ? gg.mutable_data_ptr<float>() : nullptr;
    const void *dxp = dx->const_data_ptr(), *dnp = dn ? dn->const_data_ptr() : nullptr;
    const int64_t lddx = row_stride(*dx), lddn = dn ? row_stride(*dn) : 0;
    int st;
    {
      const NoGil unlocked;
      st = g_norm_backward(&n.c, dxp, lddx, dnp, lddn, b, D, r, D, w, p, g, s, need, wsp, ws_bytes, stream);
    }
    if (st != 0) return raise_status(st);
  } else {
    for (at::Tensor* t : {&gw, &gp, &gg})
      if (t->defined() && t->numel()) C10_CUDA_CHECK(cudaMemsetAsync(t->mutable_data_ptr(), 0, (size_t)t->numel() * 4, stream));
  }
  auto wrap = [](at::Tensor& t) -> PyObject* {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
  };
  return PyTuple_Pack(5, THPObjectPtr(wrap(gb)).get(), THPObjectPtr(wrap(gr)).get(), THPObjectPtr(wrap(gw)).get(),
                      THPObjectPtr(wrap(gp)).get(), THPObjectPtr(wrap(gg)).get());
  END_HANDLE_TH_ERRORS
}

// bind_int8(per_token_cast_int, igemm, igemm_swiglu, block_norm, block_norm_scratch_bytes, block_norm_backward): addresses
PyObject* bind_int8(PyObject*, PyObject* args) {
  unsigned long long f[6];
  if (!PyArg_ParseTuple(args, "KKKKKK", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5])) return nullptr;
  g_cast_int = reinterpret_cast<decltype(g_cast_int)>(f[0]);
  g_igemm = reinterpret_cast<decltype(g_igemm)>(f[1]);
  g_igemm_swiglu = reinterpret_cast<decltype(g_igemm_swiglu)>(f[2]);
  g_norm = reinterpret_cast<decltype(g_norm)>(f[3]);
  g_norm_scratch = reinterpret_cast<decltype(g_norm_scratch)>(f[4]);
  g_norm_backward = reinterpret_cast<decltype(g_norm_backward)>(f[5]);
  Py_RETURN_NONE;
}

// bind(gemm, gemm_host, gemm_swiglu_cast, workspace_bytes, raise_status, raise_unsupported): addresses in
// libb200q and the Python callables that raise for a status
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long gemm, host, cast, ws;
  PyObject *status, *unsupported;
  if (!PyArg_ParseTuple(args, "KKKKOO", &gemm, &host, &cast, &ws, &status, &unsupported)) return nullptr;
  g_gemm = reinterpret_cast<GemmFn>(gemm);
  g_gemm_host = reinterpret_cast<GemmHostFn>(host);
  g_gemm_cast = reinterpret_cast<GemmCastFn>(cast);
  g_workspace_bytes = reinterpret_cast<WorkspaceFn>(ws);
  Py_INCREF(status);
  Py_INCREF(unsupported);
  Py_XSETREF(g_raise_status, status);
  Py_XSETREF(g_raise_unsupported, unsupported);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"linear_host", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear_host)), METH_FASTCALL, nullptr},
    {"gate_up_cast", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gate_up_cast)), METH_FASTCALL, nullptr},
    {"workspace", workspace, METH_VARARGS, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"cast_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cast_int8)), METH_FASTCALL, nullptr},
    {"igemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(igemm)), METH_FASTCALL, nullptr},
    {"block_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(block_norm)), METH_FASTCALL, nullptr},
    {"block_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(block_norm_backward)), METH_FASTCALL, nullptr},
    {"bind_int8", bind_int8, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__native() { return PyModule_Create(&module); }
