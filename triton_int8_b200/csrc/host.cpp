// Host side of the composed calls and of the expert layers for plain tensors: argument checks, allocations and the autograd nodes
// without the Python interpreter in between.  Small calls are bound by it: 128x1024x1024 forward 47 us a call in
// Python against 18 us on the device, forward and backward of 512x1024x1024 205 us against 58.
//
// Everything here handles one case, contiguous CUDA tensors (bf16, in the expert layers fp16 and fp32 too) of matching shapes outside of
// tracing, transforms and modes, and returns None for any other: the callers in kernels.py and linear.py then take the Python path, which
// accepts or refuses it.  The entry points of libi8linear.so are passed in by address (setup), so that the library in
// use is the one that _lib.py has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/PythonFallbackKernel.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <atomic>

#include "../../include/i8linear.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&i8l_quant_gemm) lib_quant_gemm = nullptr;
decltype(&i8l_linear_backward_bias) lib_linear_backward = nullptr;
decltype(&i8l_status_peek) lib_status_peek = nullptr;
decltype(&i8l_sort_workspace) lib_sort_workspace = nullptr;
decltype(&i8l_sort_tokens) lib_sort_tokens = nullptr;
decltype(&i8l_combine) lib_combine = nullptr;
decltype(&i8l_combine_backward) lib_combine_backward = nullptr;
decltype(&i8l_token_linear_workspace) lib_token_workspace = nullptr;
decltype(&i8l_token_linear) lib_token_linear = nullptr;
PyObject* py_combine_backward = nullptr;   // (rows or None, weights, pos, src, dy, wants drows, wants dweights) -> (drows, dweights)
PyObject* on_error = nullptr;       // (entry point, code, device index): raises
PyObject* on_timeout = nullptr;     // (device index): raises, or returns where there is nothing to report now
PyObject* open_status = nullptr;    // (device index) -> (status word, poller), as integers
PyObject* py_backward = nullptr;    // the Python path of the backward pass

class WithGil {
 public:
  WithGil() : state_(PyGILState_Ensure()) {}
  ~WithGil() { PyGILState_Release(state_); }

 private:
  PyGILState_STATE state_;
};
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }

 private:
  PyThreadState* state_;
};

[[noreturn]] void throw_python_error() {   // the Python error that is set, carried through C++ frames and threads
  python_error e;
  e.persist();
  throw e;
}

struct Status {
  std::atomic<int32_t*> word{nullptr};
  std::atomic<void*> poller{nullptr};
};
constexpr int MAX_DEVICES = 64;
std::array<Status, MAX_DEVICES> statuses;

Status& status_of(int dev) {
  Status& s = statuses[dev];
  if (!s.word.load(std::memory_order_acquire)) {
    const WithGil gil;
    PyObject* r = PyObject_CallFunction(open_status, "i", dev);
    if (!r) throw_python_error();
    unsigned long long word = 0, poller = 0;
    const int ok = PyArg_ParseTuple(r, "KK", &word, &poller);
    Py_DECREF(r);
    if (!ok) throw_python_error();
    s.poller.store(reinterpret_cast<void*>(poller), std::memory_order_relaxed);   // the same pair for every thread that comes here
    s.word.store(reinterpret_cast<int32_t*>(word), std::memory_order_release);
  }
  return s;
}

void check(const char* name, int rc, int dev) {
  if (rc == I8L_OK) return;
  const WithGil gil;
  PyObject* r = PyObject_CallFunction(on_error, "sii", name, rc, dev);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed with code %d", name, rc);
  throw_python_error();
}

void report_timeout(int dev) {   // an earlier GEMM gave up a wait
  if (lib_status_peek(status_of(dev).poller.load(std::memory_order_relaxed)) == I8L_OK) return;
  const WithGil gil;
  PyObject* r = PyObject_CallFunction(on_timeout, "i", dev);
  if (!r) throw_python_error();
  Py_DECREF(r);
}

// A dense CUDA tensor with its own memory and nothing that a dispatcher would have to see.
bool dense(const Tensor& t) {
  const auto ks = t.key_set();
  return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && t.get_device() < MAX_DEVICES &&
         !ks.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                          c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate,
                                          c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor,
                                          c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                          c10::DispatchKey::FuncTorchBatchedDecomposition, c10::DispatchKey::BatchedNestedTensor,
                                          c10::DispatchKey::Batched}));
}
bool forward_mode(const Tensor& t) { return t._fw_grad(0).defined(); }
bool plain(const Tensor& t) { return t.scalar_type() == at::kBFloat16 && dense(t); }
// No mode, transform or tracer looks at what this thread does.
bool plain_thread() {
  const auto inc = c10::impl::tls_local_dispatch_key_set().included_;
  return !c10::impl::dispatch_mode_enabled() && !at::impl::torch_function_mode_enabled() &&
         !inc.has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                           c10::DispatchKey::FuncTorchDynamicLayerBackMode, c10::DispatchKey::FuncTorchVmapMode,
                                           c10::DispatchKey::VmapMode, c10::DispatchKey::Tracer, c10::DispatchKey::Python,
                                           c10::DispatchKey::Functionalize}));
}

int64_t pad(int64_t n) { return (n + 255) & -256; }
int64_t scale_count(int gran, int64_t batch, int64_t rows, int64_t cols) {
  switch (gran) {
    case I8L_GRAN_TILE128: return batch * (rows / 128) * (cols / 128);
    case I8L_GRAN_TILE128X256: return batch * (rows / 128) * (cols / 256);
    case I8L_GRAN_GROUP128: return batch * rows * (cols / 128);
    default: return batch * rows;
  }
}
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kChar)); }

struct Transposed {
  Tensor q, scale;
};

// a [B, M, K] x b [N, K] or [B, N, K], as [B, M, N]; the caller has checked shapes and tensors.
Tensor quant_gemm(const Tensor& a, int64_t B, int64_t M, const Tensor& b, bool b_batched, int a_gran, int b_gran, int qmode,
                  int hadamard, const Tensor* bias, double post, int flags, Transposed* at_out) {
  const int64_t K = b.size(-1), N = b.size(-2), nb = b_batched ? B : 1;
  const int dev = a.get_device();
  const c10::cuda::CUDAGuard guard(dev);
  Status& status = status_of(dev);
  Tensor out = at::empty({B, M, N}, a.options().dtype(flags & I8L_GEMM_OUT_F32 ? at::kFloat : at::kBFloat16));
  const int64_t size = pad(B * M * K) + pad(nb * N * K) + pad(4 * scale_count(a_gran, B, M, K)) +
                       pad(4 * scale_count(b_gran, nb, N, K)) + (at_out ? pad(4 * K) : 0);
  const Tensor ws = bytes(size, a);
  int8_t* qt = nullptr;
  float* st = nullptr;
  if (at_out) {
    at_out->q = at::empty({B, K, M}, a.options().dtype(at::kChar));
    const auto f32 = a.options().dtype(at::kFloat);
    at_out->scale = a_gran == I8L_GRAN_TILE128 ? at::empty({B, K / 128, M / 128}, f32)
                    : a_gran == I8L_GRAN_ROW   ? at::empty({B, K}, f32)
                                               : at::empty({B, K, M / 128}, f32);
    qt = static_cast<int8_t*>(at_out->q.data_ptr());
    st = static_cast<float*>(at_out->scale.data_ptr());
  }
  check("i8l_quant_gemm",
        lib_quant_gemm(a.data_ptr(), b.data_ptr(), bias ? bias->data_ptr() : nullptr, out.data_ptr(), qt, st, B, M, N, K, b_batched,
                       a_gran, b_gran, qmode, hadamard, (float)post, flags, ws.data_ptr(), size,
                       status.word.load(std::memory_order_relaxed), c10::cuda::getCurrentCUDAStream(dev).stream()),
        dev);
  return out;
}

bool plain_bias(const Tensor& bias, const Tensor& a, int64_t N) {
  return plain(bias) && bias.device() == a.device() && bias.numel() >= N;
}

// What a linear layer needs to know of its Int8Config.
struct Config {
  int gran, qmode, hadamard, flags;
  bool whole_k;
  double post(int64_t) const { return hadamard ? 1.0 / hadamard : 1.0; }
  int64_t code() const { return gran | qmode << 8 | flags << 16 | (int64_t)whole_k << 31 | (int64_t)hadamard << 32; }
  static Config from(int64_t c) {
    return Config{(int)(c & 0xff), (int)(c >> 8 & 0xff), (int)(c >> 32), (int)(c >> 16 & 0xff), (bool)(c >> 31 & 1)};
  }
};

Tensor linear_forward(const Tensor& x, const Tensor& weight, const Tensor* bias, const Config& c, Transposed* xt) {
  const int64_t K = weight.size(1), M = x.numel() / K;
  const int b_gran = I8L_GRAN_ROW, a_gran = c.whole_k ? I8L_GRAN_ROW : c.gran;
  const Tensor y = quant_gemm(x, 1, M, weight, false, a_gran, b_gran, c.whole_k ? I8L_QMODE_ROWRCP : c.qmode, c.hadamard, bias,
                              c.post(K), c.whole_k ? 0 : c.flags, xt);
  auto shape = x.sizes().vec();
  shape.back() = weight.size(0);
  return y.select(0, 0).view(shape);   // a view, as the Python path returns it
}

// The Python path of the backward pass, for what the native one does not take.
void backward_in_python(const Tensor& dy, const Tensor& weight, const Tensor& q, const Tensor& s, const Config& c, bool need_dx,
                        bool need_dw, Tensor& dx, Tensor& dw) {
  const WithGil gil;
  PyObject *pd = THPVariable_Wrap(dy), *pw = THPVariable_Wrap(weight), *pq = THPVariable_Wrap(q), *ps = THPVariable_Wrap(s);
  PyObject* r = PyObject_CallFunction(py_backward, "NNNNiiiiiii", pd, pw, pq, ps, c.gran, c.qmode, c.hadamard, c.flags, (int)c.whole_k,
                                      (int)need_dx, (int)need_dw);
  if (!r) throw_python_error();
  PyObject *px = nullptr, *pdw = nullptr;
  const int ok = PyArg_ParseTuple(r, "OO", &px, &pdw);
  if (ok && THPVariable_Check(px)) dx = THPVariable_Unpack(px);
  if (ok && THPVariable_Check(pdw)) dw = THPVariable_Unpack(pdw);
  Py_DECREF(r);
  if (!ok) throw_python_error();
}

void linear_backward(const Tensor& dy, const Tensor& weight, const Tensor& q, const Tensor& s, const Config& c, bool need_dx,
                     bool need_dw, bool need_db, Tensor& dx, Tensor& dw, Tensor& db) {
  const int64_t M = dy.size(0), N = dy.size(1), K = weight.size(1);
  const int gran = c.whole_k ? I8L_GRAN_ROW : c.gran;
  bool ok = plain_thread() && plain(dy) && !forward_mode(dy) && plain(weight) && weight.size(0) == N && weight.device() == dy.device();
  if (ok && need_dw) {
    ok = q.defined() && s.defined() && q.device() == dy.device() && s.device() == dy.device() && q.scalar_type() == at::kChar &&
         s.scalar_type() == at::kFloat && q.is_contiguous() && s.is_contiguous() && q.sizes() == at::IntArrayRef({1, K, M}) &&
         s.numel() == scale_count(gran, 1, K, M);
  }
  // torch's sum where its graph (create_graph) or tangent is wanted, and where the kernel's 16-byte loads do not fit
  const bool own_sum = need_db && ok && !at::GradMode::is_enabled() && reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0;
  if (need_db && !own_sum) db = dy.sum(0);
  if (!ok) {
    if (need_dx || need_dw) backward_in_python(dy, weight, q, s, c, need_dx, need_dw, dx, dw);
    return;
  }
  if (!need_dx && !need_dw && !own_sum) return;
  const int dev = dy.get_device();
  const c10::cuda::CUDAGuard guard(dev);
  Status& status = status_of(dev);
  if (need_dx) dx = at::empty({M, K}, dy.options());
  if (need_dw) dw = at::empty({N, K}, dy.options());
  if (own_sum) db = at::empty({N}, dy.options());
  int64_t size = pad(4 * std::max(K, N));
  if (need_dx) size += pad(M * N) + pad(4 * scale_count(gran, 1, M, N)) + pad(4 * K) + (need_dw ? 0 : pad(K * N));
  if (need_dw) size += pad(N * M) + pad(4 * scale_count(gran, 1, N, M));
  const Tensor ws = bytes(size, dy);
  check("i8l_linear_backward_bias",
        lib_linear_backward(dy.data_ptr(), weight.data_ptr(), need_dw ? static_cast<const int8_t*>(q.data_ptr()) : nullptr,
                            need_dw ? static_cast<const float*>(s.data_ptr()) : nullptr, need_dx ? dx.data_ptr() : nullptr,
                            need_dw ? dw.data_ptr() : nullptr, own_sum ? db.data_ptr() : nullptr, M, N, K, gran, c.whole_k ? I8L_QMODE_ROWRCP : c.qmode, c.hadamard,
                            (float)c.post(N), (float)c.post(M), c.whole_k ? 0 : c.flags, ws.data_ptr(), size,
                            status.word.load(std::memory_order_relaxed), c10::cuda::getCurrentCUDAStream(dev).stream()),
        dev);
}

struct Int8LinearNode : torch::autograd::Function<Int8LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, int64_t config,
                        bool need_w) {
    Transposed xt;
    const Tensor y = linear_forward(x, weight, bias ? &*bias : nullptr, Config::from(config), need_w ? &xt : nullptr);
    ctx->saved_data["config"] = config;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["shape"] = x.sizes().vec();
    if (need_w) ctx->save_for_backward({weight, xt.q, xt.scale});
    else ctx->save_for_backward({weight});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Config c = Config::from(ctx->saved_data["config"].toInt());
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const Tensor& dy = grads[0];
    const Tensor dy2 = dy.reshape({-1, dy.size(-1)}).contiguous();
    Tensor dx, dw, db;
    linear_backward(dy2, saved[0], saved.size() > 1 ? saved[1] : Tensor(), saved.size() > 1 ? saved[2] : Tensor(), c,
                    ctx->needs_input_grad(0), ctx->needs_input_grad(1), has_bias && ctx->needs_input_grad(2), dx, dw, db);
    if (dx.defined()) dx = dx.view(ctx->saved_data["shape"].toIntVector());
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------------ expert layers
int dtype_of(const Tensor& t) {   // negative: a type that the kernels do not take
  switch (t.scalar_type()) {
    case at::kBFloat16: return I8L_DTYPE_BF16;
    case at::kHalf: return I8L_DTYPE_F16;
    case at::kFloat: return I8L_DTYPE_F32;
    default: return -1;
  }
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
template <typename T> T* at_of(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

struct Sorted {
  Tensor rows, offsets, pos, src;
};
Sorted sort_tokens(const Tensor& x, const Tensor& ids, int experts, int64_t align) {
  const int64_t T = x.size(0), H = x.size(1), k = ids.size(1), n = T * k;
  const int64_t R = (n + std::min<int64_t>(experts, n) * (align - 1) + align - 1) / align * align;
  const int dev = x.get_device();
  const c10::cuda::CUDAGuard guard(dev);
  const auto i32 = x.options().dtype(at::kInt);
  Sorted s{at::empty({R, H}, x.options()), at::empty({experts + 1}, i32), at::empty({T, k}, i32), at::empty({R}, i32)};
  const int64_t size = lib_sort_workspace(T, (int)k, experts);
  const Tensor ws = size ? bytes(size, x) : Tensor();
  check("i8l_sort_tokens",
        lib_sort_tokens(x.data_ptr(), ids.data_ptr(), ids.scalar_type() == at::kLong, T, H, (int)k, experts, align, dtype_of(x), R,
                        s.rows.data_ptr(), at_of<int32_t>(s.offsets), at_of<int32_t>(s.pos), at_of<int32_t>(s.src),
                        size ? ws.data_ptr() : nullptr, size, stream_of(dev)),
        dev);
  return s;
}
// weights undefined: ones
Tensor combine(const Tensor& rows, const Tensor& weights, const Tensor& pos) {
  const int64_t T = pos.size(0), k = pos.size(1), R = rows.size(0), H = rows.size(1);
  const int dev = rows.get_device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor y = at::empty({T, H}, rows.options());
  check("i8l_combine",
        lib_combine(rows.data_ptr(), weights.defined() ? weights.data_ptr() : nullptr, at_of<int32_t>(pos), R, T, H, (int)k, dtype_of(rows),
                    weights.defined() ? dtype_of(weights) : I8L_DTYPE_F32, y.data_ptr(), stream_of(dev)),
        dev);
  return y;
}
bool ints(const Tensor& t, const Tensor& like, at::IntArrayRef shape) {
  return t.scalar_type() == at::kInt && dense(t) && t.device() == like.device() && t.sizes() == shape;
}
// A gradient that came in, contiguous.
Tensor incoming(const char* name, const Tensor& d) {
  TORCH_CHECK_NOT_IMPLEMENTED(!forward_mode(d), "the gradient of ", name, " has no forward-mode derivative");
  return d.contiguous();
}
// The gradients have no gradient of their own: where a graph of them is made, going back through it is an error.
Tensor once(const char* name, const Tensor& result, const Tensor& dy) {
  if (!result.defined() || !at::GradMode::is_enabled() || !dy.requires_grad()) return result;
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate twice ") + name + ", which has a first gradient only", 1);
  return (*error)({result.detach().requires_grad_(true)})[0];
}

// The Python path of both backward passes, for what the native one does not take; it makes contiguous what is not and refuses what does not
// fit.  rows undefined: sort_tokens'.
variable_list combine_backward_in_python(const Tensor& rows, const Tensor& weights, const Tensor& pos, const Tensor& src, const Tensor& dy,
                                         bool need_rows, bool need_weights) {
  const WithGil gil;
  auto wrap = [](const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t.detach());
  };
  PyObject* r = PyObject_CallFunction(py_combine_backward, "NNNNNii", wrap(rows), wrap(weights), wrap(pos), wrap(src), wrap(dy), (int)need_rows,
                                      (int)need_weights);
  if (!r) throw_python_error();
  PyObject *a = nullptr, *b = nullptr;
  const int ok = PyArg_ParseTuple(r, "OO", &a, &b);
  variable_list grads(2);
  if (ok && THPVariable_Check(a)) grads[0] = THPVariable_Unpack(a);
  if (ok && THPVariable_Check(b)) grads[1] = THPVariable_Unpack(b);
  Py_DECREF(r);
  if (!ok) throw_python_error();
  return grads;
}

struct SortNode : torch::autograd::Function<SortNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& ids, int64_t experts, int64_t align) {
    const Sorted s = sort_tokens(x, ids, (int)experts, align);
    ctx->mark_non_differentiable({s.offsets, s.pos, s.src});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({s.pos});
    return {s.rows, s.offsets, s.pos, s.src};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor pos = ctx->get_saved_variables()[0], dy = incoming("sort_tokens", grads[0]);
    const bool ok = plain_thread() && dense(dy) && pos.dim() == 2 && ints(pos, dy, pos.sizes());
    const Tensor dx = ok ? combine(dy.detach(), Tensor(), pos) : combine_backward_in_python(Tensor(), Tensor(), pos, Tensor(), dy, true, false)[0];
    return {once("sort_tokens", dx, grads[0]), Tensor(), Tensor(), Tensor()};   // the sum of a token's rows
  }
};

struct CombineNode : torch::autograd::Function<CombineNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& pos, const Tensor& src) {
    ctx->save_for_backward({rows, weights, pos, src});
    return combine(rows, weights, pos);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &weights = saved[1], &pos = saved[2], &src = saved[3], dy = incoming("combine", grads[0]);
    const bool need_rows = ctx->needs_input_grad(0), need_weights = ctx->needs_input_grad(1);
    Tensor drows, dweights;
    if (plain_thread() && dense(dy) && dense(rows) && rows.dim() == 2 && rows.scalar_type() == dy.scalar_type() &&
        rows.device() == dy.device() && rows.size(1) == dy.size(1) && dense(weights) && weights.dim() == 2 && weights.size(0) == dy.size(0) && weights.device() == dy.device() &&
        (weights.scalar_type() == at::kFloat || weights.scalar_type() == dy.scalar_type()) && ints(pos, dy, weights.sizes()) &&
        ints(src, dy, {rows.size(0)})) {
      const int64_t T = pos.size(0), k = pos.size(1), R = rows.size(0), H = rows.size(1);
      const int dev = rows.get_device();
      const c10::cuda::CUDAGuard guard(dev);
      if (need_rows) drows = at::empty({R, H}, rows.options());
      if (need_weights) dweights = at::empty({T, k}, weights.options());
      check("i8l_combine_backward",
            lib_combine_backward(rows.data_ptr(), weights.data_ptr(), at_of<int32_t>(pos), at_of<int32_t>(src), dy.data_ptr(), R, T, H, (int)k,
                                 dtype_of(rows), dtype_of(weights), drows.defined() ? drows.data_ptr() : nullptr,
                                 dweights.defined() ? dweights.data_ptr() : nullptr, stream_of(dev)),
            dev);
    } else {   // a mode that the forward pass did not see, or hooks on saved tensors, which give back what they like
      const variable_list r = combine_backward_in_python(rows, weights, pos, src, dy, need_rows, need_weights);
      drows = r[0];
      dweights = r[1];
    }
    // a graph of the gradients would lead to dy, the rows and the weights alike
    const Tensor& any = rows.requires_grad() ? rows : weights.requires_grad() ? weights : grads[0];
    return {once("combine", drows, any), once("combine", dweights, any), Tensor(), Tensor()};
  }
};

Tensor token_linear(const Tensor& x, const Tensor& wq, const Tensor& ws, const Tensor& offsets, const Tensor& bias, int64_t E, bool f32) {
  const int64_t N = wq.size(-2), K = wq.size(-1), R = x.numel() / K;
  const int dev = x.get_device();
  const c10::cuda::CUDAGuard guard(dev);
  Status& status = status_of(dev);
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty(shape, x.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  const int64_t size = lib_token_workspace(R, (int)E, N, K);
  const Tensor work = size ? bytes(size, x) : Tensor();
  check("i8l_token_linear",
        lib_token_linear(x.data_ptr(), at_of<int8_t>(wq), at_of<float>(ws), offsets.defined() ? at_of<int32_t>(offsets) : nullptr,
                         bias.defined() ? bias.data_ptr() : nullptr, y.data_ptr(), R, (int)E, N, K, f32 ? I8L_GEMM_OUT_F32 : 0,
                         size ? work.data_ptr() : nullptr, size, status.word.load(std::memory_order_relaxed), stream_of(dev)),
        dev);
  return y;
}

// ------------------------------------------------------------------------------------------------ Python
bool exact_tensor(PyObject* o) { return THPVariable_CheckExact(o); }
bool at_16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// sort_tokens(x, ids, experts, align) -> (rows, offsets, pos, src), or None
PyObject* py_sort_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "sort_tokens takes 4 arguments");
    return nullptr;
  }
  if (!exact_tensor(args[0]) || !exact_tensor(args[1])) Py_RETURN_NONE;
  const Tensor x = THPVariable_Unpack(args[0]), ids = THPVariable_Unpack(args[1]);
  const long long experts = PyLong_AsLongLong(args[2]), align = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  constexpr int64_t MOST = 1ll << 30;   // sizes whose products fit 64 bits; the library refuses what is too large for it
  if (!plain_thread() || !dense(x) || dtype_of(x) < 0 || x.dim() != 2 || !dense(ids) || ids.dim() != 2 || ids.device() != x.device() ||
      (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || ids.size(0) != x.size(0) || x.size(0) > MOST || ids.size(1) > MOST ||
      experts < 1 || experts > 1024 || align < 1 || align > 65536 || forward_mode(x))
    Py_RETURN_NONE;
  Sorted s;
  {
    const WithoutGil no_gil;
    if (at::GradMode::is_enabled() && x.requires_grad()) {
      const variable_list r = SortNode::apply(x, ids, (int64_t)experts, (int64_t)align);
      s = Sorted{r[0], r[1], r[2], r[3]};
    } else {
      const at::AutoGradMode off(false);
      s = sort_tokens(x, ids, (int)experts, align);
    }
  }
  return Py_BuildValue("NNNN", THPVariable_Wrap(s.rows), THPVariable_Wrap(s.offsets), THPVariable_Wrap(s.pos), THPVariable_Wrap(s.src));
  END_HANDLE_TH_ERRORS
}

// combine(rows, weights, pos, src) -> y, or None
PyObject* py_combine(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "combine takes 4 arguments");
    return nullptr;
  }
  for (int i = 0; i < 4; ++i)
    if (!exact_tensor(args[i])) Py_RETURN_NONE;
  const Tensor rows = THPVariable_Unpack(args[0]), weights = THPVariable_Unpack(args[1]), pos = THPVariable_Unpack(args[2]),
               src = THPVariable_Unpack(args[3]);
  if (!plain_thread() || !dense(rows) || dtype_of(rows) < 0 || rows.dim() != 2 || !dense(weights) || weights.dim() != 2 ||
      (weights.scalar_type() != at::kFloat && weights.scalar_type() != rows.scalar_type()) || weights.device() != rows.device() ||
      !ints(pos, rows, weights.sizes()) || !ints(src, rows, {rows.size(0)}) || forward_mode(rows) || forward_mode(weights))
    Py_RETURN_NONE;
  Tensor y;
  {
    const WithoutGil no_gil;
    if (at::GradMode::is_enabled() && (rows.requires_grad() || weights.requires_grad())) y = CombineNode::apply(rows, weights, pos, src);
    else {
      const at::AutoGradMode off(false);
      y = combine(rows, weights, pos);
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// token_linear(x, wq, ws, offsets or None, bias or None, fp32 output) -> y, or None.  wq [N, K] without offsets, [E, N, K] with them.
PyObject* py_token_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "token_linear takes 6 arguments");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i)
    if (!exact_tensor(args[i]) && !(i >= 3 && args[i] == Py_None)) Py_RETURN_NONE;
  const Tensor x = THPVariable_Unpack(args[0]), wq = THPVariable_Unpack(args[1]), ws = THPVariable_Unpack(args[2]);
  Tensor offsets, bias;
  if (args[3] != Py_None) offsets = THPVariable_Unpack(args[3]);
  if (args[4] != Py_None) bias = THPVariable_Unpack(args[4]);
  const int dims = offsets.defined() ? 3 : 2;
  if (!plain_thread() || !plain(x) || !dense(wq) || !dense(ws) || wq.scalar_type() != at::kChar || ws.scalar_type() != at::kFloat ||
      wq.dim() != dims || (dims == 3 ? x.dim() != 2 : x.dim() < 1) || x.size(-1) != wq.size(-1) || wq.size(-1) == 0 ||
      ws.sizes() != wq.sizes().slice(0, dims - 1) || wq.device() != x.device() || ws.device() != x.device() ||
      (offsets.defined() && !ints(offsets, x, {wq.size(0) + 1})) || wq.size(0) > 65536 * (dims == 2 ? 65536ll : 1) ||
      (bias.defined() && (!plain(bias) || bias.device() != x.device() || bias.sizes() != ws.sizes() || !at_16(bias))) || !at_16(x) || !at_16(wq) ||
      forward_mode(x) || forward_mode(ws) || (bias.defined() && forward_mode(bias)) ||
      (at::GradMode::is_enabled() && (x.requires_grad() || ws.requires_grad() || (bias.defined() && bias.requires_grad()))))
    Py_RETURN_NONE;
  Tensor y;
  {
    const WithoutGil no_gil;
    report_timeout(x.get_device());
    const at::AutoGradMode off(false);
    y = token_linear(x, wq, ws, offsets, bias, dims == 3 ? wq.size(0) : 1, args[5] == Py_True);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// linear(x, weight, bias or None, gran, qmode, hadamard, flags, whole_k) -> y, or None
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "linear takes 8 arguments");
    return nullptr;
  }
  if (!exact_tensor(args[0]) || !exact_tensor(args[1]) || (args[2] != Py_None && !exact_tensor(args[2]))) Py_RETURN_NONE;
  const Tensor x = THPVariable_Unpack(args[0]), weight = THPVariable_Unpack(args[1]);
  std::optional<Tensor> bias;
  if (args[2] != Py_None) bias = THPVariable_Unpack(args[2]);
  const Config c{(int)PyLong_AsLong(args[3]), (int)PyLong_AsLong(args[4]), (int)PyLong_AsLong(args[5]), (int)PyLong_AsLong(args[6]),
                 args[7] == Py_True};
  if (PyErr_Occurred()) return nullptr;
  if ((c.hadamard != 0 && c.hadamard != 128) || !plain_thread() || !plain(x) || !plain(weight) || x.dim() < 1 || weight.dim() != 2 ||
      x.numel() == 0 || weight.numel() == 0 || x.size(-1) != weight.size(1) || weight.device() != x.device() ||
      (bias && !plain_bias(*bias, x, weight.size(0))) || x._fw_grad(0).defined() || weight._fw_grad(0).defined() ||
      (bias && bias->_fw_grad(0).defined()))
    Py_RETURN_NONE;
  Tensor y;
  {
    const WithoutGil no_gil;
    report_timeout(x.get_device());
    const bool grad = at::GradMode::is_enabled();
    if (grad && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad())))
      y = Int8LinearNode::apply(x, weight, bias, c.code(), weight.requires_grad());
    else {
      const at::AutoGradMode off(false);   // as inside the node: a view made here is one made without gradients
      y = linear_forward(x, weight, bias ? &*bias : nullptr, c, nullptr);
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// quant_gemm(a, b, a_gran, b_gran, qmode, hadamard, bias or None, post_scale, flags, want_at) -> (out, (qt, st)), or None
PyObject* py_quant_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "quant_gemm takes 10 arguments");
    return nullptr;
  }
  if (!exact_tensor(args[0]) || !exact_tensor(args[1]) || (args[6] != Py_None && !exact_tensor(args[6]))) Py_RETURN_NONE;
  const Tensor a = THPVariable_Unpack(args[0]), b = THPVariable_Unpack(args[1]);
  Tensor bias;
  if (args[6] != Py_None) bias = THPVariable_Unpack(args[6]);
  const int a_gran = (int)PyLong_AsLong(args[2]), b_gran = (int)PyLong_AsLong(args[3]), qmode = (int)PyLong_AsLong(args[4]),
            hadamard = (int)PyLong_AsLong(args[5]), flags = (int)PyLong_AsLong(args[8]), want = PyObject_IsTrue(args[9]);
  const double post = PyFloat_AsDouble(args[7]);
  if (PyErr_Occurred()) return nullptr;
  if (!plain_thread() || !plain(a) || !plain(b) || a.dim() != 3 || (b.dim() != 2 && b.dim() != 3) || a.numel() == 0 || b.numel() == 0 ||
      b.size(-1) != a.size(2) || (b.dim() == 3 && b.size(0) != a.size(0)) || b.device() != a.device() ||
      (bias.defined() && !plain_bias(bias, a, b.size(-2))))
    Py_RETURN_NONE;
  Transposed t;
  Tensor out;
  {
    const WithoutGil no_gil;
    out = quant_gemm(a, a.size(0), a.size(1), b, b.dim() == 3, a_gran, b_gran, qmode, hadamard, bias.defined() ? &bias : nullptr, post,
                     flags, want ? &t : nullptr);
  }
  if (!want) return Py_BuildValue("N(OO)", THPVariable_Wrap(out), Py_None, Py_None);
  return Py_BuildValue("N(NN)", THPVariable_Wrap(out), THPVariable_Wrap(t.q), THPVariable_Wrap(t.scale));
  END_HANDLE_TH_ERRORS
}

// setup(address of i8l_quant_gemm, of i8l_linear_backward_bias, of i8l_status_peek, on_error, on_timeout, open_status, py_backward)
PyObject* py_setup(PyObject*, PyObject* args) {
  unsigned long long qg = 0, lb = 0, sp = 0;
  PyObject *err = nullptr, *timeout = nullptr, *open = nullptr, *bwd = nullptr;
  if (!PyArg_ParseTuple(args, "KKKOOOO", &qg, &lb, &sp, &err, &timeout, &open, &bwd)) return nullptr;
  lib_quant_gemm = reinterpret_cast<decltype(lib_quant_gemm)>(qg);
  lib_linear_backward = reinterpret_cast<decltype(lib_linear_backward)>(lb);
  lib_status_peek = reinterpret_cast<decltype(lib_status_peek)>(sp);
  Py_INCREF(err);
  Py_INCREF(timeout);
  Py_INCREF(open);
  Py_INCREF(bwd);
  on_error = err;
  on_timeout = timeout;
  open_status = open;
  py_backward = bwd;
  Py_RETURN_NONE;
}

// setup_experts(addresses of i8l_sort_workspace, i8l_sort_tokens, i8l_combine, i8l_combine_backward, i8l_token_linear_workspace,
// i8l_token_linear, combine_backward_in_python)
PyObject* py_setup_experts(PyObject*, PyObject* args) {
  unsigned long long a[6];
  PyObject* backward = nullptr;
  if (!PyArg_ParseTuple(args, "KKKKKKO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &backward)) return nullptr;
  Py_INCREF(backward);
  Py_XDECREF(py_combine_backward);
  py_combine_backward = backward;
  lib_sort_workspace = reinterpret_cast<decltype(lib_sort_workspace)>(a[0]);
  lib_sort_tokens = reinterpret_cast<decltype(lib_sort_tokens)>(a[1]);
  lib_combine = reinterpret_cast<decltype(lib_combine)>(a[2]);
  lib_combine_backward = reinterpret_cast<decltype(lib_combine_backward)>(a[3]);
  lib_token_workspace = reinterpret_cast<decltype(lib_token_workspace)>(a[4]);
  lib_token_linear = reinterpret_cast<decltype(lib_token_linear)>(a[5]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"setup", py_setup, METH_VARARGS, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_linear)), METH_FASTCALL, nullptr},
    {"quant_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_quant_gemm)), METH_FASTCALL, nullptr},
    {"setup_experts", py_setup_experts, METH_VARARGS, nullptr},
    {"sort_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_sort_tokens)), METH_FASTCALL, nullptr},
    {"combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_combine)), METH_FASTCALL, nullptr},
    {"token_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_token_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "abi", I8L_HOST_ABI)) Py_CLEAR(m);   // see host_abi in build.py
  return m;
}
