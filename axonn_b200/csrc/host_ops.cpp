// Host paths of the operators that short calls are bound by: the same launches as the Python code beside them (ops/norm.py,
// ops/attention_cuda.py, ops/kv_cache.py, ops/beam.py, ops/token_probs.py, ops/embedding.py, intra_layer/fully_connected.py), with the questions
// asked and the tensors allocated in C++, and the autograd nodes of the normalisation, the token log-probabilities and the table lookup in
// C++, so that neither their backward nor the launches of a layer wait for the interpreter.
//
// A function returns None where the call is not one of those it takes; the caller then goes its general way, which accepts or
// refuses it.  Nothing is kept from one call to the next.  The kernels are those of the library that ops/_lib.py has loaded: bind()
// is given the addresses of its launchers.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/autocast_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <string>

#include "axonn_b200.h"

namespace {

using at::Tensor;
using std::optional;

// Launchers of the kernel library, of the types that its header gives them; bind() fills them in.  The header's number comes from
// the build, and a library of another one is not bound.
#define AXB_LAUNCHERS(X) \
  X(axb_norm_fwd, norm_fwd) X(axb_norm_bwd, norm_bwd) X(axb_add_norm_fwd, add_norm_fwd) X(axb_add_norm_bwd, add_norm_bwd) \
  X(axb_norm_grid, norm_grid) X(axb_gemm, gemm) X(axb_flash_attn_fwd, flash_fwd) X(axb_last_error, last_error) \
  X(axb_plan_blocks, plan_blocks) X(axb_store_blocks, store_blocks) X(axb_reorder_blocks, reorder_blocks) \
  X(axb_cached_attention_words, attention_words) X(axb_cached_attention, cached_attention) \
  X(axb_beam_select_words, beam_words) X(axb_beam_select, beam_select) \
  X(axb_token_log_probs, token_log_probs) X(axb_token_log_probs_bwd, token_log_probs_bwd) \
  X(axb_embedding_sorted_words, embedding_sorted_words) X(axb_embedding, embedding) X(axb_embedding_grad_words, embedding_grad_words) X(axb_embedding_grad, embedding_grad)
#define AXB_DECLARE(symbol, name) decltype(&::symbol) name = nullptr;
AXB_LAUNCHERS(AXB_DECLARE)
PyObject *kernel_error = nullptr, *parameter_type = nullptr;
std::atomic<long long> launches{0};

struct KernelError : torch::PyTorchError {
  explicit KernelError(const std::string& what) : torch::PyTorchError(what) {}
  PyObject* python_type() override { return kernel_error; }
};

void check(int status, const char* what, int count = 1) {
  if (status != 0) {
    const char* msg = last_error();
    throw KernelError(std::string(what) + " failed (status " + std::to_string(status) + "): " + (msg ? msg : ""));
  }
  launches += count;
}

int dtype_code(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : t.scalar_type() == at::kFloat ? 2 : -1;
}
const void* addr(const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }
// The norm kernels read 16 bytes at a time.
bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor dense(const Tensor& t) {
  const Tensor d = t.contiguous();
  return on_16_bytes(d) ? d : d.clone();
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// Other Python threads run while this one allocates (the allocator may have to free blocks, which synchronises) and launches (a full
// launch queue lets the caller wait).
struct NoGil {
  PyThreadState* const state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// An ordinary CUDA tensor or parameter.
bool plain(PyObject* o) {
  return (Py_TYPE(o) == reinterpret_cast<PyTypeObject*>(THPVariableClass) || Py_TYPE(o) == reinterpret_cast<PyTypeObject*>(parameter_type)) &&
         THPVariable_Unpack(o).is_cuda();
}
// Neither a tracer nor a function transform looks at the call (the caller has asked for forward-mode levels and compilation).
bool observed() {
  const auto keys = c10::impl::tls_local_dispatch_key_set().included_;
  return keys.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || keys.has(c10::DispatchKey::FuncTorchDynamicLayerBackMode) ||
         torch::jit::tracer::isTracing();
}

// ---------------------------------------------------------------------------------------------------------------- norms
// y = norm(x), or h = x + delta and norm(h); stats [rows, 2] receives mean and reciprocal deviation of the rows.
void run_norm(const Tensor& x, const optional<Tensor>& delta, const Tensor& gamma, const optional<Tensor>& beta, double eps, bool rms,
              Tensor& h, Tensor& y, Tensor& stats) {
  const int H = static_cast<int>(x.size(-1)), rows = static_cast<int>(x.numel() / H), device = x.get_device();
  y = at::empty_like(x);
  stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  if (delta) {
    h = at::empty_like(x);
    check(add_norm_fwd(x.data_ptr(), delta->data_ptr(), h.data_ptr(), gamma.data_ptr(), addr(beta), y.data_ptr(), stats.data_ptr<float>(),
                       rows, H, H, static_cast<float>(eps), rms, 0, dtype_code(x), device, stream()), "axb_add_norm_fwd");
  } else {
    h = x;
    check(norm_fwd(x.data_ptr(), gamma.data_ptr(), addr(beta), y.data_ptr(), stats.data_ptr<float>(), rows, H, H, static_cast<float>(eps),
                   rms, 0, dtype_code(x), device, stream()), "axb_norm_fwd");
  }
}

// A gradient that stands for many (is_grads_batched, vectorised Jacobians) is a wrapper without memory of its own.
bool batched(const Tensor& t) { return t.defined() && !t.has_storage(); }

// Node::gradients() of kernels that leave no graph: differentiating them again is an error (first_derivative_only in ops/direct.py).
template <typename Node>
torch::autograd::variable_list first_derivative(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads, const char* why) {
  if (!at::GradMode::is_enabled()) return Node::gradients(ctx, grads);
  torch::autograd::variable_list out, inputs = ctx->get_saved_variables();
  {
    at::AutoGradMode no_grad(false);
    out = Node::gradients(ctx, grads);
  }
  inputs.insert(inputs.end(), grads.begin(), grads.end());
  if (!std::any_of(inputs.begin(), inputs.end(), [](const Tensor& t) { return t.defined() && t.requires_grad(); })) return out;
  const auto node = std::make_shared<torch::autograd::Error>(why, torch::autograd::collect_next_edges(inputs));
  for (Tensor& t : out)
    if (t.defined()) torch::autograd::set_history(t = t.detach(), node);
  return out;
}

// Inputs: x, delta (may be missing), gamma, beta (may be missing).  Outputs: y, or h and y.
struct NormNode : torch::autograd::Function<NormNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const optional<Tensor>& delta,
                                                const Tensor& gamma, const optional<Tensor>& beta, double eps, bool rms) {
    Tensor h, y, stats;
    run_norm(x, delta, gamma, beta, eps, rms, h, y, stats);
    ctx->save_for_backward({h, gamma, stats});
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["beta"] = beta.has_value();
    ctx->saved_data["delta"] = delta.has_value();
    if (delta) return {h, y};
    return {y};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    return first_derivative<NormNode>(ctx, grads, "Norm: second derivatives are not implemented");
  }
  static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    // what hooks (offloading, compression) give back may lie in another layout
    const Tensor h = dense(saved[0]), gamma = dense(saved[1]), stats = dense(saved[2]);
    const bool rms = ctx->saved_data["rms"].toBool(), delta = ctx->saved_data["delta"].toBool();
    const Tensor dy = dense(grads[delta ? 1 : 0]);
    const int H = static_cast<int>(h.size(-1)), rows = static_cast<int>(stats.size(0)), device = h.get_device();
    const int grid = norm_grid(device, rows);
    Tensor dx = at::empty_like(h), part = at::empty({2, grid, H}, stats.options()), dgamma = at::empty_like(gamma), dbeta;
    if (!rms) dbeta = at::empty_like(gamma);
    float* pa = part.data_ptr<float>();
    float* pb = pa + static_cast<size_t>(grid) * H;
    void* db = rms ? nullptr : dbeta.data_ptr();
    if (delta) {
      const Tensor dh = dense(grads[0]);
      check(add_norm_bwd(dy.data_ptr(), dh.data_ptr(), h.data_ptr(), gamma.data_ptr(), stats.data_ptr<float>(), dx.data_ptr(), nullptr, pa, pb,
                         dgamma.data_ptr(), db, rows, H, H, rms, 0, dtype_code(h), dtype_code(gamma), device, stream()),
            "axb_add_norm_bwd", 2);
    } else {
      check(norm_bwd(dy.data_ptr(), h.data_ptr(), gamma.data_ptr(), stats.data_ptr<float>(), dx.data_ptr(), nullptr, pa, pb, dgamma.data_ptr(),
                     db, rows, H, H, rms, 0, dtype_code(h), dtype_code(gamma), device, stream()), "axb_norm_bwd", 2);
    }
    return {dx, delta ? dx : Tensor(), dgamma, ctx->saved_data["beta"].toBool() ? dbeta : Tensor(), Tensor(), Tensor()};
  }
};

// norm(x, delta | None, gamma, beta | None, eps, rms) -> y, (h, y) with delta, or None
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !plain(a[0]) || !plain(a[2]) || (a[1] != Py_None && !plain(a[1])) || (a[3] != Py_None && !plain(a[3])) || observed()) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(a[0]), &gamma = THPVariable_Unpack(a[2]);
  optional<Tensor> delta, beta;
  if (a[1] != Py_None) delta = THPVariable_Unpack(a[1]);
  if (a[3] != Py_None) beta = THPVariable_Unpack(a[3]);
  const double eps = PyFloat_AsDouble(a[4]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  const bool rms = PyObject_IsTrue(a[5]) == 1;
  const auto type = x.scalar_type();
  if (x.dim() == 0 || x.numel() == 0 || dtype_code(x) < 0 || !x.is_contiguous()) Py_RETURN_NONE;
  const int64_t H = x.size(-1);
  if (H > INT32_MAX || x.numel() / H > INT32_MAX) Py_RETURN_NONE;
  for (const Tensor* v : {&gamma, beta ? &*beta : &gamma})
    if (v->scalar_type() != type || v->dim() != 1 || v->size(0) != H || !v->is_contiguous() || v->device() != x.device() || !on_16_bytes(*v)) Py_RETURN_NONE;
  if (!on_16_bytes(x) || (delta && !on_16_bytes(*delta))) Py_RETURN_NONE;
  if (delta && (delta->sizes() != x.sizes() || delta->scalar_type() != type || !delta->is_contiguous() || delta->device() != x.device())) Py_RETURN_NONE;
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || gamma.requires_grad() || (delta && delta->requires_grad()) ||
                                                   (beta && beta->requires_grad()));
  Tensor h, y, stats;
  {
    NoGil no_gil;
    if (grad) {
      const auto out = NormNode::apply(x, delta, gamma, beta, eps, rms);
      h = out[0];
      y = out[delta ? 1 : 0];
    } else {
      run_norm(x, delta, gamma, beta, eps, rms, h, y, stats);
    }
  }
  if (!delta) return THPVariable_Wrap(y);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(h));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(y));
  return pair;
  END_HANDLE_TH_ERRORS
}

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// -------------------------------------------------------------------------------------------------------------- a linear layer
// linear(x, weight [n * k], bias | None, n, k, gelu) -> gelu?(x @ weight.T + bias) without a graph, or None
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !plain(a[0]) || !plain(a[1]) || (a[2] != Py_None && !plain(a[2])) || observed()) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(a[0]), &w = THPVariable_Unpack(a[1]);
  optional<Tensor> b;
  if (a[2] != Py_None) b = THPVariable_Unpack(a[2]);
  const long rows_out = PyLong_AsLong(a[3]), k = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  const bool gelu = PyObject_IsTrue(a[5]) == 1;
  const auto type = w.scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || x.scalar_type() != type || x.dim() == 0 || x.size(-1) != k || rows_out % 8 || k % 8 ||
      x.numel() == 0 || x.numel() / k > INT32_MAX || w.dim() != 1 || w.size(0) != static_cast<int64_t>(rows_out) * k || !x.is_contiguous() ||
      !w.is_contiguous() || w.device() != x.device() || wants_grad(x) || wants_grad(w) || at::autocast::is_autocast_enabled(at::kCUDA))
    Py_RETURN_NONE;
  if (b && (b->scalar_type() != type || b->device() != x.device() || !b->is_contiguous() || b->numel() != rows_out || wants_grad(*b))) Py_RETURN_NONE;
  c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = rows_out;
  const int code = type == at::kBFloat16 ? 0 : 1, epilogue = gelu ? (b ? 2 : 3) : (b ? 1 : 0);
  Tensor out;
  {
    NoGil no_gil;
    out = at::empty(shape, x.options());
    check(gemm(0, x.data_ptr(), w.data_ptr(), out.data_ptr(), addr(b), nullptr, static_cast<int>(x.numel() / k), static_cast<int>(rows_out),
               static_cast<int>(k), code, code, epilogue, 0, x.get_device(), stream()), "axb_gemm");
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------------------------ attention
// attention(qkv [B, S, G, q_per_kv + 2, D], scale) -> causal attention without a graph, or None
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !plain(a[0]) || observed()) Py_RETURN_NONE;
  const Tensor& qkv = THPVariable_Unpack(a[0]);
  const double scale = PyFloat_AsDouble(a[1]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  if (qkv.dim() != 5 || qkv.scalar_type() != at::kBFloat16 || !qkv.is_contiguous() || qkv.numel() == 0 || wants_grad(qkv)) Py_RETURN_NONE;
  const int64_t B = qkv.size(0), S = qkv.size(1), G = qkv.size(2), qpk = qkv.size(3) - 2, D = qkv.size(4);
  // 2^-100 < scale < 2^100, dense and on 16 bytes: see supported() in ops/attention_cuda.py
  if (qpk < 1 || (D != 64 && D != 128) || !(scale > 0x1p-100 && scale < 0x1p100) || reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 ||
      std::max({B, S, G, qpk}) > INT32_MAX) Py_RETURN_NONE;
  Tensor out;
  {
    NoGil no_gil;
    out = at::empty({B, S, G * qpk, D}, qkv.options());
    const Tensor lse = at::empty({B, G * qpk, S}, qkv.options().dtype(at::kFloat));
    check(flash_fwd(qkv.data_ptr(), out.data_ptr(), lse.data_ptr<float>(), static_cast<int>(B), static_cast<int>(S), static_cast<int>(G),
                    static_cast<int>(qpk), static_cast<int>(D), static_cast<float>(scale), qkv.get_device(), stream()), "axb_flash_attn_fwd");
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------- block cache
// Dense, of the type and the shape.
bool is(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape) {
  return t.scalar_type() == type && t.sizes() == at::IntArrayRef(shape) && t.is_contiguous();
}
bool block_size(int64_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }

// The tensors of the arguments named, all on the current device, none with a gradient to be had; where the second of a pair says so,
// None may stand there and gives an undefined tensor.
bool take_tensors(PyObject* const* a, std::initializer_list<std::pair<int, bool>> which, Tensor* out) {
  const int device = c10::cuda::current_device();
  for (const auto& [i, missing] : which) {
    if (missing && a[i] == Py_None) { *out++ = Tensor(); continue; }
    if (!plain(a[i])) return false;
    *out = THPVariable_Unpack(a[i]);
    if (out->get_device() != device || wants_grad(*out)) return false;
    ++out;
  }
  return true;
}

// Codes and scales of a layer (dims 4) or of stacked layers (5), as the kernels take them.
bool layer_ok(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int dims) {
  const auto type = k.scalar_type();
  if ((type != at::kFloat8_e4m3fn && type != at::kChar) || v.scalar_type() != type || k.dim() != dims || v.sizes() != k.sizes() || k.numel() == 0 ||
      !block_size(k.size(dims - 2)) || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || ks.dim() != dims - 2 ||
      vs.dim() != dims - 2 || !k.is_contiguous() || !v.is_contiguous() || !ks.is_contiguous() || !vs.is_contiguous() || !on_16_bytes(k) || !on_16_bytes(v))
    return false;
  for (int i = 0; i < dims - 2; ++i)
    if (ks.size(i) != k.size(i) || vs.size(i) != k.size(i)) return false;
  for (int i = 0; i < dims; ++i)
    if (k.size(i) > INT32_MAX) return false;
  return true;
}

PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) { Py_DECREF(tuple); return nullptr; }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// plan_blocks(lengths, new, tables, free, taken, tokens, block_tokens) -> (slots, positions, lengths, taken) or None
PyObject* py_plan_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[5];
  if (n != 7 || observed() || !take_tensors(a, {{0, false}, {1, false}, {2, false}, {3, false}, {4, false}}, t)) Py_RETURN_NONE;
  const auto& [lengths, fresh, tables, free_blocks, taken] = t;
  const long tokens = PyLong_AsLong(a[5]), block = PyLong_AsLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (lengths.dim() != 1 || tables.dim() != 2 || free_blocks.dim() != 1) Py_RETURN_NONE;
  const int64_t R = lengths.size(0), W = tables.size(1), N = free_blocks.size(0);
  if (R == 0 || W == 0 || N == 0 || tokens <= 0 || std::max({R, W * block, N, static_cast<int64_t>(tokens)}) > INT32_MAX || !block_size(block) ||
      !is(lengths, at::kInt, {R}) || !is(fresh, at::kInt, {R}) || !is(tables, at::kInt, {R, W}) || !is(free_blocks, at::kInt, {N}) ||
      !is(taken, at::kInt, {1}))
    Py_RETURN_NONE;
  Tensor slots, positions, after, used;
  {
    NoGil no_gil;
    slots = at::empty({R, tokens}, lengths.options().dtype(at::kLong));
    positions = at::empty({R, tokens}, lengths.options());
    after = at::empty({R}, lengths.options());
    used = at::empty({1}, lengths.options());
    check(plan_blocks(lengths.data_ptr<int>(), fresh.data_ptr<int>(), tables.data_ptr<int>(), free_blocks.data_ptr<int>(), taken.data_ptr<int>(),
                      reinterpret_cast<long long*>(slots.data_ptr<int64_t>()), positions.data_ptr<int>(), after.data_ptr<int>(), used.data_ptr<int>(),
                      static_cast<int>(R), static_cast<int>(tokens), static_cast<int>(W), static_cast<int>(N), static_cast<int>(block), stream()),
          "axb_plan_blocks");
  }
  return tuple_of({slots, positions, after, used});
  END_HANDLE_TH_ERRORS
}

// Strides of rows, tokens and groups of [R, S, G, heads, D] with dense heads, as the kernels can read them.
bool head_strides(const Tensor& x, int64_t (&strides)[3]) {
  if (x.stride(4) != 1 || (x.stride(3) != x.size(4) && x.size(3) != 1) || !on_16_bytes(x)) return false;
  for (int i = 0; i < 3; ++i) {
    strides[i] = x.size(i) == 1 ? 0 : x.stride(i);
    if (strides[i] % 8) return false;
  }
  return true;
}

// store_blocks(qkv, k, v, k_scale, v_scale, slots, positions | None, rope table | None) -> (queries | None,) or None
PyObject* py_store_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[8];
  if (n != 8 || observed() ||
      !take_tensors(a, {{0, false}, {1, false}, {2, false}, {3, false}, {4, false}, {5, false}, {6, true}, {7, true}}, t)) Py_RETURN_NONE;
  const auto& [qkv, k, v, ks, vs, slots, positions, table] = t;
  if (!layer_ok(k, v, ks, vs, 4) || qkv.dim() != 5 || (qkv.scalar_type() != at::kBFloat16 && qkv.scalar_type() != at::kHalf)) Py_RETURN_NONE;
  const int64_t N = k.size(0), G = k.size(1), BT = k.size(2), D = k.size(3), R = qkv.size(0), S = qkv.size(1), P = qkv.size(3) - 2;
  int64_t strides[3];
  if (R == 0 || S == 0 || qkv.size(2) != G || P < 0 || qkv.size(4) != D || (D != 64 && D != 128) || std::max({R, S, P}) > INT32_MAX ||
      !is(slots, at::kLong, {R, S}) || qkv.size(3) == 1 || !head_strides(qkv, strides))
    Py_RETURN_NONE;
  const bool rope = table.defined();
  if (rope && (!positions.defined() || !is(positions, at::kInt, {R, S}) || table.dim() != 3 || !is(table, at::kFloat, {table.size(0), D / 2, 2}) ||
               table.size(0) > INT32_MAX || !on_16_bytes(table)))
    Py_RETURN_NONE;
  Tensor q;
  {
    NoGil no_gil;
    if (rope) q = at::empty({R, S, G * P, D}, qkv.options());
    check(store_blocks(qkv.data_ptr(), strides[0], strides[1], strides[2], reinterpret_cast<const long long*>(slots.data_ptr<int64_t>()),
                       rope ? positions.data_ptr<int>() : nullptr, rope ? table.data_ptr<float>() : nullptr, rope ? q.data_ptr() : nullptr,
                       k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), static_cast<int>(R), static_cast<int>(S),
                       static_cast<int>(G), static_cast<int>(P), static_cast<int>(D), static_cast<int>(N), static_cast<int>(BT),
                       rope ? static_cast<int>(table.size(0)) : 0, dtype_code(qkv), k.scalar_type() == at::kChar, stream()), "axb_store_blocks");
  }
  return tuple_of({q});
  END_HANDLE_TH_ERRORS
}

// cached_attention(q, k, v, k_scale, v_scale, tables, lengths, new | None, scale | None) -> output or None
PyObject* py_cached_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[8];
  if (n != 9 || observed() ||
      !take_tensors(a, {{0, false}, {1, false}, {2, false}, {3, false}, {4, false}, {5, false}, {6, false}, {7, true}}, t)) Py_RETURN_NONE;
  const auto& [given, k, v, ks, vs, tables, lengths, fresh] = t;
  if (!layer_ok(k, v, ks, vs, 4) || (given.scalar_type() != at::kBFloat16 && given.scalar_type() != at::kHalf)) Py_RETURN_NONE;
  const int64_t N = k.size(0), G = k.size(1), BT = k.size(2), D = k.size(3);
  Tensor q = given;
  if (q.dim() == 4) {
    if (q.size(2) % G || q.size(2) == 0 || (q.stride(2) != q.size(3) && q.size(2) != 1)) Py_RETURN_NONE;
    q = q.unflatten(2, {G, q.size(2) / G});
  }
  if (q.dim() != 5 || q.size(2) != G || q.size(4) != D || q.numel() == 0 || (D != 64 && D != 128) || tables.dim() != 2) Py_RETURN_NONE;
  const int64_t R = q.size(0), S = q.size(1), P = q.size(3), W = tables.size(1);
  int64_t strides[3];
  if (std::max({R, S * P, W}) > INT32_MAX || W == 0 || !head_strides(q, strides) || !is(tables, at::kInt, {R, W}) || !is(lengths, at::kInt, {R}) ||
      (fresh.defined() && !is(fresh, at::kInt, {R})))
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt(static_cast<double>(D));
  if (a[8] != Py_None) {
    scale = PyFloat_AsDouble(a[8]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!std::isfinite(scale)) Py_RETURN_NONE;
  }
  Tensor out;
  {
    NoGil no_gil;
    out = at::empty({R, S, G * P, D}, q.options());
    const Tensor work = at::empty({attention_words(static_cast<int>(R), static_cast<int>(S), static_cast<int>(G), static_cast<int>(P), static_cast<int>(D))},
                                  q.options().dtype(at::kFloat));
    check(cached_attention(q.data_ptr(), strides[0], strides[1], strides[2], k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(),
                           tables.data_ptr<int>(), lengths.data_ptr<int>(), fresh.defined() ? fresh.data_ptr<int>() : nullptr, out.data_ptr(),
                           work.data_ptr(), static_cast<int>(R), static_cast<int>(S), static_cast<int>(G), static_cast<int>(P), static_cast<int>(D),
                           static_cast<int>(W), static_cast<int>(N), static_cast<int>(BT), static_cast<float>(scale), dtype_code(q),
                           k.scalar_type() == at::kChar, stream()), "axb_cached_attention", 2);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// reorder_blocks(k, v, k_scale, v_scale, tables, lengths, spare, parents) -> (tables, lengths, spare) or None
PyObject* py_reorder_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[8];
  if (n != 8 || observed() ||
      !take_tensors(a, {{0, false}, {1, false}, {2, false}, {3, false}, {4, false}, {5, false}, {6, false}, {7, false}}, t)) Py_RETURN_NONE;
  const auto& [k, v, ks, vs, tables, lengths, spare, parents] = t;
  if (!layer_ok(k, v, ks, vs, 5) || tables.dim() != 2 || parents.dim() != 2) Py_RETURN_NONE;
  const int64_t R = tables.size(0), W = tables.size(1), K = parents.size(1);
  if (R == 0 || W == 0 || parents.numel() != R || std::max(R, W) > INT32_MAX || k.size(4) % 16 || !is(tables, at::kInt, {R, W}) ||
      !is(lengths, at::kInt, {R}) || !is(spare, at::kInt, {R}) || !is(parents, at::kInt, {R / K, K}))
    Py_RETURN_NONE;
  Tensor out[3];
  {
    NoGil no_gil;
    out[0] = at::empty({R, W}, tables.options());
    out[1] = at::empty({R}, tables.options());
    out[2] = at::empty({R}, tables.options());
    check(reorder_blocks(k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), tables.data_ptr<int>(), lengths.data_ptr<int>(),
                         spare.data_ptr<int>(), parents.data_ptr<int>(), out[0].data_ptr<int>(), out[1].data_ptr<int>(), out[2].data_ptr<int>(),
                         static_cast<int>(k.size(0)), static_cast<int>(R), static_cast<int>(K), static_cast<int>(W), static_cast<int>(k.size(1)),
                         static_cast<int>(k.size(2)), static_cast<int>(k.size(3)), static_cast<int>(k.size(4)), stream()), "axb_reorder_blocks");
  }
  return tuple_of({out[0], out[1], out[2]});
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------- beam search
// beam_select(logits, scores, done | None, eos | None) -> (scores, tokens, parents, done | None) or None
PyObject* py_beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[3];
  if (n != 4 || observed() || !take_tensors(a, {{0, false}, {1, false}, {2, true}}, t)) Py_RETURN_NONE;
  const auto& [logits, scores, done] = t;
  if (logits.dim() != 3 || dtype_code(logits) < 0 || !logits.is_contiguous() || logits.numel() == 0 || done.defined() == (a[3] == Py_None)) Py_RETURN_NONE;
  const int64_t B = logits.size(0), K = logits.size(1), V = logits.size(2);
  long eos = -1;
  if (done.defined()) {
    eos = PyLong_AsLong(a[3]);
    if (eos == -1 && PyErr_Occurred()) return nullptr;
    if (eos < 0 || eos >= V || !is(done, at::kBool, {B, K})) Py_RETURN_NONE;
  }
  if (K > 32 || V > (1 << 30) || B > INT32_MAX / K || !is(scores, at::kFloat, {B, K})) Py_RETURN_NONE;
  Tensor out_scores, tokens, parents, out_done;
  {
    NoGil no_gil;
    out_scores = at::empty({B, K}, scores.options());
    tokens = at::empty({B, K}, scores.options().dtype(at::kLong));
    parents = at::empty({B, K}, scores.options().dtype(at::kInt));
    if (done.defined()) out_done = at::empty({B, K}, done.options());
    const Tensor work = at::empty({beam_words(static_cast<int>(B), static_cast<int>(K), static_cast<int>(V), dtype_code(logits))},
                                  scores.options().dtype(at::kInt));
    check(beam_select(logits.data_ptr(), scores.data_ptr<float>(), done.defined() ? done.data_ptr() : nullptr, static_cast<int>(eos),
                      out_scores.data_ptr<float>(), reinterpret_cast<long long*>(tokens.data_ptr<int64_t>()), parents.data_ptr<int>(),
                      done.defined() ? out_done.data_ptr() : nullptr, work.data_ptr(), static_cast<int>(B), static_cast<int>(K),
                      static_cast<int>(V), dtype_code(logits), stream()), "axb_beam_select", 2);
  }
  return tuple_of({out_scores, tokens, parents, out_done});
  END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------------------------------------------- log-probabilities of tokens
// logits [(batches,) (rows,) V] whose last dimension is dense, with the strides of the other two; tokens likewise without the last.
struct TokenRows {
  int64_t batches = 1, per_batch = 1, batch_stride = 0, row_stride = 0, token_batch_stride = 0, token_stride = 0, V = 0;
  TokenRows(const Tensor& z, const Tensor& tokens) {
    const int64_t d = z.dim();
    V = z.size(d - 1);
    if (d > 1) { per_batch = z.size(d - 2); row_stride = z.stride(d - 2); if (tokens.defined()) token_stride = tokens.stride(d - 2); }
    if (d > 2) { batches = z.size(0); batch_stride = z.stride(0); if (tokens.defined()) token_batch_stride = tokens.stride(0); }
  }
};
const long long* words(const Tensor& t) { return t.defined() ? reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) : nullptr; }
long long* words_out(const Tensor& t) { return t.defined() ? reinterpret_cast<long long*>(t.data_ptr<int64_t>()) : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

struct TokenResults { Tensor log_probs, entropy, top_log_probs, top_tokens, stats; };
TokenResults run_token_log_probs(const Tensor& logits, const Tensor& tokens, bool entropy, int64_t top, double scale, int64_t ignored) {
  const TokenRows r(logits, tokens);
  const auto f32 = logits.options().dtype(at::kFloat);
  c10::SmallVector<int64_t, 5> shape(logits.sizes().begin(), logits.sizes().end() - 1);
  TokenResults out;
  if (tokens.defined()) out.log_probs = at::empty(shape, f32);
  if (entropy) out.entropy = at::empty(shape, f32);
  if (top) {
    shape.push_back(top);
    out.top_log_probs = at::empty(shape, f32);
    out.top_tokens = at::empty(shape, f32.dtype(at::kLong));
  }
  out.stats = at::empty({r.batches * r.per_batch, 4}, f32);
  check(token_log_probs(logits.data_ptr(), r.batch_stride, r.row_stride, words(tokens), r.token_batch_stride, r.token_stride, floats(out.log_probs),
                        floats(out.entropy), floats(out.top_log_probs), words_out(out.top_tokens), floats(out.stats), static_cast<int>(r.batches),
                        static_cast<int>(r.per_batch), static_cast<int>(r.V), 0, r.V, static_cast<int>(top), static_cast<float>(scale), ignored, 1,
                        dtype_code(logits), stream()), "axb_token_log_probs");
  return out;
}

// A node without the conveniences of torch::autograd::Function, which cost a short step 5 us (a table of named values, wrapped outputs).
template <typename Node> std::shared_ptr<Node> node_of(const Tensor& input) {
  std::shared_ptr<Node> node(new Node(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(input));
  return node;
}

// Outputs: those asked for of log_probs, entropy and top_log_probs.
struct TokenLogProbsNode : torch::autograd::Node {
  torch::autograd::SavedVariable logits, tokens, stats, top_tokens;
  bool has_tokens = false, entropy = false;
  int64_t top = 0, ignored = 0;
  double scale = 1;

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!std::any_of(grads.begin(), grads.end(), batched), "TokenLogProbs: batched gradients are not implemented");
    const Tensor z = logits.unpack(), t = has_tokens ? tokens.unpack() : Tensor(), s = stats.unpack(), best = top ? top_tokens.unpack() : Tensor();
    if (!at::GradMode::is_enabled()) return {gradient(z, t, s, best, grads)};
    Tensor out;
    {
      at::AutoGradMode no_grad(false);
      out = gradient(z, t, s, best, grads);
    }
    // the kernels leave no graph (first_derivative_only in ops/direct.py)
    torch::autograd::variable_list inputs(grads.begin(), grads.end());
    inputs.push_back(z);
    if (out.defined() && std::any_of(inputs.begin(), inputs.end(), [](const Tensor& x) { return x.defined() && x.requires_grad(); }))
      torch::autograd::set_history(out = out.detach(), std::make_shared<torch::autograd::Error>("TokenLogProbs: second derivatives are not implemented",
                                                                                              torch::autograd::collect_next_edges(inputs)));
    return {out};
  }
  Tensor gradient(const Tensor& given, const Tensor& t, const Tensor& s, const Tensor& best, const torch::autograd::variable_list& grads) {
    // what hooks (offloading, compression) give back may lie in another layout
    const Tensor z = given.dim() > 3 || (given.stride(-1) != 1 && given.size(-1) != 1) ? given.contiguous() : given;
    const Tensor by = dense(s), at_ = best.defined() ? best.contiguous() : best;
    size_t i = 0;
    Tensor d[3], out;
    const bool asked[3] = {has_tokens, entropy, top > 0};
    for (int k = 0; k < 3; ++k)
      if (asked[k]) {
        if (grads[i].defined()) d[k] = grads[i].contiguous();
        ++i;
      }
    if (d[0].defined() || d[1].defined() || d[2].defined()) {
      const TokenRows r(z, t);
      out = at::empty(z.sizes(), z.options());
      check(token_log_probs_bwd(z.data_ptr(), r.batch_stride, r.row_stride, words(t), r.token_batch_stride, r.token_stride, by.data_ptr<float>(),
                                floats(d[0]), floats(d[1]), floats(d[2]), words(at_), out.data_ptr(), static_cast<int>(r.batches),
                                static_cast<int>(r.per_batch), static_cast<int>(r.V), 0, r.V, static_cast<int>(top), static_cast<float>(scale), ignored,
                                dtype_code(z), ::stream()), "axb_token_log_probs_bwd");
    }
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data(); tokens.reset_data(); stats.reset_data(); top_tokens.reset_data();
  }
  std::string name() const override { return "TokenLogProbsBackward"; }
};

// token_log_probs(logits, tokens | None, entropy, top, 1 / temperature, ignore_index) -> (log_probs | None, entropy | None,
// top_log_probs | None, top_tokens | None) or None
PyObject* py_token_log_probs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !plain(a[0]) || (a[1] != Py_None && !plain(a[1])) || observed()) Py_RETURN_NONE;
  const Tensor& logits = THPVariable_Unpack(a[0]);
  const Tensor tokens = a[1] == Py_None ? Tensor() : THPVariable_Unpack(a[1]);
  const bool entropy = PyObject_IsTrue(a[2]) == 1;
  const long top = PyLong_AsLong(a[3]);
  const double scale = PyFloat_AsDouble(a[4]);
  const long long ignored = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t d = logits.dim();
  if (d == 0 || d > 3 || dtype_code(logits) < 0 || logits.numel() == 0 || logits.get_device() != c10::cuda::current_device() ||
      (logits.stride(d - 1) != 1 && logits.size(d - 1) != 1) || logits.size(d - 1) > (1 << 30) || logits.numel() / logits.size(d - 1) > INT32_MAX ||
      top < 0 || top > std::min<int64_t>(32, logits.size(d - 1)) || (!tokens.defined() && !entropy && !top) ||
      !(scale >= 0x1p-100 && scale <= 0x1p100))
    Py_RETURN_NONE;
  if (tokens.defined() && (tokens.scalar_type() != at::kLong || tokens.device() != logits.device() || tokens.sizes() != logits.sizes().slice(0, d - 1)))
    Py_RETURN_NONE;
  Tensor out[4];
  {
    NoGil no_gil;
    const TokenResults r = run_token_log_probs(logits, tokens, entropy, top, scale, ignored);
    out[0] = r.log_probs; out[1] = r.entropy; out[2] = r.top_log_probs; out[3] = r.top_tokens;
    if (wants_grad(logits)) {
      const auto node = node_of<TokenLogProbsNode>(logits);
      node->logits = torch::autograd::SavedVariable(logits, false);
      if (tokens.defined()) node->tokens = torch::autograd::SavedVariable(tokens, false);
      node->stats = torch::autograd::SavedVariable(r.stats, false);
      if (top) node->top_tokens = torch::autograd::SavedVariable(r.top_tokens, false);
      node->has_tokens = tokens.defined();
      node->entropy = entropy;
      node->top = top;
      node->ignored = ignored;
      node->scale = scale;
      for (int k = 0; k < 3; ++k)
        if (out[k].defined()) torch::autograd::set_history(out[k], node);
    }
  }
  return tuple_of({out[0], out[1], out[2], out[3]});
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------- table lookup
int index_bytes(const Tensor& tokens) { return tokens.scalar_type() == at::kLong ? 8 : tokens.scalar_type() == at::kInt ? 4 : 0; }

// With `sorted` also what the gradient needs of the tokens (nothing for few).
Tensor run_embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding = -1, Tensor* sorted = nullptr) {
  const Tensor t = tokens.contiguous(), w = weight.stride(1) != 1 && weight.size(1) != 1 ? weight.contiguous() : weight;
  const int V = static_cast<int>(w.size(0)), H = static_cast<int>(w.size(1));
  c10::SmallVector<int64_t, 5> shape(t.sizes().begin(), t.sizes().end());
  shape.push_back(H);
  const Tensor out = at::empty(shape, w.options());
  const int64_t count = sorted ? embedding_sorted_words(t.numel(), V) : 0;
  if (count) *sorted = at::empty({count}, w.options().dtype(at::kInt));
  if (out.numel())
    check(embedding(t.data_ptr(), index_bytes(t), t.numel(), w.data_ptr(), w.stride(0), V, H, static_cast<float>(scale), out.data_ptr(), padding,
                    count ? sorted->data_ptr() : nullptr, dtype_code(w), stream()), "axb_embedding", count ? 2 : 1);
  return out;
}
Tensor run_embedding_grad(const Tensor& tokens, const Tensor& sorted, const Tensor& dy, int64_t V, double scale, int64_t padding) {
  const int64_t H = dy.size(-1);
  Tensor rows = dy.dim() == 2 ? dy : dy.reshape({-1, H});
  if (rows.stride(1) != 1 && H != 1) rows = rows.contiguous();
  const int64_t n = rows.size(0);
  const Tensor out = at::empty({V, H}, rows.options()), t = tokens.contiguous(), by = sorted.defined() ? dense(sorted) : sorted;
  const int64_t count = embedding_grad_words(n, static_cast<int>(H));
  Tensor work;
  if (count) work = at::empty({count}, rows.options().dtype(at::kInt));
  check(embedding_grad(t.data_ptr(), index_bytes(t), by.defined() ? by.data_ptr() : nullptr, n, rows.data_ptr(), rows.stride(0), static_cast<int>(V),
                       static_cast<int>(H), static_cast<float>(scale), padding, out.data_ptr(), count ? work.data_ptr() : nullptr, dtype_code(rows),
                       stream()), "axb_embedding_grad", n == 0 ? 0 : count ? 2 : 1);
  return out;
}

// The gradient of the table as a function of that of the rows; and its own: rows of the table that it is asked with.
struct EmbeddingGradNode : torch::autograd::Function<EmbeddingGradNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& tokens, const optional<Tensor>& sorted, const Tensor& dy, int64_t V,
                        double scale, int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return run_embedding_grad(tokens, sorted ? *sorted : Tensor(), dy, V, scale, padding);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads);
};
// Of a gradient that stands for many, which torch's operators know.  Sums in 32 bits; tokens without a gradient go to a row behind the table's.
Tensor batched_embedding_grad(const Tensor& tokens, const Tensor& dy, int64_t V, double scale, int64_t padding) {
  const Tensor none = tokens.lt(0).logical_or(tokens.ge(V)).logical_or(tokens.eq(padding));
  const Tensor sums = at::embedding_dense_backward(dy.to(at::kFloat), tokens.to(at::kLong).masked_fill(none, V), V + 1, -1, false);
  return sums.narrow(0, 0, V).mul(scale).to(dy.scalar_type());
}
struct EmbeddingNode : torch::autograd::Node {
  torch::autograd::SavedVariable tokens, sorted;
  bool has_sorted = false;
  int64_t V = 0, padding = -1;
  double scale = 1;

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    const Tensor t = tokens.unpack(), s = has_sorted ? sorted.unpack() : Tensor();
    if (batched(grads[0]) || observed()) return {batched_embedding_grad(t, grads[0], V, scale, padding)};
    if (wants_grad(grads[0]))
      return {EmbeddingGradNode::apply(t, s.defined() ? optional<Tensor>(s) : std::nullopt, grads[0], V, scale, padding)};
    return {run_embedding_grad(t, s, grads[0], V, scale, padding)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens.reset_data(); sorted.reset_data();
  }
  std::string name() const override { return "EmbeddingRowsBackward"; }
};
Tensor embedding_with_graph(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  Tensor sorted;
  const Tensor out = run_embedding(tokens, weight, scale, padding, &sorted);
  const auto node = node_of<EmbeddingNode>(weight);
  node->tokens = torch::autograd::SavedVariable(tokens, false);
  if (sorted.defined()) node->sorted = torch::autograd::SavedVariable(sorted, false);
  node->has_sorted = sorted.defined();
  node->V = weight.size(0);
  node->padding = padding;
  node->scale = scale;
  torch::autograd::set_history(out, node);
  return out;
}
torch::autograd::variable_list EmbeddingGradNode::backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
  const Tensor tokens = ctx->get_saved_variables()[0], &table = grads[0];
  const double scale = ctx->saved_data["scale"].toDouble();
  const Tensor none = tokens.lt(0).logical_or(tokens.ge(table.size(0))).logical_or(tokens.eq(ctx->saved_data["padding"].toInt()));
  const Tensor there = tokens.masked_fill(none, 0);
  const Tensor rows = wants_grad(table) ? embedding_with_graph(there, table, scale, -1) : run_embedding(there, table, scale);
  return {Tensor(), Tensor(), rows.masked_fill(none.unsqueeze(-1), 0), Tensor(), Tensor(), Tensor()};
}

// embedding(tokens, weight [V, H], scale, padding | -1) -> weight[tokens] * scale or None
PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !plain(a[0]) || !plain(a[1]) || observed()) Py_RETURN_NONE;
  const Tensor &tokens = THPVariable_Unpack(a[0]), &weight = THPVariable_Unpack(a[1]);
  const double scale = PyFloat_AsDouble(a[2]);
  const long padding = PyLong_AsLong(a[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!index_bytes(tokens) || weight.dim() != 2 || dtype_code(weight) < 0 || weight.numel() == 0 || weight.size(0) > (1 << 30) ||
      weight.size(1) > (1 << 25) || tokens.numel() > INT32_MAX || tokens.device() != weight.device() ||
      weight.get_device() != c10::cuda::current_device() || !std::isfinite(scale) || !std::isfinite(static_cast<float>(scale)) || padding < -1 ||
      padding >= weight.size(0))
    Py_RETURN_NONE;
  Tensor out;
  {
    NoGil no_gil;
    out = wants_grad(weight) ? embedding_with_graph(tokens, weight, scale, padding) : run_embedding(tokens, weight, scale);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// bind({launcher name: address}, KernelError, Parameter, axb_interface() of the library they are from) -> False if it is another one
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 4 && PyDict_Check(a[0]), "bind(launchers, error type, parameter type, interface)");
  if (PyLong_AsUnsignedLong(a[3]) != AXB_INTERFACE) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_FALSE;
  }
  const auto take = [&](const char* symbol, auto& fn) {
    PyObject* v = PyDict_GetItemString(a[0], symbol);
    TORCH_CHECK(v, "launcher ", symbol, " is missing");
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(PyLong_AsVoidPtr(v));
  };
#define AXB_TAKE(symbol, name) take(#symbol, name);
  AXB_LAUNCHERS(AXB_TAKE)
  Py_INCREF(a[1]); Py_INCREF(a[2]);
  kernel_error = a[1]; parameter_type = a[2];
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_launches(PyObject*, PyObject*) { return PyLong_FromLongLong(launches.load()); }

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_bind)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_norm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention)), METH_FASTCALL, nullptr},
    {"plan_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_plan_blocks)), METH_FASTCALL, nullptr},
    {"store_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_store_blocks)), METH_FASTCALL, nullptr},
    {"cached_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_cached_attention)), METH_FASTCALL, nullptr},
    {"reorder_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_reorder_blocks)), METH_FASTCALL, nullptr},
    {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_beam_select)), METH_FASTCALL, nullptr},
    {"token_log_probs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_token_log_probs)), METH_FASTCALL, nullptr},
    {"embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_embedding)), METH_FASTCALL, nullptr},
    {"launches", py_launches, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "axonn_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_axonn_host() { return PyModule_Create(&module); }
