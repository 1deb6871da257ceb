// Native half of the pulsar_cuda op surface: output allocation, the current stream and the
// library call of each op, for the Python wrappers in pulsar_cuda/__init__.py, which have
// checked the operands (device, dtype, shape, contiguity) before they come here; the linear ops'
// operands are checked here.
//
// A call through ctypes with its outputs from torch.empty costs 5 us of Python beside the
// 3.4 us of the launch itself (output tensors 2.6, torch.cuda.current_stream 2.0, argument
// conversion 0.5); from here it is 1.5.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/pulsar_hip.h"

namespace {

using at::Tensor;

// Positional arguments of one call.
struct Args {
  PyObject* const* a;
  Py_ssize_t n;
  const Tensor& t(int i) const {
    TORCH_CHECK_TYPE(i < n && THPVariable_Check(a[i]), "argument ", i, " must be a tensor");
    return THPVariable_Unpack(a[i]);
  }
  Tensor opt(int i) const { return a[i] == Py_None ? Tensor() : t(i); }
  int64_t i64(int i) const {
    const long long v = PyLong_AsLongLong(a[i]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  float f32(int i) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
  }
};

struct Unlocked {  // the interpreter lock given up for a scope
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The library call, without the interpreter lock (as through ctypes): a launch can wait for
// room in the queue.
template <typename F, typename... A>
void run(F f, A... args) {
  int rc;
  {
    Unlocked scope;
    rc = f(args...);
  }
  if (rc != PULSAR_OK) {
    const char* m = pulsar_last_error();
    throw std::runtime_error(m && *m ? m : "pulsar_hip error " + std::to_string(rc));
  }
}

int code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? PULSAR_BF16 : PULSAR_F32; }

hipStream_t stream(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A tensor with elements but without memory (a fake one, while a program is traced) is an error
// here: the kernels would read and write address 0. Out of line: a call takes 3 to 8 pointers.
[[gnu::noinline, gnu::cold]] void* no_memory(const Tensor& t) {
  TORCH_CHECK(t.numel() == 0, "the tensor has no memory to read or write");
  return nullptr;
}
void* q(const Tensor& t) {
  void* d = t.data_ptr();
  return d ? d : no_memory(t);
}
const void* p(const Tensor& t) { return t.defined() ? q(t) : nullptr; }
template <typename X>
const X* p(const Tensor& t) { return reinterpret_cast<const X*>(p(t)); }
template <typename X>
X* q(const Tensor& t) { return reinterpret_cast<X*>(q(t)); }

// An output of the layout of argument i. A subclass of torch.Tensor allocates it by its own
// empty_like, so that it is of the subclass's type.
Tensor like(const Args& a, int i) {
  const Tensor& t = a.t(i);
  if (THPVariable_CheckExact(a.a[i])) return at::empty_like(t);
  THPObjectPtr torch(PyImport_ImportModule("torch"));
  if (!torch) throw python_error();
  THPObjectPtr r(PyObject_CallMethod(torch.get(), "empty_like", "O", a.a[i]));
  if (!r) throw python_error();
  TORCH_CHECK_TYPE(THPVariable_Check(r.get()), "empty_like of a tensor subclass gave no tensor");
  return THPVariable_Unpack(r.get());
}
// The gradient of weight argument i. The library zeroes the used entries that it adds to; a
// longer weight's others are zero too.
Tensor like_weight(const Args& a, int i, int64_t used) {
  Tensor dw = like(a, i);
  if (dw.numel() != used) dw.zero_();
  return dw;
}
Tensor make(const Tensor& on, at::IntArrayRef shape, at::ScalarType dt) {
  return at::empty(shape, on.options().dtype(dt).requires_grad(false));
}
Tensor make(const Tensor& on, at::IntArrayRef shape) { return make(on, shape, on.scalar_type()); }

PyObject* out(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(const Tensor& a, const Tensor& b, bool list) {
  THPObjectPtr x(out(a)), y(out(b));
  if (!x || !y) throw python_error();
  PyObject* r = list ? PyList_New(2) : PyTuple_New(2);
  if (!r) throw python_error();
  if (list) {
    PyList_SET_ITEM(r, 0, x.release());
    PyList_SET_ITEM(r, 1, y.release());
  } else {
    PyTuple_SET_ITEM(r, 0, x.release());
    PyTuple_SET_ITEM(r, 1, y.release());
  }
  return r;
}

// (x, weight, eps) -> (y, rsqrt)
PyObject* rmsnorm_forward(const Args& a) {
  const Tensor &x = a.t(0), &w = a.t(1);
  const int64_t dim = x.size(-1), rows = dim ? x.numel() / dim : 0;
  Tensor y = like(a, 0), rs = make(x, {rows}, at::kFloat);
  if (rows)
    run(pulsar_rmsnorm_forward, p(x), p<float>(w), q(y), q<float>(rs), rows, dim, a.f32(2), code(x),
                                 stream(x));
  return pair(y, rs, false);
}

// (x, weight, cos, sin, B, H, T, sB, sH, sT, eps) -> (y, rsqrt)
PyObject* qk_rmsnorm_rope_forward(const Args& a) {
  const Tensor &x = a.t(0), &w = a.t(1), &c = a.t(2), &s = a.t(3);
  Tensor y = make(x, x.sizes()), rs = make(x, {x.numel() / 64}, at::kFloat);
  run(pulsar_qk_rmsnorm_rope_forward, p(x), a.i64(7), a.i64(8), a.i64(9), a.i64(4), a.i64(5),
                                       a.i64(6), 64, p<float>(w), p<float>(c), p<float>(s), q(y),
                                       q<float>(rs), a.f32(10), code(x), stream(x));
  return pair(y, rs, false);
}

// (attn, gate) -> out
PyObject* fused_attn_gate_forward(const Args& a) {
  const Tensor &x = a.t(0), &g = a.t(1);
  const int64_t B = x.size(0), H = x.size(1), T = x.size(2), D = x.size(3);
  Tensor o = make(x, {B, T, H * D});
  run(pulsar_fused_attn_gate_forward, p(x), p<float>(g), q(o), B, H, T, D, code(x), stream(x));
  return out(o);
}

// (x, weight) -> y
PyObject* causal_conv1d_k4_forward(const Args& a) {
  const Tensor &x = a.t(0), &w = a.t(1);
  Tensor y = like(a, 0);
  run(pulsar_causal_conv1d_k4_forward, p(x), p<float>(w), q(y), x.size(0), x.size(1), x.size(2),
                                        code(x), stream(x));
  return out(y);
}

// (gu, d_ff) -> out
PyObject* fused_swiglu_forward(const Args& a) {
  const Tensor& gu = a.t(0);
  TORCH_CHECK(gu.dim() > 0, "gu must have at least one dimension");
  const int64_t d = a.i64(1), rows = d ? gu.numel() / (2 * d) : 0;
  std::vector<int64_t> shape = gu.sizes().vec();
  shape.back() = d;
  Tensor o = make(gu, shape);
  if (rows) run(pulsar_fused_swiglu_forward, p(gu), q(o), rows, d, code(gu), stream(gu));
  return out(o);
}

// (logits, bias, top_k, z_loss_weight) -> (idx, weights, z_loss, probs_mean)
PyObject* moe_router_topk_forward(const Args& a) {
  const Tensor &l = a.t(0), &b = a.t(1);
  const int64_t N = l.size(0), E = l.size(1), K = a.i64(2);
  Tensor idx = make(l, {N, K}, at::kLong), w = make(l, {N, K}, at::kBFloat16);
  Tensor z = make(l, {}, at::kFloat), pm = make(l, {E}, at::kFloat);
  // per-workgroup partial statistics (merged in a fixed order inside the library)
  Tensor ws = make(l, {std::max<int64_t>(1, pulsar_moe_router_workspace_bytes(N, E) / 4)}, at::kFloat);
  run(pulsar_moe_router_topk_forward_ws, p(l), code(l), p<float>(b), q<int64_t>(idx),
                                          q<uint16_t>(w), q<float>(z), q<float>(pm), N, E, K,
                                          a.f32(3), q<float>(ws), stream(l));
  THPObjectPtr r(PyTuple_New(4));
  if (!r) throw python_error();
  const Tensor* o[4] = {&idx, &w, &z, &pm};
  for (int i = 0; i < 4; ++i) {
    PyObject* t = out(*o[i]);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(r.get(), i, t);
  }
  return r.release();
}

// (x, topk_idx, slots, E, C, counts) -> expert_inputs
PyObject* moe_dispatch_forward(const Args& a) {
  const Tensor &x = a.t(0), &ti = a.t(1), &ts = a.t(2);
  const int64_t E = a.i64(3), C = a.i64(4);
  const Tensor n = a.opt(5);
  Tensor o = make(x, {E, C, x.size(1)});
  run(pulsar_moe_dispatch_forward, p(x), p<int64_t>(ti), p<int32_t>(ts), p<int64_t>(n), q(o),
                                    x.size(0), x.size(1), ti.size(1), E, C, code(x), stream(x));
  return out(o);
}

// (expert_outputs, topk_idx, weights, slots, shared) -> out
PyObject* moe_combine_forward(const Args& a) {
  const Tensor &eo = a.t(0), &ti = a.t(1), &w = a.t(2), &ts = a.t(3);
  const Tensor sh = a.opt(4);
  const int64_t N = ti.size(0), D = eo.size(2);
  Tensor o = make(eo, {N, D});
  if (N)
    run(pulsar_moe_combine_forward, p(eo), p<int64_t>(ti), p<uint16_t>(w), p<int32_t>(ts), p(sh),
                                     q(o), N, D, ti.size(1), eo.size(0), eo.size(1), code(eo),
                                     stream(eo));
  return out(o);
}

// (flat_e, order, E, C) -> (slots, counts)
PyObject* moe_slots_from_order(const Args& a) {
  const Tensor &f = a.t(0), &o = a.t(1);
  const int64_t M = f.numel(), E = a.i64(2);
  Tensor s = make(f, {M}, at::kInt), n = make(f, {E}, at::kLong);
  run(pulsar_moe_slots_from_order, p<int64_t>(f), p<int64_t>(o), q<int32_t>(s), q<int64_t>(n), M, E,
                                    a.i64(3), stream(f));
  return pair(s, n, false);
}

// (dy, x, weight, rsqrt, dw's layout) -> [dx, dw]
PyObject* rmsnorm_backward(const Args& a) {
  const Tensor &dy = a.t(0), &x = a.t(1), &w = a.t(2), &rs = a.t(3);
  const int64_t dim = x.size(-1);
  Tensor dx = like(a, 1), dw = like_weight(a, 4, dim);
  run(pulsar_rmsnorm_backward, p(dy), p(x), p<float>(w), p<float>(rs), q(dx), q<float>(dw),
                                x.numel() / dim, dim, code(x), stream(x));
  return pair(dx, dw, true);
}

// (dy, x, weight, rsqrt, cos, sin, dx, B, H, T, sB, sH, sT, dB, dH, dT) -> [dx, dw]
PyObject* qk_rmsnorm_rope_backward(const Args& a) {
  const Tensor &dy = a.t(0), &x = a.t(1), &w = a.t(2), &rs = a.t(3), &c = a.t(4), &s = a.t(5);
  const Tensor& dx = a.t(6);
  Tensor dw = like_weight(a, 2, 64 * a.i64(8));
  run(pulsar_qk_rmsnorm_rope_backward, p(dy), p(x), a.i64(10), a.i64(11), a.i64(12), q(dx),
                                        a.i64(13), a.i64(14), a.i64(15), a.i64(7), a.i64(8), a.i64(9),
                                        64, p<float>(w), p<float>(rs), p<float>(c), p<float>(s),
                                        q<float>(dw), code(x), stream(x));
  return pair(dx, dw, true);
}

// (grad_out, attn, gate) -> [d_attn, d_gate]
PyObject* fused_attn_gate_backward(const Args& a) {
  const Tensor &go = a.t(0), &x = a.t(1), &g = a.t(2);
  const int64_t B = x.size(0), H = x.size(1), T = x.size(2);
  Tensor da = like(a, 1), dg = make(x, {B, T, H}, at::kFloat);
  if (da.numel())
    run(pulsar_fused_attn_gate_backward, p(go), p(x), p<float>(g), q(da), q<float>(dg), B, H, T, 64,
                                          code(x), stream(x));
  return pair(da, dg, true);
}

// (dout, gu, d_ff) -> dgu
PyObject* fused_swiglu_backward(const Args& a) {
  const Tensor &d = a.t(0), &gu = a.t(1);
  const int64_t f = a.i64(2), rows = f ? gu.numel() / (2 * f) : 0;
  Tensor o = like(a, 1);
  if (rows) run(pulsar_fused_swiglu_backward, p(d), p(gu), q(o), rows, f, code(gu), stream(gu));
  return out(o);
}

// (dout, x, weight) -> [dx, dw]
PyObject* causal_conv1d_k4_backward(const Args& a) {
  const Tensor &d = a.t(0), &x = a.t(1), &w = a.t(2);
  Tensor dx = like(a, 1), dw = like_weight(a, 2, 4 * x.size(2));
  run(pulsar_causal_conv1d_k4_backward, p(d), p(x), p<float>(w), q(dx), q<float>(dw), x.size(0),
                                         x.size(1), x.size(2), code(x), stream(x));
  return pair(dx, dw, true);
}

// (d_weights, logits, topk_idx, z_loss_weight, d_z_loss, d_probs_mean) -> d_logits
PyObject* moe_router_topk_backward(const Args& a) {
  const Tensor &dw = a.t(0), &l = a.t(1), &ti = a.t(2);
  const Tensor dz = a.opt(4), dp = a.opt(5);
  Tensor o = like(a, 1);
  if (l.size(0))
    run(pulsar_moe_router_topk_backward, p<uint16_t>(dw), p(l), code(l), p<int64_t>(ti), a.f32(3),
                                          p<float>(dz), p<float>(dp), q(o), l.size(0), l.size(1),
                                          ti.size(1), stream(l));
  return out(o);
}

// (d_expert_inputs, topk_idx, slots, N, D) -> dx
PyObject* moe_dispatch_backward(const Args& a) {
  const Tensor &d = a.t(0), &ti = a.t(1), &ts = a.t(2);
  const int64_t N = a.i64(3), D = a.i64(4);
  Tensor o = make(d, {N, D});
  if (N)
    run(pulsar_moe_dispatch_backward, p(d), p<int64_t>(ti), p<int32_t>(ts), q(o), N, D, ti.size(1),
                                       d.size(0), d.size(1), code(d), stream(d));
  return out(o);
}

// (d_out, expert_outputs, topk_idx, weights, slots) -> [d_expert_outputs, d_weights]
PyObject* moe_combine_backward(const Args& a) {
  const Tensor &d = a.t(0), &eo = a.t(1), &ti = a.t(2), &w = a.t(3), &ts = a.t(4);
  const int64_t N = ti.size(0), K = ti.size(1);
  Tensor de = like(a, 1), dw = make(eo, {N, K}, at::kBFloat16);
  run(pulsar_moe_combine_backward, p(d), p(eo), p<int64_t>(ti), p<uint16_t>(w), p<int32_t>(ts),
                                    q(de), q<uint16_t>(dw), N, eo.size(2), K, eo.size(0), eo.size(1),
                                    code(eo), stream(eo));
  return pair(de, dw, true);
}

// Row stride of a tensor read as [rows, last dimension]: 2-dimensional with any row stride, or
// contiguous.
int64_t row_stride(const Tensor& t, const char* name) {
  const int64_t n = t.size(-1), rows = n ? t.numel() / n : 0;
  if (rows <= 1) {
    TORCH_CHECK(n <= 1 || t.stride(-1) == 1, name, " must have stride(-1) == 1");
    return n;
  }
  if (t.is_contiguous()) return n;
  TORCH_CHECK(t.dim() == 2 && (n == 1 || t.stride(1) == 1), name,
              " must be contiguous, or 2-dimensional with stride(-1) == 1");
  return t.stride(0);
}
// Strides of a weight's last two dimensions, one of them 1 (a dimension of size 1 has no stride
// of its own).
void weight_strides(const Tensor& w, int64_t& s0, int64_t& s1) {
  const int64_t n0 = w.size(-2), n1 = w.size(-1);
  s0 = w.stride(-2);
  s1 = w.stride(-1);
  if (n1 == 1) s1 = 1;
  if (n0 == 1) s0 = s1 == 1 ? n1 : 1;
  TORCH_CHECK(s0 == 1 || s1 == 1, "weight must have a unit stride in one of its last two dimensions");
}
// A gradient of weight w, dense in w's own order of the last two dimensions.
Tensor weight_grad(const Tensor& w, bool last_contiguous) {
  std::vector<int64_t> shape = w.sizes().vec();
  if (last_contiguous) return make(w, shape);
  std::swap(shape[shape.size() - 1], shape[shape.size() - 2]);
  return make(w, shape).transpose(-2, -1);
}
PyObject* triple(const Tensor& a, const Tensor& b, const Tensor& c, bool list) {
  PyObject* o[3] = {out(a), out(b), c.defined() ? out(c) : Py_NewRef(Py_None)};
  PyObject* r = o[0] && o[1] && o[2] ? (list ? PyList_New(3) : PyTuple_New(3)) : nullptr;
  if (!r) {
    for (PyObject* x : o) Py_XDECREF(x);
    throw python_error();
  }
  for (int i = 0; i < 3; ++i) {
    if (list)
      PyList_SET_ITEM(r, i, o[i]);
    else
      PyTuple_SET_ITEM(r, i, o[i]);
  }
  return r;
}

// Workspace of the given size (an error for -1: what the library refuses), undefined when none.
Tensor workspace(const Tensor& on, int64_t bytes) {
  if (bytes < 0) throw std::runtime_error(pulsar_last_error());
  return bytes ? make(on, {bytes}, at::kByte) : Tensor();
}
void* wp(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The checks of the linear ops are here, not in Python, where they took 3 us of an 8 us call. Types
// and shapes first, the device last, before anything is allocated or launched.
void on_device(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK(t.device() == x.device(), name, " must be on the device of x");
}
void float_type(const Tensor& x) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat,
              "x must be bfloat16 or float32, got ", x.scalar_type());
}
void same_type(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the dtype of x");
}
void on_gpu(const Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
}
void shaped(const Tensor& t, const char* name, at::IntArrayRef shape) {
  TORCH_CHECK(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
}
int64_t out_cols(int64_t act, int64_t d_out) {
  if (act != PULSAR_ACT_SWIGLU) return d_out;
  TORCH_CHECK(d_out % 2 == 0, "swiglu needs an even number of output columns, got ", d_out);
  return d_out / 2;
}
// An optional bias, of x's type or fp32.
Tensor checked_bias(const Tensor& b, const Tensor& x, at::IntArrayRef shape) {
  if (!b.defined()) return b;
  TORCH_CHECK(b.scalar_type() == x.scalar_type() || b.scalar_type() == at::kFloat,
              "bias must have the dtype of x or be float32");
  shaped(b, "bias", shape);
  on_device(b, "bias", x);
  return b.contiguous();
}
Tensor checked_index(const Tensor& t, const char* name, const Tensor& x) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1, name, " must be 1-dimensional int32");
  on_device(t, name, x);
  return t.contiguous();
}
// The pre-activation values of a backward call that needs them.
Tensor checked_pre(const Tensor& pre, int64_t act, const Tensor& x, at::IntArrayRef shape) {
  if (act == PULSAR_ACT_NONE) return Tensor();
  TORCH_CHECK(pre.defined(), "pre is needed for every activation but none");
  same_type(pre, "pre", x);
  shaped(pre, "pre", shape);
  on_device(pre, "pre", x);
  return pre.contiguous();
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  return shape;
}

// (topk_idx, E) -> (offsets, rows, slots)
PyObject* moe_group_rows(const Args& a) {
  const Tensor& t = a.t(0);
  const int64_t E = a.i64(1);
  TORCH_CHECK(t.scalar_type() == at::kLong, "topk_idx must be int64");
  TORCH_CHECK(t.dim() == 2 && t.size(1) > 0, "topk_idx must be [N, K]");
  TORCH_CHECK(E > 0 && E <= 1024, "moe_group_rows supports 1 <= E <= 1024, got ", E);
  on_gpu(t, "topk_idx");
  const Tensor idx = t.contiguous();
  const int64_t N = idx.size(0), K = idx.size(1);
  const c10::DeviceGuard guard(idx.device());
  const Tensor ws = workspace(idx, pulsar_moe_group_rows_workspace_bytes(N, K, E));
  Tensor o = make(idx, {E + 1}, at::kInt), r = make(idx, {N * K}, at::kInt);
  Tensor s = make(idx, {N, K}, at::kInt);
  run(pulsar_moe_group_rows, p<int64_t>(idx), q<int32_t>(o), q<int32_t>(r), q<int32_t>(s), N, K, E,
      wp(ws), stream(idx));
  return triple(o, r, s, false);
}

struct Linear {  // operands of the dense ops
  const Tensor &x, &w;
  int64_t act, I, O, cols, rows, so, si, xs;
  Linear(const Tensor& x_, const Tensor& w_, int64_t act_) : x(x_), w(w_), act(act_) {
    float_type(x);
    same_type(w, "weight", x);
    TORCH_CHECK(w.dim() == 2, "weight must be [d_out, d_in]");
    O = w.size(0);
    I = w.size(1);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == I, "x must be [..., d_in]");
    TORCH_CHECK(O > 0 && I > 0, "weight must not be empty");
    cols = out_cols(act, O);
    rows = x.numel() / I;
    weight_strides(w, so, si);
    xs = row_stride(x, "x");
  }
  void device() const {
    on_gpu(x, "x");
    on_device(w, "weight", x);
  }
};

// (x, weight [O, I], bias, residual, activation, save_pre) -> y or (y, pre)
PyObject* fused_linear_forward(const Args& a) {
  const Linear l(a.t(0), a.t(1), a.i64(4));
  const Tensor b = checked_bias(a.opt(2), l.x, {l.O}), res = a.opt(3);
  int64_t rs = 0;
  if (res.defined()) {
    same_type(res, "residual", l.x);
    shaped(res, "residual", with_last(l.x, l.cols));
    on_device(res, "residual", l.x);
    rs = row_stride(res, "residual");
  }
  l.device();
  const c10::DeviceGuard guard(l.x.device());
  Tensor pre;
  if (a.i64(5)) pre = make(l.x, with_last(l.x, l.O));
  Tensor y = make(l.x, with_last(l.x, l.cols));
  const Tensor ws = workspace(l.x, pulsar_fused_linear_forward_workspace_bytes(
      l.x.data_ptr(), l.xs, l.w.data_ptr(), l.so, l.si, l.rows, l.I, l.O, (int)l.act, code(l.x)));
  run(pulsar_fused_linear_forward, p(l.x), l.xs, p(l.w), l.so, l.si, p(b), b.defined() ? code(b) : 0,
      p(res), rs, q(y), pre.defined() ? q(pre) : nullptr, l.rows, l.I, l.O, (int)l.act, code(l.x),
      wp(ws), stream(l.x));
  return pre.defined() ? pair(y, pre, false) : out(y);
}

// (dy, x, weight [O, I], pre, activation, bias) -> [dx, dw, db]
PyObject* fused_linear_backward(const Args& a) {
  const Linear l(a.t(1), a.t(2), a.i64(4));
  const Tensor& d = a.t(0);
  same_type(d, "dy", l.x);
  shaped(d, "dy", with_last(l.x, l.cols));
  on_device(d, "dy", l.x);
  const Tensor pre = checked_pre(a.opt(3), l.act, l.x, with_last(l.x, l.O));
  l.device();
  const c10::DeviceGuard guard(l.x.device());
  const Tensor dy = d.contiguous();
  Tensor dx = make(l.x, l.x.sizes()), dw = weight_grad(l.w, l.si == 1), db;
  if (a.i64(5)) db = make(l.x, {l.O});
  const Tensor ws = workspace(l.x, pulsar_fused_linear_backward_workspace_bytes(
      dy.data_ptr(), l.x.data_ptr(), l.xs, l.w.data_ptr(), l.so, l.si, l.rows, l.I, l.O, (int)l.act,
      code(l.x)));
  run(pulsar_fused_linear_backward, p(dy), p(l.x), l.xs, p(l.w), l.so, l.si, p(pre), q(dx), q(dw),
      db.defined() ? q(db) : nullptr, l.rows, l.I, l.O, (int)l.act, code(l.x), wp(ws), stream(l.x));
  return triple(dx, dw, db, true);
}

struct Grouped {  // operands of the ragged ops
  const Tensor &x, &w;
  Tensor off, idx;
  int64_t act, E, I, O, cols, M, si, so, xs;
  Grouped(const Tensor& x_, const Tensor& w_, const Tensor& off_, const Tensor& idx_, int64_t act_)
      : x(x_), w(w_), act(act_) {
    float_type(x);
    same_type(w, "weight", x);
    TORCH_CHECK(w.dim() == 3, "weight must be [E, d_in, d_out]");
    E = w.size(0);
    I = w.size(1);
    O = w.size(2);
    TORCH_CHECK(x.dim() == 2 && x.size(1) == I, "x must be [R, d_in]");
    TORCH_CHECK(E > 0 && I > 0 && O > 0, "weight must not be empty");
    cols = out_cols(act, O);
    off = checked_index(off_, "offsets", x);
    TORCH_CHECK(off.numel() == E + 1, "offsets must have E + 1 elements");
    idx = checked_index(idx_, "rows", x);
    M = idx.defined() ? idx.numel() : x.size(0);
    weight_strides(w, si, so);
    xs = row_stride(x, "x");
  }
  void device() const {
    on_gpu(x, "x");
    on_device(w, "weight", x);
  }
};

// (x, weight [E, I, O], offsets, rows, bias, activation, save_pre) -> y or (y, pre)
PyObject* grouped_linear_forward(const Args& a) {
  const Grouped l(a.t(0), a.t(1), a.t(2), a.opt(3), a.i64(5));
  const Tensor b = checked_bias(a.opt(4), l.x, {l.E, l.O});
  l.device();
  const c10::DeviceGuard guard(l.x.device());
  Tensor pre;
  if (a.i64(6)) pre = make(l.x, {l.M, l.O});
  Tensor y = make(l.x, {l.M, l.cols});
  const Tensor ws = workspace(l.x, pulsar_grouped_linear_forward_workspace_bytes(
      l.x.data_ptr(), l.xs, l.x.size(0), l.w.data_ptr(), l.w.stride(0), l.si, l.so, l.M, l.E, l.I,
      l.O, (int)l.act, code(l.x)));
  run(pulsar_grouped_linear_forward, p(l.x), l.xs, l.x.size(0), p<int32_t>(l.idx),
      p<int32_t>(l.off), p(l.w), l.w.stride(0), l.si, l.so, p(b), b.defined() ? code(b) : 0, q(y),
      pre.defined() ? q(pre) : nullptr, l.M, l.E, l.I, l.O, (int)l.act, code(l.x), wp(ws),
      stream(l.x));
  return pre.defined() ? pair(y, pre, false) : out(y);
}

// (dy, x, weight [E, I, O], offsets, rows, pre, activation, bias) -> [dx, dw, db]
PyObject* grouped_linear_backward(const Args& a) {
  const Grouped l(a.t(1), a.t(2), a.t(3), a.opt(4), a.i64(6));
  const Tensor& d = a.t(0);
  same_type(d, "dy", l.x);
  shaped(d, "dy", {l.M, l.cols});
  on_device(d, "dy", l.x);
  const Tensor pre = checked_pre(a.opt(5), l.act, l.x, {l.M, l.O});
  l.device();
  const c10::DeviceGuard guard(l.x.device());
  const Tensor dy = d.contiguous();
  // the library writes dw with the input dimension contiguous where the weight's is
  Tensor dx = make(l.x, {l.M, l.I}), dw = weight_grad(l.w, l.si != 1), db;
  if (a.i64(7)) db = make(l.x, {l.E, l.O});
  const Tensor ws = workspace(l.x, pulsar_grouped_linear_backward_workspace_bytes(
      dy.data_ptr(), l.x.data_ptr(), l.xs, l.x.size(0), l.w.data_ptr(), l.w.stride(0), l.si, l.so,
      l.M, l.E, l.I, l.O, (int)l.act, code(l.x)));
  run(pulsar_grouped_linear_backward, p(dy), p(l.x), l.xs, l.x.size(0), p<int32_t>(l.idx),
      p<int32_t>(l.off), p(l.w), l.w.stride(0), l.si, l.so, p(pre), q(dx), q(dw),
      db.defined() ? q(db) : nullptr, l.M, l.E, l.I, l.O, (int)l.act, code(l.x), wp(ws),
      stream(l.x));
  return triple(dx, dw, db, true);
}

template <PyObject* (*F)(const Args&), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == N, "expected ", N, " arguments, got ", n);
  return F(Args{args, n});
  END_HANDLE_TH_ERRORS
}

#define OP(name, n) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&call<name, n>)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {
    OP(rmsnorm_forward, 3),          OP(qk_rmsnorm_rope_forward, 11),
    OP(fused_attn_gate_forward, 2),  OP(causal_conv1d_k4_forward, 2),
    OP(fused_swiglu_forward, 2),     OP(moe_router_topk_forward, 4),
    OP(moe_dispatch_forward, 6),     OP(moe_combine_forward, 5),
    OP(moe_slots_from_order, 4),     OP(rmsnorm_backward, 5),
    OP(qk_rmsnorm_rope_backward, 16), OP(fused_attn_gate_backward, 3),
    OP(fused_swiglu_backward, 3),    OP(causal_conv1d_k4_backward, 3),
    OP(moe_router_topk_backward, 6), OP(moe_dispatch_backward, 5),
    OP(moe_combine_backward, 5),     OP(moe_group_rows, 2),
    OP(fused_linear_forward, 6),     OP(fused_linear_backward, 6),
    OP(grouped_linear_forward, 7),   OP(grouped_linear_backward, 8),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
