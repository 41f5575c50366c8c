// rustorch_b200._ops: the Python calls of the training, 8-bit and 4-bit operators.
//
// These operators' smallest calls take less time on the GPU than an interpreted
// wrapper takes to check their arguments, allocate their outputs and convert a
// dozen values for a foreign call (15 us of host time for layer_norm_fwd of 16
// x 1024 against 3 us of kernel).  This module does that part in C++ over the
// same C ABI (include/rustorch_b200.h): ValueError for what the library's
// Python layer refuses, RtbError (raised by rustorch_b200._lib.check) for a
// non-zero status.  Tensors give memory and streams only.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../../include/rustorch_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

struct PyFailure {};  // a Python exception is set

[[noreturn]] void refuse(const std::string& what) { throw std::invalid_argument(what); }

// The context of a device: rustorch_b200.get_context(dev).handle, asked for
// every time (a closed or replaced context is seen at once).
PyObject* g_get_context = nullptr;
PyObject* g_check = nullptr;
PyObject* g_handle_name = nullptr;
PyObject* g_value_name = nullptr;

rtb_ctx* context(int dev) {
  PyObject* arg = PyLong_FromLong(dev);
  PyObject* c = arg ? PyObject_CallOneArg(g_get_context, arg) : nullptr;
  Py_XDECREF(arg);
  PyObject* h = c ? PyObject_GetAttr(c, g_handle_name) : nullptr;
  Py_XDECREF(c);
  if (!h) throw PyFailure();
  if (h == Py_None) {
    Py_DECREF(h);
    return nullptr;
  }
  PyObject* v = PyObject_GetAttr(h, g_value_name);
  Py_DECREF(h);
  if (!v) throw PyFailure();
  rtb_ctx* ctx = v == Py_None ? nullptr : static_cast<rtb_ctx*>(PyLong_AsVoidPtr(v));
  Py_DECREF(v);
  if (PyErr_Occurred()) throw PyFailure();
  return ctx;
}

void check(int status, const char* where) {
  if (status == RTB_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", status, where);  // raises RtbError
  Py_XDECREF(r);
  throw PyFailure();
}

// ------------------------------------------------------------------ arguments
const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", what);
    throw PyFailure();
  }
  return THPVariable_Unpack(o);
}
const Tensor* optional(PyObject* o, const char* what) {
  return o == Py_None ? nullptr : &tensor(o, what);
}
bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailure();
  return v != 0;
}
int integer(PyObject* o) {
  int over = 0;
  const long v = PyLong_AsLongAndOverflow(o, &over);
  if (v == -1 && PyErr_Occurred()) throw PyFailure();
  if (over || v < INT_MIN || v > INT_MAX) refuse("rustorch_b200: whole number out of range");
  return (int)v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailure();
  return v;
}

void need_f32(const Tensor* t) {
  if (t && !(t->is_cuda() && t->scalar_type() == ScalarType::Float))
    refuse("rustorch_b200 expects float32 CUDA tensors");
}
void need_fp8(const Tensor& t, const char* who) {
  if (!(t.is_cuda() && t.scalar_type() == ScalarType::Float8_e4m3fn))
    refuse(std::string(who) + " expects float8_e4m3fn CUDA tensors");
}
void same_device(const Tensor& first, std::initializer_list<const Tensor*> rest) {
  for (const Tensor* t : rest)
    if (t && t->device() != first.device()) refuse("rustorch_b200: tensors on different devices");
}

// A tensor as rows of d contiguous elements that do not overlap; a copy only
// where it has no such view (transposed, expanded).
struct Rows {
  Tensor hold;
  int64_t rows = 0, ld = 0;
  void* p() const { return hold.data_ptr(); }
};
Rows rows_of(const Tensor& t, int64_t d) {
  Rows r;
  if (t.is_contiguous()) {
    r.hold = t;
    r.ld = d;
  } else {
    r.hold = t.dim() == 2 ? t : t.reshape({-1, d});
    if ((d > 1 && r.hold.stride(1) != 1) || (r.hold.size(0) > 1 && r.hold.stride(0) < d))
      r.hold = r.hold.contiguous();
    r.ld = r.hold.stride(0) > d ? r.hold.stride(0) : d;
  }
  r.rows = d ? r.hold.numel() / d : 0;
  return r;
}

// A vector of n elements, contiguous; none stays none.
struct Vec {
  Tensor hold;
  float* p = nullptr;
};
Vec vec(const Tensor* t, int64_t n, const char* message) {
  Vec v;
  if (!t) return v;
  if (t->numel() != n) refuse(message);
  v.hold = t->is_contiguous() ? *t : t->contiguous();
  v.p = v.hold.data_ptr<float>();
  return v;
}

struct Scales {
  Tensor hold;
  int64_t ld = 0;
  int block_rows = 1, type = RTB_SCALE_E8M0;
};
Scales scales(const Tensor& s, int64_t rows, int64_t cols, const char* who) {
  Scales r;
  const bool e8m0 = s.scalar_type() == ScalarType::Float8_e8m0fnu;
  if (!s.is_cuda() || !(e8m0 || s.scalar_type() == ScalarType::Float))
    refuse(std::string(who) + ": scales are float8_e8m0fnu or float32 CUDA tensors");
  const int64_t cb = (cols + 127) / 128, nb = (rows + 127) / 128;
  if (s.dim() < 1 || s.size(-1) != cb ||
      (cb > 0 && s.numel() != rows * cb && s.numel() != nb * cb) ||
      (cb == 0 && s.dim() == 2 && s.size(0) != rows && s.size(0) != nb))
    refuse(std::string(who) + ": scales must be [rows or ceil(rows / 128), ceil(cols / 128)]");
  Rows v = rows_of(s, cb);
  r.hold = v.hold;
  r.ld = v.ld;
  r.block_rows = s.numel() == rows * cb ? 1 : 128;
  r.type = e8m0 ? RTB_SCALE_E8M0 : RTB_SCALE_F32;
  return r;
}

Tensor empty_f32(const Tensor& like, at::IntArrayRef shape) {
  return at::empty(shape, like.options().dtype(at::kFloat));
}

// The tensor that a gradient is written or added to.
std::optional<Tensor> result(const Tensor* out, bool need, bool accumulate, at::IntArrayRef shape,
                             const Tensor& like, const char* who) {
  if (!need) return std::nullopt;
  if (!out) {
    if (accumulate) refuse(std::string(who) + ": accumulate adds to given outputs");
    return empty_f32(like, shape);
  }
  if (!out->is_contiguous() || out->sizes() != shape)
    refuse(std::string(who) + ": outputs must be contiguous and of the gradient's shape");
  return *out;
}
float* ptr(std::optional<Tensor>& t) { return t ? t->data_ptr<float>() : nullptr; }
PyObject* wrap(std::optional<Tensor>& t) {
  if (!t) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}
PyObject* pack(std::initializer_list<PyObject*> items) {
  PyObject* r = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    if (!o || !r) {
      Py_XDECREF(r);
      throw PyFailure();
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// The C call without the interpreter lock, which is held again where the call
// throws (a tensor's data pointer does where the tensor has none).
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
void call(const char* where, const F& f) {
  int st;
  {
    Unlocked u;
    st = f();
  }
  check(st, where);
}

const char* const kShape = "LayerNorm: Input shape does not match normalized shape";

// ------------------------------------------------------------------ operators
PyObject* layer_norm_fwd(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x");
  const Tensor *w = optional(a[1], "norm_weight"), *b = optional(a[2], "norm_bias");
  const float eps = (float)real(a[3]);
  const int act = integer(a[4]);
  const Tensor* out = optional(a[5], "out");
  for (const Tensor* t : {&x, w, b, out}) need_f32(t);
  same_device(x, {w, b, out});
  const int64_t d = x.dim() ? x.size(-1) : 0;
  if (d == 0) refuse("LayerNorm: Input shape smaller than normalized shape");
  const Vec wv = vec(w, d, kShape), bv = vec(b, d, kShape);
  const Rows xr = rows_of(x, d);
  Tensor y;
  int64_t ldy = d;
  if (!out) {
    y = empty_f32(x, x.sizes());
  } else {
    if (out->sizes() != x.sizes() || (d > 1 && out->stride(-1) != 1))
      refuse("layer_norm_fwd: out must have x's shape and contiguous rows");
    y = *out;
    if (!out->is_contiguous()) {
      const Tensor y2 = out->dim() == 2 ? *out : out->view({-1, d});
      if (y2.size(0) > 1 && y2.stride(0) < d) refuse("layer_norm_fwd: out's rows overlap");
      ldy = y2.stride(0) > d ? y2.stride(0) : d;
    }
  }
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  Tensor mean = empty_f32(x, lead), rstd = empty_f32(x, lead);
  rtb_ctx* ctx = context(x.device().index());
  void* s = stream_of(x);
  call("rtb_layer_norm_fwd", [&] {
    return rtb_layer_norm_fwd(ctx, xr.rows, d, (const float*)xr.p(), xr.ld, wv.p, bv.p, eps, act,
                              y.data_ptr<float>(), ldy, mean.data_ptr<float>(),
                              rstd.data_ptr<float>(), s);
  });
  return pack({THPVariable_Wrap(y), THPVariable_Wrap(mean), THPVariable_Wrap(rstd)});
}

PyObject* layer_norm_backward(PyObject* const* a) {
  const char* who = "layer_norm_backward";
  const Tensor& x = tensor(a[0], "x");
  const Tensor &mean = tensor(a[1], "mean"), &rstd = tensor(a[2], "rstd"), &grad = tensor(a[3], "grad");
  const Tensor *w = optional(a[4], "norm_weight"), *b = optional(a[5], "norm_bias");
  const int act = integer(a[6]);
  const Tensor* xs = optional(a[7], "x_scale");
  const bool need_x = flag(a[8]), need_w = flag(a[9]), need_b = flag(a[10]);
  const Tensor *ox = optional(a[11], "out_x"), *ow = optional(a[12], "out_weight"),
               *ob = optional(a[13], "out_bias");
  const bool accumulate = flag(a[14]);
  const bool saved = x.scalar_type() == ScalarType::Float8_e4m3fn;
  for (const Tensor* t : {&mean, &rstd, &grad, w, b, ox, ow, ob}) need_f32(t);
  if (saved) need_fp8(x, who);
  else need_f32(&x);
  same_device(x, {&mean, &rstd, &grad, w, b, xs, ox, ow, ob});
  const int64_t d = x.dim() ? x.size(-1) : 0;
  if (d == 0 || grad.sizes() != x.sizes())
    refuse("layer_norm_backward: grad must have x's shape, with a last dimension");
  const Rows xr = rows_of(x, d), gr = rows_of(grad, d);
  const char* per_row = "layer_norm_backward: one mean and rstd for each row";
  const Vec mv = vec(&mean, xr.rows, per_row), rv = vec(&rstd, xr.rows, per_row);
  const Vec wv = vec(w, d, kShape), bv = vec(b, d, kShape);
  if (saved != (xs != nullptr))
    refuse("layer_norm_backward: x_scale goes with an 8-bit x, and only with one");
  auto dx = result(ox, need_x, accumulate, x.sizes(), grad, who);
  auto dw = result(ow, need_w, accumulate, {d}, grad, who);
  auto db = result(ob, need_b, accumulate, {d}, grad, who);
  Scales sc;
  if (saved) {
    sc = scales(*xs, xr.rows, d, who);
    if (sc.type != RTB_SCALE_E8M0 || sc.block_rows != 1)
      refuse("layer_norm_backward: a checkpoint has a power-of-two scale for each 128 columns of a row");
  }
  rtb_ctx* ctx = context(x.device().index());
  void* s = stream_of(x);
  float *px = ptr(dx), *pw = ptr(dw), *pb = ptr(db);
  if (saved) {
    call("rtb_layer_norm_backward_fp8", [&] {
      return rtb_layer_norm_backward_fp8(ctx, xr.rows, d, (const uint8_t*)xr.p(), xr.ld,
                                         (const uint8_t*)sc.hold.data_ptr(), sc.ld, mv.p, rv.p,
                                         wv.p, bv.p, act, (const float*)gr.p(), gr.ld, px, d, pw,
                                         pb, accumulate, s);
    });
  } else {
    call("rtb_layer_norm_backward", [&] {
      return rtb_layer_norm_backward(ctx, xr.rows, d, (const float*)xr.p(), xr.ld, mv.p, rv.p, wv.p,
                                     bv.p, act, (const float*)gr.p(), gr.ld, px, d, pw, pb,
                                     accumulate, s);
    });
  }
  return pack({wrap(dx), wrap(dw), wrap(db)});
}

PyObject* fp8_quantize(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x");
  const int block_rows = integer(a[1]);
  need_f32(&x);
  if (block_rows != 1 && block_rows != 128) refuse("fp8_quantize: block_rows must be 1 or 128");
  if (x.dim() == 0 || (block_rows != 1 && x.dim() != 2))
    refuse("fp8_quantize: x needs a last dimension, and two for 128-row blocks");
  const int64_t cols = x.size(-1), cb = (cols + 127) / 128;
  Tensor q = at::empty(x.sizes(), x.options().dtype(ScalarType::Float8_e4m3fn));
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = cb;
  if (block_rows != 1) shape[0] = (x.size(0) + 127) / 128;
  Tensor scale = at::empty(shape, x.options().dtype(ScalarType::Float8_e8m0fnu));
  if (x.numel()) {
    const Rows xr = rows_of(x, cols);
    rtb_ctx* ctx = context(x.device().index());
    void* s = stream_of(x);
    call("rtb_fp8_quantize", [&] {
      return rtb_fp8_quantize(ctx, xr.rows, cols, (const float*)xr.p(), xr.ld, block_rows,
                              (uint8_t*)q.data_ptr(), cols, (uint8_t*)scale.data_ptr(), cb, s);
    });
  }
  return pack({THPVariable_Wrap(q), THPVariable_Wrap(scale)});
}

PyObject* fp8_dequantize(PyObject* const* a) {
  const char* who = "fp8_dequantize";
  const Tensor &q = tensor(a[0], "q"), &scale = tensor(a[1], "scale");
  const Tensor* out = optional(a[2], "out");
  need_fp8(q, who);
  need_f32(out);
  same_device(q, {&scale, out});
  if (q.dim() == 0) refuse("fp8_dequantize: q needs a last dimension");
  const int64_t cols = q.size(-1);
  if (out && (out->sizes() != q.sizes() || !out->is_contiguous()))
    refuse("fp8_dequantize: out must be contiguous and have q's shape");
  Tensor y = out ? *out : empty_f32(q, q.sizes());
  if (q.numel()) {
    const Rows qr = rows_of(q, cols);
    const Scales sc = scales(scale, qr.rows, cols, who);
    if (sc.type != RTB_SCALE_E8M0) refuse("fp8_dequantize: scales are float8_e8m0fnu");
    rtb_ctx* ctx = context(q.device().index());
    void* s = stream_of(q);
    call("rtb_fp8_dequantize", [&] {
      return rtb_fp8_dequantize(ctx, qr.rows, cols, (const uint8_t*)qr.p(), qr.ld,
                                (const uint8_t*)sc.hold.data_ptr(), sc.ld, sc.block_rows,
                                y.data_ptr<float>(), cols, s);
    });
  }
  return THPVariable_Wrap(y);
}

PyObject* fp8_matmul(PyObject* const* a) {
  const char* who = "fp8_matmul";
  const Tensor &A = tensor(a[0], "a"), &As = tensor(a[1], "a_scale"), &B = tensor(a[2], "b"),
               &Bs = tensor(a[3], "b_scale");
  const Tensor* bias = optional(a[4], "bias");
  const int act = integer(a[5]);
  const Tensor* out = optional(a[6], "out");
  need_fp8(A, who);
  need_fp8(B, who);
  need_f32(bias);
  need_f32(out);
  same_device(A, {&As, &B, &Bs, bias, out});
  if (A.dim() != 2 || B.dim() != 2 || Bs.dim() != 2) refuse("Matmul only supports 2D");
  const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
  if (B.size(0) != K) refuse("Matmul dimension mismatch");
  const Vec bv = vec(bias, N, "fp8_matmul: bias must have N elements");
  if (out && (out->dim() != 2 || out->size(0) != M || out->size(1) != N ||
              (N > 1 && out->stride(1) != 1) || (M > 1 && out->stride(0) < N)))
    refuse("fp8_matmul: out must be [M, N] with contiguous rows");
  Tensor y = out ? *out : empty_f32(A, {M, N});
  const int64_t ldc = out && out->stride(0) > N ? out->stride(0) : N;
  const Rows ar = rows_of(A, K);
  const Scales sa = scales(As, M, K, who);
  const bool trans = B.stride(0) == 1 || B.stride(1) != 1;  // w.t() of a weight [N, K]
  const Rows br = trans ? rows_of(B.t(), K) : rows_of(B, N);
  Scales sb = trans ? scales(Bs.t(), N, K, who) : scales(Bs, K, N, who);
  if (!trans) {
    if (sb.block_rows != 128 && K > 1) refuse("fp8_matmul: a row-major b needs 128 x 128 blocks");
    sb.block_rows = 128;
  }
  rtb_ctx* ctx = context(A.device().index());
  void* s = stream_of(A);
  call("rtb_fp8_matmul", [&] {
    return rtb_fp8_matmul(ctx, M, N, K, (const uint8_t*)ar.p(), ar.ld, sa.hold.data_ptr(), sa.ld,
                          sa.block_rows, sa.type, (const uint8_t*)br.p(), br.ld, trans,
                          sb.hold.data_ptr(), sb.ld, sb.block_rows, sb.type, bv.p, act,
                          y.data_ptr<float>(), ldc, s);
  });
  return THPVariable_Wrap(y);
}

// A caller's output of x's shape as rows; a fresh one where none is given.
struct Out {
  Tensor t;
  int64_t ld = 0;
};
Out output(const Tensor* out, const Tensor& x, int64_t d, const char* who, const char* name) {
  Out o;
  o.ld = d;
  if (!out) {
    o.t = empty_f32(x, x.sizes());
    return o;
  }
  if (out->sizes() != x.sizes() || (d > 1 && out->stride(-1) != 1))
    refuse(std::string(who) + ": " + name + " must have x's shape and contiguous rows");
  o.t = *out;
  if (!out->is_contiguous()) {
    const Tensor o2 = out->dim() == 2 ? *out : out->view({-1, d});
    if (o2.size(0) > 1 && o2.stride(0) < d) refuse(std::string(who) + ": " + name + "'s rows overlap");
    o.ld = o2.stride(0) > d ? o2.stride(0) : d;
  }
  return o;
}

const char* const kRmsShape = "RMSNorm: Input shape does not match normalized shape";

// rms_norm_fwd and rms_norm_fp8
PyObject* rms_norm(const char* who, bool fp8, PyObject* ax, PyObject* aw, PyObject* aeps, PyObject* ar,
                   PyObject* aout, PyObject* asum) {
  const Tensor& x = tensor(ax, "x");
  const Tensor* w = optional(aw, "norm_weight");
  const float eps = (float)real(aeps);
  const Tensor *res = optional(ar, "residual"), *out = optional(aout, "out"),
               *out_sum = optional(asum, "out_sum");
  for (const Tensor* t : {&x, w, res, out, out_sum}) need_f32(t);
  same_device(x, {w, res, out, out_sum});
  const int64_t d = x.dim() ? x.size(-1) : 0;
  if (d == 0) refuse("RMSNorm: Input shape smaller than normalized shape");
  if (res && res->sizes() != x.sizes()) refuse(std::string(who) + ": residual must have x's shape");
  const Vec wv = vec(w, d, kRmsShape);
  const Rows xr = rows_of(x, d);
  Rows rr;
  if (res) rr = rows_of(*res, d);
  const bool store = res || out_sum;  // without a residual the sum is x
  Out sum, y;
  if (store) sum = output(out_sum, x, d, who, "out_sum");
  Tensor q, scale;
  const int64_t cb = (d + 127) / 128;
  if (fp8) {
    q = at::empty(x.sizes(), x.options().dtype(ScalarType::Float8_e4m3fn));
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = cb;
    scale = at::empty(shape, x.options().dtype(ScalarType::Float8_e8m0fnu));
  } else {
    y = output(out, x, d, who, "out");
  }
  Tensor rstd = empty_f32(x, x.sizes().slice(0, x.dim() - 1));
  rtb_ctx* ctx = context(x.device().index());
  void* s = stream_of(x);
  call(fp8 ? "rtb_rms_norm_fp8" : "rtb_rms_norm_fwd", [&] {
    const float* px = (const float*)xr.p();
    const float* pr = res ? (const float*)rr.p() : nullptr;
    float* ps = store ? sum.t.data_ptr<float>() : nullptr;
    float* prstd = rstd.data_ptr<float>();
    if (fp8)
      return rtb_rms_norm_fp8(ctx, xr.rows, d, px, xr.ld, pr, rr.ld, wv.p, eps, ps, sum.ld,
                              (uint8_t*)q.data_ptr(), d, (uint8_t*)scale.data_ptr(), cb, prstd, s);
    return rtb_rms_norm_fwd(ctx, xr.rows, d, px, xr.ld, pr, rr.ld, wv.p, eps, ps, sum.ld,
                            y.t.data_ptr<float>(), y.ld, prstd, s);
  });
  PyObject* total = THPVariable_Wrap(store ? sum.t : x);
  if (fp8) return pack({THPVariable_Wrap(q), THPVariable_Wrap(scale), total, THPVariable_Wrap(rstd)});
  return pack({THPVariable_Wrap(y.t), total, THPVariable_Wrap(rstd)});
}
PyObject* rms_norm_fwd(PyObject* const* a) {
  return rms_norm("rms_norm_fwd", false, a[0], a[1], a[2], a[3], a[4], a[5]);
}
PyObject* rms_norm_fp8(PyObject* const* a) {
  return rms_norm("rms_norm_fp8", true, a[0], a[1], a[2], a[3], Py_None, a[4]);
}

PyObject* rms_norm_backward(PyObject* const* a) {
  const char* who = "rms_norm_backward";
  const Tensor& x = tensor(a[0], "x");
  const Tensor &rstd = tensor(a[1], "rstd"), &grad = tensor(a[2], "grad");
  const Tensor *w = optional(a[3], "norm_weight"), *gs = optional(a[4], "grad_sum"),
               *xs = optional(a[5], "x_scale");
  const bool need_x = flag(a[6]), need_w = flag(a[7]);
  const Tensor *ox = optional(a[8], "out_x"), *ow = optional(a[9], "out_weight");
  const bool accumulate = flag(a[10]);
  const bool saved = x.scalar_type() == ScalarType::Float8_e4m3fn;
  for (const Tensor* t : {&rstd, &grad, w, gs, ox, ow}) need_f32(t);
  if (saved) need_fp8(x, who);
  else need_f32(&x);
  same_device(x, {&rstd, &grad, w, gs, xs, ox, ow});
  const int64_t d = x.dim() ? x.size(-1) : 0;
  if (d == 0 || grad.sizes() != x.sizes() || (gs && gs->sizes() != x.sizes()))
    refuse("rms_norm_backward: grad and grad_sum must have x's shape, with a last dimension");
  const Rows xr = rows_of(x, d), gr = rows_of(grad, d);
  Rows sr;
  if (gs) sr = rows_of(*gs, d);
  const Vec rv = vec(&rstd, xr.rows, "rms_norm_backward: one rstd for each row");
  const Vec wv = vec(w, d, kRmsShape);
  if (saved != (xs != nullptr))
    refuse("rms_norm_backward: x_scale goes with an 8-bit x, and only with one");
  auto dx = result(ox, need_x, accumulate, x.sizes(), grad, who);
  auto dw = result(ow, need_w, accumulate, {d}, grad, who);
  Scales sc;
  if (saved) {
    sc = scales(*xs, xr.rows, d, who);
    if (sc.type != RTB_SCALE_E8M0 || sc.block_rows != 1)
      refuse("rms_norm_backward: a checkpoint has a power-of-two scale for each 128 columns of a row");
  }
  rtb_ctx* ctx = context(x.device().index());
  void* s = stream_of(x);
  float *px = ptr(dx), *pw = ptr(dw);
  call(saved ? "rtb_rms_norm_backward_fp8" : "rtb_rms_norm_backward", [&] {
    const float* pg = (const float*)gr.p();
    const float* ps = gs ? (const float*)sr.p() : nullptr;
    if (saved)
      return rtb_rms_norm_backward_fp8(ctx, xr.rows, d, (const uint8_t*)xr.p(), xr.ld,
                                       (const uint8_t*)sc.hold.data_ptr(), sc.ld, rv.p, wv.p, pg,
                                       gr.ld, ps, sr.ld, px, d, pw, accumulate, s);
    return rtb_rms_norm_backward(ctx, xr.rows, d, (const float*)xr.p(), xr.ld, rv.p, wv.p, pg, gr.ld,
                                 ps, sr.ld, px, d, pw, accumulate, s);
  });
  return pack({wrap(dx), wrap(dw)});
}

// The rows that a tensor's leading dimensions count (a last dimension of 0 has some too).
int64_t leading(const Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}
// A tensor of one-byte elements as rows of d contiguous bytes that do not overlap; trans:
// as the rows of its transpose.  No view is made where it lies so already.
Rows byte_rows(const Tensor& t, bool trans) {
  if (t.dim() == 2) {
    const int64_t rows = t.size(trans ? 1 : 0), d = t.size(trans ? 0 : 1);
    const int64_t rs = t.stride(trans ? 1 : 0), cs = t.stride(trans ? 0 : 1);
    if ((d <= 1 || cs == 1) && (rows <= 1 || rs >= d)) {
      Rows r;
      r.hold = t;
      r.rows = rows;
      r.ld = rs > d ? rs : d;
      return r;
    }
  }
  const Tensor bytes = t.view(ScalarType::Byte);
  return rows_of(trans ? bytes.t() : bytes, t.size(trans ? 0 : -1));
}
// A 4-bit tensor's codes (its last dimension, or its first, counts bytes).
Rows codes(const Tensor& t, bool trans, const char* who) {
  if (!(t.is_cuda() && t.scalar_type() == ScalarType::Float4_e2m1fn_x2))
    refuse(std::string(who) + " expects float4_e2m1fn_x2 CUDA tensors");
  if (t.dim() == 0) refuse(std::string(who) + ": a 4-bit tensor needs a last dimension");
  return byte_rows(t, trans);
}
Rows scales4(const Tensor& s, bool trans, int64_t rows, int64_t cols, const char* who) {
  if (!(s.is_cuda() && s.scalar_type() == ScalarType::Float8_e8m0fnu))
    refuse(std::string(who) + ": scales are float8_e8m0fnu CUDA tensors");
  const int64_t cb = (cols + 31) / 32;
  if (s.dim() < 1 || s.size(trans ? 0 : -1) != cb || (trans ? s.size(1) : leading(s)) != rows)
    refuse(std::string(who) + ": scales must be [rows, ceil(cols / 32)]");
  return byte_rows(s, trans);
}

PyObject* fp4_quantize(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x");
  need_f32(&x);
  if (x.dim() == 0) refuse("fp4_quantize: x needs a last dimension");
  const int64_t cols = x.size(-1), half = (cols + 1) / 2, cb = (cols + 31) / 32;
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = half;
  Tensor q = at::empty(shape, x.options().dtype(ScalarType::Float4_e2m1fn_x2));
  shape.back() = cb;
  Tensor scale = at::empty(shape, x.options().dtype(ScalarType::Float8_e8m0fnu));
  if (x.numel()) {
    // the transposed view of a row-major matrix stays where it is
    const bool trans = x.dim() == 2 && !x.is_contiguous() && x.stride(0) == 1 && x.stride(1) >= x.size(0);
    Rows xr;
    if (trans) {
      xr.hold = x;
      xr.rows = x.size(0);
      xr.ld = x.stride(1);
    } else {
      xr = rows_of(x, cols);
    }
    rtb_ctx* ctx = context(x.device().index());
    void* s = stream_of(x);
    call("rtb_fp4_quantize", [&] {
      return rtb_fp4_quantize(ctx, xr.rows, cols, (const float*)xr.p(), xr.ld, trans,
                              (uint8_t*)q.data_ptr(), half, (uint8_t*)scale.data_ptr(), cb, s);
    });
  }
  return pack({THPVariable_Wrap(q), THPVariable_Wrap(scale)});
}

PyObject* fp4_dequantize(PyObject* const* a) {
  const char* who = "fp4_dequantize";
  const Tensor &q = tensor(a[0], "q"), &scale = tensor(a[1], "scale");
  int64_t cols = integer(a[2]);
  const Tensor* out = optional(a[3], "out");
  need_f32(out);
  same_device(q, {&scale, out});
  const Rows qr = codes(q, false, who);
  if (cols == -1) cols = 2 * q.size(-1);
  if (cols < 0 || (cols + 1) / 2 != q.size(-1))
    refuse("fp4_dequantize: q holds two columns in each byte of its last dimension");
  const Rows sr = scales4(scale, false, leading(q), cols, who);
  c10::SmallVector<int64_t, 6> shape(q.sizes().begin(), q.sizes().end());
  shape.back() = cols;
  if (out && (out->sizes() != at::IntArrayRef(shape) || !out->is_contiguous()))
    refuse("fp4_dequantize: out must be contiguous, with q's leading shape and its columns");
  Tensor y = out ? *out : empty_f32(q, shape);
  if (y.numel()) {
    rtb_ctx* ctx = context(q.device().index());
    void* s = stream_of(q);
    call("rtb_fp4_dequantize", [&] {
      return rtb_fp4_dequantize(ctx, qr.rows, cols, (const uint8_t*)qr.p(), qr.ld,
                                (const uint8_t*)sr.p(), sr.ld, y.data_ptr<float>(), cols, s);
    });
  }
  return THPVariable_Wrap(y);
}

PyObject* fp4_matmul(PyObject* const* a) {
  const char* who = "fp4_matmul";
  const Tensor &A = tensor(a[0], "a"), &As = tensor(a[1], "a_scale"), &B = tensor(a[2], "b"),
               &Bs = tensor(a[3], "b_scale");
  const Tensor* bias = optional(a[4], "bias");
  const int act = integer(a[5]);
  const Tensor* out = optional(a[6], "out");
  need_f32(bias);
  need_f32(out);
  same_device(A, {&As, &B, &Bs, bias, out});
  if (A.dim() != 2 || B.dim() != 2 || Bs.dim() != 2) refuse("Matmul only supports 2D");
  const int64_t M = A.size(0), K = 2 * A.size(1), N = B.size(1);
  if (2 * B.size(0) != K) refuse("Matmul dimension mismatch");
  const Rows ar = codes(A, false, who), br = codes(B, true, who);
  const Rows sa = scales4(As, false, M, K, who), sb = scales4(Bs, true, N, K, who);
  const Vec bv = vec(bias, N, "fp4_matmul: bias must have N elements");
  if (out && (out->dim() != 2 || out->size(0) != M || out->size(1) != N ||
              (N > 1 && out->stride(1) != 1) || (M > 1 && out->stride(0) < N)))
    refuse("fp4_matmul: out must be [M, N] with contiguous rows");
  Tensor y = out ? *out : empty_f32(A, {M, N});
  const int64_t ldc = out && out->stride(0) > N ? out->stride(0) : N;
  rtb_ctx* ctx = context(A.device().index());
  void* s = stream_of(A);
  call("rtb_fp4_matmul", [&] {
    return rtb_fp4_matmul(ctx, M, N, K, (const uint8_t*)ar.p(), ar.ld, (const uint8_t*)sa.p(), sa.ld,
                          (const uint8_t*)br.p(), br.ld, (const uint8_t*)sb.p(), sb.ld, bv.p, act,
                          y.data_ptr<float>(), ldc, s);
  });
  return THPVariable_Wrap(y);
}

PyObject* matmul_backward_fp8(PyObject* const* a) {
  const char* who = "matmul_backward_fp8";
  const Tensor &A = tensor(a[0], "a"), &As = tensor(a[1], "a_scale");
  const Tensor* B = optional(a[2], "b");
  const Tensor& grad = tensor(a[3], "grad");
  const bool need_a = flag(a[4]), need_b = flag(a[5]);
  const Tensor *oa = optional(a[6], "out_a"), *ob = optional(a[7], "out_b");
  const bool accumulate = flag(a[8]);
  const int precision = integer(a[9]);
  need_fp8(A, who);
  for (const Tensor* t : {B, &grad, oa, ob}) need_f32(t);
  same_device(A, {&As, B, &grad, oa, ob});
  if (A.dim() != 2 || grad.dim() != 2) refuse("Matmul only supports 2D");
  const int64_t M = A.size(0), K = A.size(1), N = grad.size(1);
  if (grad.size(0) != M || (B && (B->dim() != 2 || B->size(0) != K || B->size(1) != N)))
    refuse("matmul_backward_fp8: shape mismatch");
  if (need_a && !B) refuse("matmul_backward_fp8: the gradient of a needs b");
  auto da = result(oa, need_a, accumulate, {M, K}, grad, who);
  auto db = result(ob, need_b, accumulate, {K, N}, grad, who);
  const Tensor g = grad.is_contiguous() ? grad : grad.contiguous();
  const Tensor b = B && need_a ? B->contiguous() : Tensor();
  const Rows ar = rows_of(A, K);
  const Scales sa = scales(As, M, K, who);
  if (sa.type != RTB_SCALE_E8M0)
    refuse("matmul_backward_fp8: a checkpoint's scales are float8_e8m0fnu");
  rtb_ctx* ctx = context(A.device().index());
  void* s = stream_of(A);
  float *pa = ptr(da), *pb = ptr(db);
  call("rtb_matmul_backward_fp8", [&] {
    return rtb_matmul_backward_fp8(ctx, M, N, K, (const uint8_t*)ar.p(), ar.ld,
                                   (const uint8_t*)sa.hold.data_ptr(), sa.ld, sa.block_rows,
                                   b.defined() ? b.data_ptr<float>() : nullptr,
                                   g.data_ptr<float>(), pa, pb, accumulate, precision, s);
  });
  return pack({wrap(da), wrap(db)});
}

// ------------------------------------------------------------------ module
template <PyObject* (*F)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
  try {
    return F(args);
  } catch (const PyFailure&) {
    return nullptr;
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {  // torch's own errors (an allocation that failed)
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// setup(get_context, check)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "expected 2 arguments, got %zd", n);
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XSETREF(g_get_context, args[0]);
  Py_XSETREF(g_check, args[1]);
  Py_RETURN_NONE;
}

#define ENTRY(name, args) \
  {#name, (PyCFunction)(void (*)(void))entry<name, args>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, nullptr},
    ENTRY(layer_norm_fwd, 6),
    ENTRY(layer_norm_backward, 15),
    ENTRY(fp8_quantize, 2),
    ENTRY(fp8_dequantize, 3),
    ENTRY(fp8_matmul, 7),
    ENTRY(matmul_backward_fp8, 10),
    ENTRY(rms_norm_fwd, 6),
    ENTRY(rms_norm_fp8, 5),
    ENTRY(rms_norm_backward, 11),
    ENTRY(fp4_quantize, 1),
    ENTRY(fp4_dequantize, 4),
    ENTRY(fp4_matmul, 7),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) {
  g_handle_name = PyUnicode_InternFromString("handle");
  g_value_name = PyUnicode_InternFromString("value");
  if (!g_handle_name || !g_value_name) return nullptr;
  return PyModule_Create(&module);
}
