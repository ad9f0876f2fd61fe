// _torchcall: the step from torch tensors to the C ABI (include/ppo_xp.h) for the operators on logits and quantised rows - argument
// checks, allocation of results with torch, torch's current stream.  Host code only; between calls it holds nothing but what setup()
// gives it and the address of torch's allocator.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>

#include "../../include/ppo_xp.h"

namespace {

struct Panic { std::string msg; };          // becomes PpoXpPanic: wrong arguments, nothing was launched
struct Raised {};                           // a Python error is set already

PyObject *g_panic = nullptr, *g_check = nullptr, *g_stream = nullptr;
decltype(&ppo_xp_shape_logits) g_shape;
decltype(&ppo_xp_shape_logits_backward) g_shape_backward;
decltype(&ppo_xp_action_stats) g_stats;
decltype(&ppo_xp_policy_loss) g_loss;
decltype(&ppo_xp_policy_workspace) g_workspace;
decltype(&ppo_xp_quantize_rows) g_quantize;
decltype(&ppo_xp_dequantize_rows) g_dequantize;

[[noreturn]] void panic(const std::string &msg) { throw Panic{msg}; }
std::string num(int64_t x) { return std::to_string(x); }

// A launch waits when the stream's queue is full: other Python threads run meanwhile.
template <class F, class... A>
int launch(F *f, A... a) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(a...);
  Py_END_ALLOW_THREADS
  return rc;
}

void done(int rc) {
  if (rc >= 0) return;
  PyObject *r = PyObject_CallFunction(g_check, "i", rc);    // raises with the library's message
  Py_XDECREF(r);
  throw Raised{};
}

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

const at::Tensor &some(PyObject *o, const char *what) {
  const at::Tensor *t = tensor(o);
  if (!t) panic(std::string(what) + ": a tensor expected");
  return *t;
}

int dtype_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PPO_XP_F32;
    case at::kBFloat16: return PPO_XP_BF16;
    case at::kHalf: return PPO_XP_F16;
    default: return -1;
  }
}

struct Matrix {
  int64_t rows, cols, stride;
  int dtype, device;
  void *p;
};

Matrix matrix(const at::Tensor &t, const char *what) {
  const int dt = dtype_of(t);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() != 2 || dt < 0) panic(std::string(what) + ": a 2-d CUDA tensor of f32, bf16 or f16 expected");
  Matrix m{t.size(0), t.size(1), t.stride(0), dt, (int)t.get_device(), t.data_ptr()};
  if ((m.cols > 1 && t.stride(1) != 1) || (m.rows > 1 && m.stride < m.cols)) panic(std::string(what) + ": rows must be contiguous and must not overlap");
  if (m.stride < m.cols) m.stride = m.cols;
  return m;
}

void *vector(PyObject *o, int64_t n, at::ScalarType type, int device, const char *what) {
  const at::Tensor *t = tensor(o);
  if (!t || t->scalar_type() != type || !t->is_cuda() || t->get_device() != device || t->dim() != 1 || t->numel() != n || !t->is_contiguous())
    panic(std::string(what) + ": contiguous " + at::toString(type) + " tensor of " + num(n) + " on cuda:" + num(device) + " expected");
  return t->data_ptr();
}

// `o`, or a new tensor of `like`'s shape and type.
at::Tensor result(PyObject *o, const at::Tensor &like, const char *what, Matrix &m) {
  at::Tensor out;
  if (o == Py_None) {
    out = at::empty(like.sizes(), like.options().memory_format(at::MemoryFormat::Contiguous).requires_grad(false));
  } else {
    out = some(o, what);
    if (out.scalar_type() != like.scalar_type() || out.device() != like.device() || out.sizes() != like.sizes())
      panic(std::string(what) + ": out must have the logits' shape, type and device");
  }
  m = matrix(out, what);
  return out;
}

// A caller's tensor has changed under autograd's eyes: what was saved of it for a backward pass is known to be stale.
void changed(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject *o, const at::Tensor &out) {
  if (o != Py_None) changed(out);
}

void *stream_of(int device) {
  PyObject *d = PyLong_FromLong(device), *r = d ? PyObject_CallOneArg(g_stream, d) : nullptr;
  Py_XDECREF(d);
  if (!r) throw Raised{};
  void *s = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  if (!s && PyErr_Occurred()) throw Raised{};
  return s;
}

float number(PyObject *o, const char *what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    panic(std::string(what) + ": a number or one f32 per row expected");
  }
  return (float)v;
}

// A rule given as one number or as one f32 per row.
void row_value(PyObject *o, int64_t rows, int device, const char *what, const float *&p, float &v) {
  p = nullptr;
  v = 1.f;
  if (tensor(o)) p = (const float *)vector(o, rows, at::kFloat, device, what);
  else v = number(o, what);
}

enum { HISTORY, HIST_ROW, HIST_BEGIN, GEN_BEGIN, HIST_END, REPETITION, PRESENCE, FREQUENCY, BIAS, MASK, MASK_ROW, TEMPERATURE, RULES };

ppo_xp_logit_rules rules_of(const Matrix &l, PyObject *const *a) {
  ppo_xp_logit_rules r{};
  r.history_bits = 64;
  if (a[HISTORY] != Py_None) {
    const at::Tensor &h = some(a[HISTORY], "history");
    const bool wide = h.scalar_type() == at::kLong;
    if (!h.is_cuda() || h.get_device() != l.device || h.dim() != 2 || (!wide && h.scalar_type() != at::kInt))
      panic("history: a 2-d int64 or int32 tensor [rows, positions] on the logits' device expected");
    r.history = h.data_ptr();
    r.hist_rows = h.size(0); r.hist_len = h.size(1); r.hist_row_stride = h.stride(0); r.hist_tok_stride = h.stride(1);
    r.history_bits = wide ? 64 : 32;
    if (a[HIST_ROW] == Py_None && r.hist_rows != l.rows) panic("history: " + num(r.hist_rows) + " rows for " + num(l.rows) + " rows of logits (pass hist_row)");
    const int32_t **to[4] = {&r.hist_row, &r.hist_begin, &r.gen_begin, &r.hist_end};
    static const char *names[4] = {"hist_row", "hist_begin", "gen_begin", "hist_end"};
    for (int i = 0; i < 4; ++i)
      if (a[HIST_ROW + i] != Py_None) *to[i] = (const int32_t *)vector(a[HIST_ROW + i], l.rows, at::kInt, l.device, names[i]);
  } else {
    for (int i = HIST_ROW; i <= HIST_END; ++i)
      if (a[i] != Py_None) panic("hist_row, hist_begin, gen_begin and hist_end belong to a history");
  }
  row_value(a[REPETITION], l.rows, l.device, "repetition", r.repetition_rows, r.repetition);
  row_value(a[PRESENCE], l.rows, l.device, "presence", r.presence_rows, r.presence);
  row_value(a[FREQUENCY], l.rows, l.device, "frequency", r.frequency_rows, r.frequency);
  row_value(a[TEMPERATURE], l.rows, l.device, "temperature", r.temperature_rows, r.temperature);
  if (r.presence_rows) r.presence = 0.f;
  if (r.frequency_rows) r.frequency = 0.f;
  if (a[BIAS] != Py_None) {
    const at::Tensor &b = some(a[BIAS], "bias");
    const int64_t dim = b.dim();
    if (!b.is_cuda() || b.get_device() != l.device || b.scalar_type() != at::kFloat || (dim != 1 && dim != 2) || b.size(dim - 1) != l.cols ||
        (dim == 2 && b.size(0) != l.rows) || (l.cols > 1 && b.stride(dim - 1) != 1))
      panic("bias: f32 tensor [vocab] or [rows, vocab] with contiguous rows on the logits' device expected");
    r.bias = b.data_ptr<float>();
    r.bias_stride = dim == 2 && l.rows > 1 ? b.stride(0) : 0;
  }
  if (a[MASK] != Py_None) {
    const at::Tensor &m = some(a[MASK], "mask");
    const int64_t dim = m.dim();
    if (!m.is_cuda() || m.get_device() != l.device || (dim != 1 && dim != 2)) panic("mask: a tensor [rows, ...] or [...] on the logits' device expected");
    int64_t need;
    switch (m.scalar_type()) {
      case at::kBool: case at::kByte: r.mask_kind = PPO_XP_MASK_BYTES; need = l.cols; break;
      case at::kInt: case at::kUInt32: r.mask_kind = PPO_XP_MASK_BITS; need = (l.cols + 31) / 32; break;
      default: panic("mask: bool / uint8 per token, or int32 words of 32 tokens expected");
    }
    r.mask_rows = dim == 2 ? m.size(0) : 1;
    if (m.size(dim - 1) != need || (need > 1 && m.stride(dim - 1) != 1)) panic("mask: contiguous rows of " + num(need) + " expected");
    if (a[MASK_ROW] != Py_None) r.mask_row = (const int32_t *)vector(a[MASK_ROW], l.rows, at::kInt, l.device, "mask_row");
    else if (dim == 2 && r.mask_rows != l.rows) panic("mask: " + num(r.mask_rows) + " rows for " + num(l.rows) + " rows of logits (pass mask_row)");
    r.mask = m.data_ptr();
    r.mask_stride = dim == 2 && r.mask_rows > 1 ? m.stride(0) : 0;
    if (r.mask_rows == 0) r.mask_kind = PPO_XP_MASK_NONE;
  } else if (a[MASK_ROW] != Py_None) {
    panic("mask_row belongs to a mask");
  }
  return r;
}

// ---- calls (positional; the Python functions above them document the arguments) --------------------------------------------

PyObject *shape(PyObject *const *a) {                       // logits, rules, out
  const at::Tensor &t = some(a[0], "shape_logits");
  const Matrix l = matrix(t, "shape_logits");
  const ppo_xp_logit_rules r = rules_of(l, a + 1);
  Matrix o;
  at::Tensor out = result(a[1 + RULES], t, "shape_logits", o);
  done(launch(g_shape, l.device, stream_of(l.device), l.dtype, l.p, l.stride, o.p, o.stride, l.rows, l.cols, &r));
  written(a[1 + RULES], out);
  return THPVariable_Wrap(out);
}

PyObject *shape_backward(PyObject *const *a) {              // grad, logits, rules, out
  const char *who = "shape_logits_backward";
  const at::Tensor &g = some(a[0], who), &t = some(a[1], who);
  const Matrix l = matrix(t, who);
  if (g.scalar_type() != t.scalar_type() || g.device() != t.device() || g.sizes() != t.sizes())
    panic("shape_logits_backward: grad must have the logits' shape, type and device");
  const Matrix m = matrix(g, who);
  const ppo_xp_logit_rules r = rules_of(l, a + 2);
  Matrix o;
  at::Tensor out = result(a[2 + RULES], g, who, o);
  done(launch(g_shape_backward, l.device, stream_of(l.device), l.dtype, m.p, m.stride, l.p, l.stride, o.p, o.stride, l.rows, l.cols, &r));
  written(a[2 + RULES], out);
  return THPVariable_Wrap(out);
}

// Results and workspace of one call, each an allocation of torch's of its own on `like`'s device: no result keeps another or the
// workspace, and calls on two streams and two captured graphs share nothing.  They come straight from the allocator that at::empty
// takes: five of them cost an objective's host time 0.8 us more than a single at::empty, as five of those 2.3 us.
class Fresh {
 public:
  explicit Fresh(const at::Tensor &like) : on_(like.device()), from_(allocator(like)) {}
  at::Tensor floats(int64_t n) const {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(c10::Storage::use_byte_size_t(), n * sizeof(float), from_->allocate(n * sizeof(float)), from_, true),
        c10::DispatchKeySet(c10::DispatchKey::CUDA), caffe2::TypeMeta::Make<float>());
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
  }
  c10::DataPtr memory(size_t bytes) const { return bytes ? from_->allocate(bytes) : c10::DataPtr(); }

 private:
  static c10::Allocator *allocator(const at::Tensor &like) {
    static c10::Allocator *a = nullptr;                       // under the interpreter's lock, so no other one is needed
    if (!a) a = at::empty({1}, at::TensorOptions().device(like.device())).storage().allocator();
    return a;
  }
  const c10::DeviceGuard on_;              // the allocator works on the current device
  c10::Allocator *const from_;
};

PyObject *stats(PyObject *const *a) {                       // logits, actions
  const at::Tensor &t = some(a[0], "action_stats");
  const Matrix l = matrix(t, "action_stats");
  const void *actions = vector(a[1], l.rows, at::kLong, l.device, "actions");
  const Fresh fresh(t);
  const at::Tensor nlp = fresh.floats(l.rows), ent = fresh.floats(l.rows);
  if (l.cols == 0) { nlp.zero_(); ent.zero_(); }
  const size_t bytes = g_workspace(l.rows, l.cols, 0);
  const c10::DataPtr ws = fresh.memory(bytes);
  done(launch(g_stats, l.device, stream_of(l.device), l.dtype, l.p, l.stride, (const int64_t *)actions, nlp.data_ptr<float>(), ent.data_ptr<float>(),
              l.rows, l.cols, ws.get(), bytes));
  PyObject *r = PyTuple_New(2);
  if (!r) throw Raised{};
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(nlp));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ent));
  return r;
}

struct Attr {                                               // an attribute, held while the call runs
  PyObject *o;
  Attr(PyObject *of, const char *name) : o(PyObject_GetAttrString(of, name)) { if (!o) throw Raised{}; }
  ~Attr() { Py_DECREF(o); }
  Attr(const Attr &) = delete;
};

PyObject *loss(PyObject *const *a) {                        // logits, values, batch, clip, ent_coef, vf_coef, denom, out
  const char *who = "policy_loss";
  const at::Tensor &t = some(a[0], who);
  const Matrix l = matrix(t, who);
  const Attr actions(a[2], "actions"), values(a[2], "values"), neglogps(a[2], "neglogps"), returns(a[2], "returns"), advantages(a[2], "advantages");
  ppo_xp_policy_batch b;
  b.actions = (const int64_t *)vector(actions.o, l.rows, at::kLong, l.device, "batch.actions");
  b.old_values = (const float *)vector(values.o, l.rows, at::kFloat, l.device, "batch.values");
  b.old_neglogps = (const float *)vector(neglogps.o, l.rows, at::kFloat, l.device, "batch.neglogps");
  b.returns = (const float *)vector(returns.o, l.rows, at::kFloat, l.device, "batch.returns");
  b.advantages = (const float *)vector(advantages.o, l.rows, at::kFloat, l.device, "batch.advantages");
  b.values = (const float *)vector(a[1], l.rows, at::kFloat, l.device, "values");
  const float clip = number(a[3], "clip"), ent_coef = number(a[4], "ent_coef"), vf = number(a[5], "vf_coef");
  double denom = l.rows ? (double)l.rows : 1.;
  if (a[6] != Py_None) {
    denom = PyFloat_AsDouble(a[6]);
    if (denom == -1.0 && PyErr_Occurred()) { PyErr_Clear(); panic("denom: a number expected"); }
  }
  Matrix o;
  at::Tensor out = result(a[7], t, who, o);
  const Fresh fresh(t);
  const at::Tensor dvalues = fresh.floats(l.rows), nlp = fresh.floats(l.rows), ent = fresh.floats(l.rows), stats = fresh.floats(6);
  if (l.rows == 0 || l.cols == 0)
    for (const at::Tensor *x : {&dvalues, &nlp, &ent, &stats}) x->zero_();
  const size_t bytes = g_workspace(l.rows, l.cols, 1);
  const c10::DataPtr ws = fresh.memory(bytes);
  done(launch(g_loss, l.device, stream_of(l.device), l.dtype, l.p, l.stride, &b, clip, ent_coef, vf, denom, o.p, o.stride, dvalues.data_ptr<float>(),
              nlp.data_ptr<float>(), ent.data_ptr<float>(), stats.data_ptr<float>(), l.rows, l.cols, ws.get(), bytes));
  written(a[7], out);
  PyObject *r = PyTuple_New(5);
  if (!r) throw Raised{};
  int i = 0;
  const at::Tensor *const all[] = {&stats, &out, &dvalues, &nlp, &ent};
  for (const at::Tensor *x : all) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(*x));
  return r;
}

int64_t whole(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

struct Store {
  at::Tensor codes, scales;
  int64_t width, kind, group;
  int64_t codes_stride, scales_stride;
};

// codes, scales, row size, PPO_XP_Q_*, group.  QuantizedRows has checked them once; its tensors may have been exchanged since.
Store store_of(PyObject *const *a) {
  Store s{some(a[0], "codes"), some(a[1], "scales"), whole(a[2]), whole(a[3]), whole(a[4]), 0, 0};
  if (s.group < 1) panic("QuantizedRows: group " + num(s.group) + " is not positive");
  const int64_t bytes = s.kind == PPO_XP_Q_INT4 ? (s.width + 1) / 2 : s.width;
  if (!s.codes.is_cuda() || s.codes.device() != s.scales.device() || s.codes.dim() != 2 || s.scales.dim() != 2 || s.codes.element_size() != 1 ||
      s.scales.scalar_type() != at::kFloat || s.codes.size(1) != bytes || s.scales.size(1) != (s.width + s.group - 1) / s.group ||
      s.codes.size(0) != s.scales.size(0) || (s.codes.size(1) > 1 && s.codes.stride(1) != 1) || (s.scales.size(1) > 1 && s.scales.stride(1) != 1))
    panic("QuantizedRows: codes and scales no longer have the shapes they were made with");
  // rows that share storage (expanded ones, say) would be addressed as if they lay apart, beyond its end
  if (s.codes.size(0) > 1 && (s.codes.stride(0) < s.codes.size(1) || s.scales.stride(0) < s.scales.size(1)))
    panic("QuantizedRows: rows of codes and scales must not overlap");
  s.codes_stride = std::max<int64_t>(s.codes.stride(0), s.codes.size(1));
  s.scales_stride = std::max<int64_t>(s.scales.stride(0), s.scales.size(1));
  return s;
}

PyObject *write(PyObject *const *a) {                       // store, rows, at
  const Store s = store_of(a);
  const Matrix m = matrix(some(a[5], "write"), "write");
  const int64_t at = whole(a[6]);
  if (m.cols != s.width || m.device != s.codes.get_device() || at < 0)
    panic("write: rows of " + num(s.width) + " on cuda:" + num(s.codes.get_device()) + " and at >= 0 expected");
  done(launch(g_quantize, m.device, stream_of(m.device), m.dtype, m.p, m.stride, m.rows, m.cols, (int)s.kind, s.group, s.codes.data_ptr(), s.codes_stride,
                  s.scales.data_ptr<float>(), s.scales_stride, s.codes.size(0), at));
  changed(s.codes);
  changed(s.scales);
  Py_RETURN_NONE;
}

PyObject *read(PyObject *const *a) {                        // store, index or None, first row, rows, dtype (PPO_XP_*), out
  const Store s = store_of(a);
  const int device = (int)s.codes.get_device();
  int64_t first = 0, n = 0;
  const void *index = nullptr;
  int bits = 0;
  if (a[5] == Py_None) {
    first = whole(a[6]);
    n = whole(a[7]);
  } else {
    const at::Tensor &i = some(a[5], "read");
    if ((i.scalar_type() != at::kInt && i.scalar_type() != at::kLong) || !i.is_cuda() || i.get_device() != device || i.dim() != 1 || !i.is_contiguous())
      panic("read: a contiguous int32 or int64 index on the store's device expected");
    n = i.numel();
    index = n ? i.data_ptr() : nullptr;
    bits = i.scalar_type() == at::kInt ? 32 : 64;
  }
  const int64_t dt = whole(a[8]);
  const at::ScalarType type = dt == PPO_XP_F32 ? at::kFloat : dt == PPO_XP_BF16 ? at::kBFloat16 : at::kHalf;
  at::Tensor out;
  if (a[9] == Py_None) {
    out = at::empty({n, s.width}, at::TensorOptions().dtype(type).device(s.codes.device()));
  } else {
    out = some(a[9], "read");
    if (out.scalar_type() != type || out.device() != s.codes.device() || out.dim() != 2 || out.size(0) != n || out.size(1) != s.width)
      panic(std::string("read: out must be ") + at::toString(type) + " [" + num(n) + ", " + num(s.width) + "] on the store's device");
  }
  const Matrix o = matrix(out, "read");
  done(launch(g_dequantize, device, stream_of(device), (int)dt, s.codes.data_ptr(), s.codes_stride, s.scales.data_ptr<float>(), s.scales_stride, s.codes.size(0),
                    s.width, (int)s.kind, s.group, index, bits, first, n, o.p, o.stride));
  written(a[9], out);
  return THPVariable_Wrap(out);
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", N, n);
  try {
    return F(args);
  } catch (const Panic &e) {
    if (PyObject *x = PyObject_CallFunction(g_panic, "is", PPO_XP_EINVAL, e.msg.c_str())) {
      PyErr_SetObject(g_panic, x);
      Py_DECREF(x);
    }
  } catch (const Raised &) {
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(PyExc_MemoryError, e.what());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject *setup(PyObject *, PyObject *args) {               // PpoXpPanic, check, raw stream of a device, addresses of the entry points
  PyObject *p, *c, *s;
  unsigned long long f[7];
  if (!PyArg_ParseTuple(args, "OOO(KKKKKKK)", &p, &c, &s, f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6)) return nullptr;
  Py_INCREF(p); Py_INCREF(c); Py_INCREF(s);
  g_panic = p; g_check = c; g_stream = s;
  g_shape = (decltype(g_shape))f[0];
  g_shape_backward = (decltype(g_shape_backward))f[1];
  g_stats = (decltype(g_stats))f[2];
  g_workspace = (decltype(g_workspace))f[3];
  g_loss = (decltype(g_loss))f[4];
  g_quantize = (decltype(g_quantize))f[5];
  g_dequantize = (decltype(g_dequantize))f[6];
  Py_RETURN_NONE;
}

#define FAST(name, f, n) {name, (PyCFunction)(void (*)(void))call<f, n>, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                           FAST("shape", shape, 2 + RULES),
                           FAST("shape_backward", shape_backward, 3 + RULES),
                           FAST("stats", stats, 2),
                           FAST("loss", loss, 8),
                           FAST("write", write, 7),
                           FAST("read", read, 10),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&g_module); }
