// Python entry points of the training-step operators (module suika_b200._train): argument checks, output
// allocation on the tensors' device, and the call of the C entry on the current stream. A small call is
// all host time, and this layer takes a third of what the same steps take in Python through ctypes.
// Kernels and everything else about the operators are behind the C ABI, which this module links.
#include "../../include/suika_reshard.h"

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/accumulate.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>
#include <vector>

namespace {

// A Python exception on its way: ValueError, AssertionError, or one that is set already.
struct Raise {
  PyObject* type;
  std::string msg;
};
[[noreturn]] void value_error(const std::string& m) { throw Raise{PyExc_ValueError, m}; }
[[noreturn]] void assertion_error(const std::string& m) { throw Raise{PyExc_AssertionError, m}; }
[[noreturn]] void already_set() { throw Raise{nullptr, ""}; }

// A status on its way to suika_b200._lib.check, which raises the exception that belongs to it.
struct Status {
  int rc;
};
void check(int rc) {
  if (rc != RS_OK) throw Status{rc};
}
void raise_status(int rc) {
  PyObject* lib = PyImport_ImportModule("suika_b200._lib");
  PyObject* r = lib ? PyObject_CallMethod(lib, "check", "i", rc) : nullptr;
  Py_XDECREF(r);
  Py_XDECREF(lib);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, rs_last_error());
}

// Allocation and launches run in `body` without the interpreter's lock: a full launch queue or a cudaMalloc
// waits in the driver, and other Python threads go on. Nothing of Python is touched in there; the arguments' own
// references, and for lists of tensors those of the caller's lists, keep the tensors until the call returns.
template <class F>
auto unlocked(F&& body) {
  struct Unlock {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlock() { PyEval_RestoreThread(state); }
  } unlock;
  return body();
}

template <class F>
PyObject* entry(F&& body) {
  try {
    return body();
  } catch (const Raise& r) {
    if (r.type) PyErr_SetString(r.type, r.msg.c_str());
  } catch (const Status& s) {
    raise_status(s.rc);
  } catch (const c10::OutOfMemoryError& e) {  // as torch's own operators raise them: the class, and no C++ stack
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
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

// ---- arguments ------------------------------------------------------------------------------
void count_args(const char* what, Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw Raise{PyExc_TypeError, std::string(what) + ": " + std::to_string(want) + " arguments are taken"};
}
const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Raise{PyExc_TypeError, std::string(what) + " must be a tensor"};
  const at::Tensor& t = THPVariable_Unpack(o);
  // a kernel would drop the tangent without a word (levels of forward-mode AD do not nest: 0 is the only one)
  if (t._fw_grad(0).defined()) value_error(std::string(what) + " with a forward-mode tangent: reverse mode alone is there");
  return t;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) already_set();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) already_set();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) already_set();
  return v != 0;
}
std::string type_name(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return RS_F32;
    case at::kBFloat16: return RS_BF16;
    case at::kHalf: return RS_F16;
    default: return -1;
  }
}
uint32_t dtype_code(const at::Tensor& t, const char* what) {
  const int c = code_of(t);
  if (c < 0) value_error(std::string(what) + " of " + type_name(t) + ": float32, bfloat16 and float16 are taken");
  return (uint32_t)c;
}
void need_cuda(const at::Tensor& t, const char* what) {
  if (!t.is_cuda()) value_error(std::string(what) + " must be a CUDA tensor");
}
c10::MaybeOwned<at::Tensor> index_tensor(const at::Tensor& t, const at::Tensor& with, const char* what) {
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    value_error(std::string(what) + " of " + type_name(t) + ": int64 and int32 are taken");
  if (t.device() != with.device()) value_error(std::string(what) + " must be on the device of the other tensors");
  return t.expect_contiguous();
}
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
// A tensor that a kernel wrote in place counts as written for autograd, as after torch's own in-place operators: a
// backward pass over what it held before is then an error. (Inference tensors keep no versions.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
std::string shape_of(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}
// [..., cols] as rows of `cols` contiguous elements; copies only what no stride describes.
at::Tensor as_rows(const at::Tensor& t, int64_t cols) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), cols});
  return r.stride(1) == 1 || cols < 2 ? r : r.contiguous();
}

// ---- embedding ------------------------------------------------------------------------------
PyObject* embed_lookup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("embed_lookup", n, 4);
    const at::Tensor& weight = tensor(a[1], "weight");
    need_cuda(weight, "weight");
    if (weight.dim() != 2) value_error("weight must be [rows, hidden]");
    const int64_t rows = weight.size(0), hidden = weight.size(1);
    const uint32_t code = dtype_code(weight, "weight");
    if (weight.stride(1) != 1 && hidden > 1) value_error("weight must have contiguous rows");
    const at::Tensor& given_ids = tensor(a[0], "ids");
    rs_embed_opts o{};
    o.rows = rows;
    o.hidden = hidden;
    o.lo = integer(a[3]);
    o.weight_stride = weight.stride(0);
    o.scale = (float)number(a[2]);
    o.dtype = o.grad_dtype = code;
    return THPVariable_Wrap(unlocked([&] {
      const auto held = index_tensor(given_ids, weight, "ids");
      const at::Tensor& ids = *held;
      std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
      shape.push_back(hidden);
      at::Tensor out = at::empty(shape, weight.options());
      o.n_tokens = ids.numel();
      o.wide_ids = ids.scalar_type() == at::kLong;
      check(rs_embed_lookup(&o, ids.data_ptr(), weight.data_ptr(), out.data_ptr(), weight.get_device(), stream_of(weight)));
      return out;
    }));
  });
}

// embed_grad(grad_out, ids, rows, scale, lo, dtype or None, out or None, accumulate)
PyObject* embed_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("embed_grad", n, 8);
    const at::Tensor& grad_out = tensor(a[0], "grad_out");
    need_cuda(grad_out, "grad_out");
    if (grad_out.dim() < 1) value_error("grad_out must be [..., hidden]");
    const int64_t hidden = grad_out.size(-1), rows = integer(a[2]);
    rs_embed_opts o{};
    o.dtype = dtype_code(grad_out, "grad_out");
    const at::Tensor& given_ids = tensor(a[1], "ids");
    o.accumulate = truth(a[7]);
    o.lo = integer(a[4]);
    o.scale = (float)number(a[3]);
    const bool has_dtype = a[5] != Py_None;
    if (has_dtype && !THPDtype_Check(a[5])) throw Raise{PyExc_TypeError, "dtype must be a torch.dtype"};
    const at::ScalarType dtype = has_dtype ? reinterpret_cast<THPDtype*>(a[5])->scalar_type : grad_out.scalar_type();
    at::Tensor out;
    if (a[6] != Py_None) out = tensor(a[6], "out");
    return THPVariable_Wrap(unlocked([&] {
      const auto held = index_tensor(given_ids, grad_out, "ids");
      const at::Tensor& ids = *held;
      if (grad_out.sizes().slice(0, grad_out.dim() - 1) != ids.sizes())
        assertion_error("grad_out has shape " + shape_of(grad_out.sizes()) + ", ids " + shape_of(ids.sizes()));
      const bool given = out.defined();
      if (!given) {
        if (o.accumulate) value_error("accumulate=True adds to `out`: give one");
        if (rows < 0) value_error("a negative number of rows");
        out = at::empty({rows, hidden}, grad_out.options().dtype(dtype));
      } else {
        if (out.device() != grad_out.device() || !out.is_contiguous()) value_error("out must be contiguous and on grad_out's device");
        if (out.dim() != 2 || out.size(0) != rows || out.size(1) != hidden)
          assertion_error("out has shape " + shape_of(out.sizes()) + ", expected " + shape_of({rows, hidden}));
        if (has_dtype && out.scalar_type() != dtype) value_error("out of " + type_name(out) + ", but a gradient of another type is asked for");
      }
      o.grad_dtype = dtype_code(out, "the gradient");
      const at::Tensor g = as_rows(grad_out, hidden);
      o.n_tokens = ids.numel();
      o.rows = rows;
      o.hidden = hidden;
      o.grad_stride = g.stride(0);
      o.wide_ids = ids.scalar_type() == at::kLong;
      const int device = grad_out.get_device();
      uint64_t bytes = 0;
      check(rs_embed_grad_workspace_bytes(&o, device, &bytes));
      const at::Tensor workspace = at::empty({(int64_t)bytes}, grad_out.options().dtype(at::kByte));
      check(rs_embed_grad(&o, ids.data_ptr(), g.data_ptr(), out.data_ptr(), workspace.data_ptr(), bytes, device, stream_of(grad_out)));
      if (given) written(out);
      return out;
    }));
  });
}

// ---- token log probabilities ------------------------------------------------------------------
struct Logits {
  at::Tensor z;
  c10::MaybeOwned<at::Tensor> targets;
  rs_logprob_opts o{};
  Logits(const at::Tensor& logits, const at::Tensor& t, int64_t top, int64_t lo, bool sharded) {
    need_cuda(logits, "logits");
    o.dtype = dtype_code(logits, "logits");
    targets = index_tensor(t, logits, "targets");
    if (logits.dim() < 1 || logits.sizes().slice(0, logits.dim() - 1) != t.sizes())
      assertion_error("logits have shape " + shape_of(logits.sizes()) + ", targets " + shape_of(t.sizes()));
    const int64_t cols = logits.size(-1);
    if (cols == 0) value_error("logits of no columns");
    z = as_rows(logits, cols);
    o.n_rows = z.size(0);
    o.cols = cols;
    o.stride = z.stride(0);
    o.lo = lo;
    o.wide_targets = t.scalar_type() == at::kLong;
    o.top = (int32_t)top;
    o.sharded = sharded;
  }
};

int64_t top_of(PyObject* p) {
  const int64_t top = integer(p);
  if (top < 0 || top > 32) value_error("top must be in 0..32");
  return top;
}

// token_logprobs(logits, targets, top, lo) -> (logprob, entropy, lse, top_logprob or None, top_index or None)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("token_logprobs", n, 4);
    const int64_t top = top_of(a[2]);
    const at::Tensor &logits = tensor(a[0], "logits"), &targets = tensor(a[1], "targets");
    const int64_t lo = integer(a[3]);
    at::Tensor out[5];
    unlocked([&] {
      const Logits l(logits, targets, top, lo, false);
      const auto f32 = logits.options().dtype(at::kFloat);
      for (int i = 0; i < 3; ++i) out[i] = at::empty(targets.sizes(), f32);
      if (top) {
        std::vector<int64_t> shape(targets.sizes().begin(), targets.sizes().end());
        shape.push_back(top);
        out[3] = at::empty(shape, f32);
        out[4] = at::empty(shape, logits.options().dtype(at::kLong));
      }
      check(rs_token_logprobs(&l.o, l.z.data_ptr(), l.targets->data_ptr(), out[0].data_ptr<float>(), out[1].data_ptr<float>(),
                              out[2].data_ptr<float>(), top ? out[3].data_ptr<float>() : nullptr, top ? out[4].data_ptr<int64_t>() : nullptr,
                              logits.get_device(), stream_of(logits)));
    });
    PyObject* r = PyTuple_New(5);
    if (!r) already_set();
    for (int i = 0; i < 5; ++i) {
      PyObject* item = i < 3 || top ? THPVariable_Wrap(std::move(out[i])) : Py_NewRef(Py_None);
      PyTuple_SET_ITEM(r, i, item);
    }
    return r;
  });
}

// token_record(logits, targets, top, lo, index_base) -> [rows, 4 + 2 top]
PyObject* token_record(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("token_record", n, 5);
    const int64_t top = top_of(a[2]);
    const at::Tensor &logits = tensor(a[0], "logits"), &targets = tensor(a[1], "targets");
    const int64_t lo = integer(a[3]), index_base = integer(a[4]);
    return THPVariable_Wrap(unlocked([&] {
      const Logits l(logits, targets, top, lo, true);
      at::Tensor out = at::empty({l.o.n_rows, 4 + 2 * top}, logits.options().dtype(at::kFloat));
      check(rs_token_record_at(&l.o, index_base, l.z.data_ptr(), l.targets->data_ptr(), out.data_ptr<float>(), logits.get_device(), stream_of(logits)));
      return out;
    }));
  });
}

// token_logprobs_grad(logits, targets, lse, entropy, grad_logprob, grad_entropy, grad_lse, lo, sharded, out, first, end): None where
// allowed; first and end are the whole vocabulary's where a shard's caller knows it
PyObject* token_logprobs_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("token_logprobs_grad", n, 12);
    const at::Tensor &logits = tensor(a[0], "logits"), &targets = tensor(a[1], "targets");
    const int64_t lo = integer(a[7]);
    const bool sharded = truth(a[8]), ranged = a[10] != Py_None;
    const int64_t first = ranged ? integer(a[10]) : 0, end = ranged ? integer(a[11]) : 0;
    need_cuda(logits, "logits");
    if (a[5] != Py_None && a[3] == Py_None) value_error("a gradient of the entropy needs the entropy");
    if (a[2] == Py_None || a[4] == Py_None) value_error("lse and grad_logprob are needed");
    static const char* names[5] = {"lse", "entropy", "grad_logprob", "grad_entropy", "grad_lse"};
    const at::Tensor* given[5] = {};
    for (int i = 0; i < 5; ++i)
      if (a[2 + i] != Py_None) given[i] = &tensor(a[2 + i], names[i]);
    const bool has_out = a[9] != Py_None;
    at::Tensor out;
    if (has_out) out = tensor(a[9], "out");
    return THPVariable_Wrap(unlocked([&] {
      const Logits l(logits, targets, 0, lo, sharded);
      c10::MaybeOwned<at::Tensor> rows[5];
      const float* p[5] = {};
      for (int i = 0; i < 5; ++i) {
        if (!given[i]) continue;
        const at::Tensor& t = *given[i];
        if (t.sizes() != targets.sizes() || t.scalar_type() != at::kFloat || t.device() != logits.device())
          value_error(std::string(names[i]) + " must be float32, of targets' shape and on their device");
        rows[i] = t.expect_contiguous();
        p[i] = rows[i]->data_ptr<float>();
      }
      if (!has_out) out = at::empty(logits.sizes(), logits.options());
      if (out.sizes() != logits.sizes() || out.scalar_type() != logits.scalar_type() || out.device() != logits.device())
        value_error("out must have the logits' shape, type and device");
      const at::Tensor o = out.dim() == 2 ? out : out.view({-1, l.o.cols});
      if (o.stride(1) != 1 && l.o.cols > 1) value_error("out must have contiguous rows");
      if (!ranged)
        check(rs_token_logprobs_grad(&l.o, l.z.data_ptr(), l.targets->data_ptr(), p[0], p[1], p[2], p[3], p[4], o.data_ptr(), o.stride(0),
                                     logits.get_device(), stream_of(logits)));
      else
        check(rs_token_logprobs_shard_grad(&l.o, first, end, l.z.data_ptr(), l.targets->data_ptr(), p[0], p[1], p[2], p[3], p[4], o.data_ptr(),
                                           o.stride(0), logits.get_device(), stream_of(logits)));
      if (has_out) written(out);
      return out;
    }));
  });
}

// ---- norm, clipping, AdamW --------------------------------------------------------------------
// The tensors of a list (None entries left out): one CUDA device, contiguous, a type the kernels take.
std::vector<const at::Tensor*> tensors_of(PyObject* list, const char* what) {
  if (!PyList_Check(list)) throw Raise{PyExc_TypeError, std::string(what) + " must be a list"};
  std::vector<const at::Tensor*> r;
  r.reserve(PyList_GET_SIZE(list));
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (o == Py_None) continue;
    const at::Tensor& t = tensor(o, what);
    if (!t.is_cuda()) value_error(std::string(what) + " must be CUDA tensors");
    if (!r.empty() && t.device() != r[0]->device()) value_error(std::string(what) + " must share one device");
    if (!t.is_contiguous()) value_error(std::string(what) + " must be contiguous");
    dtype_code(t, what);
    r.push_back(&t);
  }
  if (r.empty()) value_error(std::string("no ") + what);
  return r;
}
std::vector<rs_grad_span> spans_of(const std::vector<const at::Tensor*>& ts) {
  std::vector<rs_grad_span> s(ts.size());
  for (size_t i = 0; i < ts.size(); ++i)
    s[i] = {(uint64_t)ts[i]->data_ptr(), (uint64_t)ts[i]->numel(), (uint32_t)code_of(*ts[i]), 0};
  return s;
}
at::Tensor sumsq_of(const std::vector<rs_grad_span>& s, const at::Tensor& like) {
  uint64_t bytes = 0;
  check(rs_grad_sumsq_workspace_bytes((int64_t)s.size(), &bytes));
  const at::Tensor workspace = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
  at::Tensor out = at::empty({1}, like.options().dtype(at::kDouble));
  check(rs_grad_sumsq(s.data(), (int64_t)s.size(), workspace.data_ptr(), bytes, out.data_ptr<double>(), like.get_device(), stream_of(like)));
  return out;
}
const double* given_sumsq(const at::Tensor& t, const at::Tensor& with) {
  if (t.scalar_type() != at::kDouble || t.numel() != 1 || t.device() != with.device())
    value_error("sumsq must be one float64 on the gradients' device");
  return t.data_ptr<double>();
}

// grad_sumsq(list): an empty list of parts that a rank counts is allowed with `like`, a tensor on the device
PyObject* grad_sumsq(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("grad_sumsq", n, 2);
    if (a[1] != Py_None && PyList_Check(a[0]) && PyList_GET_SIZE(a[0]) == 0) {
      const at::Tensor& like = tensor(a[1], "gradients");
      need_cuda(like, "gradients");
      return THPVariable_Wrap(unlocked([&] { return sumsq_of({}, like); }));
    }
    const auto ts = tensors_of(a[0], "gradients");
    const auto s = spans_of(ts);
    const at::Tensor& first = *ts[0];
    return THPVariable_Wrap(unlocked([&] { return sumsq_of(s, first); }));
  });
}

// grad_clip(list, max_norm, sumsq or None) -> norm
PyObject* grad_clip(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("grad_clip", n, 3);
    const auto ts = tensors_of(a[0], "gradients");
    const auto s = spans_of(ts);
    const at::Tensor& first = *ts[0];
    const float max_norm = (float)number(a[1]);
    at::Tensor sumsq;
    if (a[2] != Py_None) sumsq = tensor(a[2], "sumsq");
    return THPVariable_Wrap(unlocked([&] {
      if (!sumsq.defined()) sumsq = sumsq_of(s, first);
      at::Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
      check(rs_grad_clip(s.data(), (int64_t)s.size(), given_sumsq(sumsq, first), max_norm, norm.data_ptr<float>(), first.get_device(),
                         stream_of(first)));
      for (const at::Tensor* t : ts) written(*t);
      return norm;
    }));
  });
}

// adamw_step(params, masters, exp_avgs, exp_avg_sqs, steps, decays, grads, lr, beta1, beta2, eps, weight_decay, max_norm or
// None, sumsq or None) -> norm or None. The first seven are lists of one length; a master may be None, an entry whose
// gradient is None is left out, a decay is 1 or 0. The tensors are looked at on every call: nothing is kept of them.
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    count_args("adamw_step", n, 14);
    for (int i = 0; i < 7; ++i)
      if (!PyList_Check(a[i]) || PyList_GET_SIZE(a[i]) != PyList_GET_SIZE(a[0])) throw Raise{PyExc_TypeError, "lists of one length are taken"};
    const auto ts = tensors_of(a[6], "gradients");
    const at::Tensor& first = *ts[0];
    const double decay = number(a[11]);
    std::vector<rs_adamw_tensor> t;
    std::vector<const at::Tensor*> updated;
    t.reserve(ts.size());
    updated.reserve(5 * ts.size());
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[6]); ++i) {
      if (PyList_GET_ITEM(a[6], i) == Py_None) continue;
      const at::Tensor& g = *ts[t.size()];
      auto who = [i] { return "entry " + std::to_string(i) + " of the state: "; };
      auto field = [&](int list, const char* what) -> const at::Tensor& {
        const at::Tensor& x = tensor(PyList_GET_ITEM(a[list], i), what);
        if (x.device() != g.device()) value_error("gradients must be on the state's device");
        if (!x.is_contiguous()) value_error(who() + what + " must be contiguous");
        if (list < 4 && x.sizes() != g.sizes()) assertion_error(who() + what + " and gradient differ in shape");
        return x;
      };
      const at::Tensor &p = field(0, "param"), &m = field(2, "exp_avg"), &v = field(3, "exp_avg_sq"), &step = field(4, "step");
      const at::Tensor* master = PyList_GET_ITEM(a[1], i) != Py_None ? &field(1, "master") : nullptr;
      if (m.scalar_type() != v.scalar_type()) value_error(who() + "moments of two types");
      if (step.scalar_type() != at::kFloat || step.numel() != 1) value_error(who() + "the step must be one float32");
      if (master && master->scalar_type() != at::kFloat) value_error(who() + "the master must be float32");
      rs_adamw_tensor e{};
      e.grad_dev = (uint64_t)g.data_ptr();
      e.param_dev = (uint64_t)p.data_ptr();
      e.master_dev = master ? (uint64_t)master->data_ptr() : 0;
      e.exp_avg_dev = (uint64_t)m.data_ptr();
      e.exp_avg_sq_dev = (uint64_t)v.data_ptr();
      e.step_dev = (uint64_t)step.data_ptr();
      e.numel = (uint64_t)g.numel();
      e.weight_decay = (float)(decay * number(PyList_GET_ITEM(a[5], i)));
      e.grad_dtype = (uint32_t)code_of(g);
      e.param_dtype = dtype_code(p, "param");
      e.moment_dtype = dtype_code(m, "exp_avg");
      t.push_back(e);
      updated.insert(updated.end(), {&p, &m, &v, &step});
      if (master) updated.push_back(master);
    }
    rs_adamw_opts o{number(a[7]), number(a[8]), number(a[9]), number(a[10]), 0.0};
    at::Tensor sumsq, norm;
    const bool clip = a[12] != Py_None;
    if (clip) {
      o.max_norm = number(a[12]);
      if (!(o.max_norm > 0)) value_error("max_norm must be positive");
      if (a[13] != Py_None) {
        sumsq = tensor(a[13], "sumsq");
        given_sumsq(sumsq, first);
      }
    }
    unlocked([&] {
      if (clip) norm = at::empty({}, first.options().dtype(at::kFloat));
      uint64_t bytes = 0;
      check(rs_adamw_workspace_bytes((int64_t)t.size(), &bytes));
      const at::Tensor workspace = at::empty({(int64_t)bytes}, first.options().dtype(at::kByte));
      check(rs_adamw_step(t.data(), (int64_t)t.size(), &o, sumsq.defined() ? sumsq.data_ptr<double>() : nullptr,
                          clip ? norm.data_ptr<float>() : nullptr, workspace.data_ptr(), bytes, first.get_device(), stream_of(first)));
      for (const at::Tensor* x : updated) written(*x);
    });
    return clip ? THPVariable_Wrap(std::move(norm)) : Py_NewRef(Py_None);
  });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(embed_lookup), METHOD(embed_grad), METHOD(token_logprobs), METHOD(token_record), METHOD(token_logprobs_grad),
                         METHOD(grad_sumsq), METHOD(grad_clip), METHOD(adamw_step), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train", "Calls of the training-step operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__train(void) { return PyModule_Create(&module); }
