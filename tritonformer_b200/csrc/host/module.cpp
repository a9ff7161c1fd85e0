// Python binding of the native host path: plain CPython calls on positional arguments, the interpreter lock released
// while kernels are enqueued (the backward pass runs on another thread).
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "functions.h"

namespace {

using namespace tfb_host;

// Positional arguments of one call; None stands for an absent tensor.
class Args {
 public:
  Args(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, const char* name) : a_(a) {
    if (n != want) throw ArgumentError(std::string(name) + ": wrong number of arguments");
  }
  const Tensor& tensor() {
    PyObject* o = a_[i_++];
    if (o == Py_None) return none_;
    if (!THPVariable_Check(o)) throw ArgumentError("expected a tensor");
    return THPVariable_Unpack(o);
  }
  int64_t integer() {
    const long long v = PyLong_AsLongLong(a_[i_++]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  double real() {
    const double v = PyFloat_AsDouble(a_[i_++]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  bool truth() {
    const int v = PyObject_IsTrue(a_[i_++]);
    if (v < 0) throw python_error();
    return v != 0;
  }
 private:
  PyObject* const* a_;
  Py_ssize_t i_ = 0;
  Tensor none_;
};

template <typename F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  return body();
  END_HANDLE_TH_ERRORS
}

template <typename F>
PyObject* tensor_result(F body) {
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = body();
  }
  return THPVariable_Wrap(out);
}

#define TFB_PY(name) PyObject* name(PyObject* self, PyObject* const* argv, Py_ssize_t argc)

PyObject* g_recorder = nullptr;  // what an operator's call goes to while torch.jit.trace records (_trace.py)

// An operator: the call itself, or while a trace is being recorded recorder(operator, *arguments).
template <typename F>
PyObject* traceable(PyObject* self, const char* name, PyObject* const* argv, Py_ssize_t argc, F body) {
  if (C10_LIKELY(!torch::jit::tracer::isTracing() || !g_recorder)) return guarded(body);
  PyObject* args = PyTuple_New(argc + 1);
  if (!args) return nullptr;
  PyObject* op = PyObject_GetAttrString(self, name);
  PyObject* out = nullptr;
  if (op) {
    PyTuple_SET_ITEM(args, 0, op);
    for (Py_ssize_t i = 0; i < argc; ++i) {
      Py_INCREF(argv[i]);
      PyTuple_SET_ITEM(args, i + 1, argv[i]);
    }
    out = PyObject_Call(g_recorder, args, nullptr);
  }
  Py_DECREF(args);
  return out;
}

TFB_PY(py_linear) {
  return traceable(self, "linear", argv, argc, [&] {
    Args a(argv, argc, 4, "linear");
    const Tensor &x = a.tensor(), &w = a.tensor(), &b = a.tensor();
    const bool relu = a.truth();
    return tensor_result([&] { return linear(x, w, b, relu); });
  });
}
TFB_PY(py_layernorm) {
  return traceable(self, "layernorm", argv, argc, [&] {
    Args a(argv, argc, 4, "layernorm");
    const Tensor &x = a.tensor(), &w = a.tensor(), &b = a.tensor();
    const double eps = a.real();
    return tensor_result([&] { return layernorm(x, w, b, eps); });
  });
}
TFB_PY(py_attention) {  // q, k, v, slopes, rounded, table, amp
  return traceable(self, "attention", argv, argc, [&] {
    Args a(argv, argc, 7, "attention");
    const Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &slopes = a.tensor();
    const int64_t rounded = a.integer();
    const Tensor& table = a.tensor();
    const bool amp = a.truth();
    return tensor_result([&] { return attention(q, k, v, slopes, rounded, table, amp); });
  });
}
TFB_PY(py_softmax) {
  return traceable(self, "softmax", argv, argc, [&] {
    Args a(argv, argc, 1, "softmax");
    const Tensor& x = a.tensor();
    return tensor_result([&] { return softmax(x); });
  });
}
TFB_PY(py_cross_entropy) {  // logits, labels, fp32 losses
  return traceable(self, "cross_entropy", argv, argc, [&] {
    Args a(argv, argc, 3, "cross_entropy");
    const Tensor &x = a.tensor(), &y = a.tensor();
    const bool f32 = a.truth();
    return tensor_result([&] { return cross_entropy(x, y, f32); });
  });
}
TFB_PY(py_lm_loss) {
  return traceable(self, "lm_loss", argv, argc, [&] {
    Args a(argv, argc, 2, "lm_loss");
    const Tensor &x = a.tensor(), &y = a.tensor();
    return tensor_result([&] { return lm_loss(x, y); });
  });
}
TFB_PY(py_embedding) {
  return traceable(self, "embedding", argv, argc, [&] {
    Args a(argv, argc, 3, "embedding");
    const Tensor &ids = a.tensor(), &tok = a.tensor(), &pos = a.tensor();
    return tensor_result([&] { return embedding(ids, tok, pos); });
  });
}
// x, ln1_w, ln1_b, wq, wk, wv, wo, ln2_w, ln2_b, w1, b1, w2, b2, slopes, rounded, table, heads, eps1, eps2
PyObject* layer_call(PyObject* const* argv, Py_ssize_t argc, Tensor* act) {
  Args a(argv, argc, 19, "layer");
  const Tensor& x = a.tensor();
  LayerWeights w;
  for (Tensor* t : {&w.ln1_w, &w.ln1_b, &w.wq, &w.wk, &w.wv, &w.wo, &w.ln2_w, &w.ln2_b, &w.w1, &w.b1, &w.w2, &w.b2})
    *t = a.tensor();
  Bias bias;
  bias.slopes = a.tensor();
  bias.rounded = (int)a.integer();
  bias.table = a.tensor();
  const int64_t heads = a.integer();
  const double eps1 = a.real(), eps2 = a.real();
  return tensor_result([&] { return layer(x, w, bias, heads, eps1, eps2, act); });
}
TFB_PY(py_layer) {
  return traceable(self, "layer", argv, argc, [&] { return layer_call(argv, argc, nullptr); });
}
TFB_PY(py_layer_and_activations) {  // (output, hidden activations): what the model's tests look at
  return guarded([&]() -> PyObject* {
    Tensor act;
    PyObject* y = layer_call(argv, argc, &act);
    return Py_BuildValue("(NN)", y, THPVariable_Wrap(act));
  });
}
// The operators of the paged cache write into their arguments, which a recorded graph would not show.
void refuse_tracing(const char* name) {
  if (torch::jit::tracer::isTracing()) throw ArgumentError(std::string(name) + " cannot be recorded by torch.jit.trace");
}
// q, k_pages, v_pages, tables, lengths, key, value, slopes, rounded, query_positions, mass, positions, mass_out
TFB_PY(py_paged_attention) {
  return guarded([&]() -> PyObject* {
    refuse_tracing("paged_attention");
    Args a(argv, argc, 13, "paged_attention");
    const Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &tables = a.tensor(), &lengths = a.tensor(), &key = a.tensor(),
                 &value = a.tensor(), &slopes = a.tensor();
    const int64_t rounded = a.integer();
    const Tensor &at = a.tensor(), &mass = a.tensor(), &positions = a.tensor(), &mass_out = a.tensor();
    return tensor_result(
        [&] { return paged_attention(q, k, v, tables, lengths, key, value, slopes, rounded, at, mass, positions, mass_out); });
  });
}
// k_pages, v_pages, tables, lengths, key, value, counts, mass, positions, key_mass, first_positions
TFB_PY(py_cache_append) {
  return guarded([&]() -> PyObject* {
    refuse_tracing("cache_append");
    Args a(argv, argc, 11, "cache_append");
    const Tensor &k = a.tensor(), &v = a.tensor(), &tables = a.tensor(), &lengths = a.tensor(), &key = a.tensor(),
                 &value = a.tensor(), &counts = a.tensor(), &mass = a.tensor(), &positions = a.tensor(), &key_mass = a.tensor(),
                 &first = a.tensor();
    {
      pybind11::gil_scoped_release no_gil;
      cache_append(k, v, tables, lengths, key, value, counts, mass, positions, key_mass, first);
    }
    Py_RETURN_NONE;
  });
}
// q, k_pages, v_pages, scales, tables, lengths, key, value, slopes, rounded
TFB_PY(py_paged_attention_int4) {
  return guarded([&]() -> PyObject* {
    refuse_tracing("paged_attention");
    Args a(argv, argc, 10, "paged_attention");
    const Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &scales = a.tensor(), &tables = a.tensor(), &lengths = a.tensor(),
                 &key = a.tensor(), &value = a.tensor(), &slopes = a.tensor();
    const int64_t rounded = a.integer();
    return tensor_result([&] { return paged_attention_int4(q, k, v, scales, tables, lengths, key, value, slopes, rounded); });
  });
}
// k_pages, v_pages, scales, tables, lengths, key, value, counts, stored -> (key, value), or None
TFB_PY(py_cache_append_int4) {
  return guarded([&]() -> PyObject* {
    refuse_tracing("cache_append");
    Args a(argv, argc, 9, "cache_append");
    const Tensor &k = a.tensor(), &v = a.tensor(), &scales = a.tensor(), &tables = a.tensor(), &lengths = a.tensor(), &key = a.tensor(),
                 &value = a.tensor(), &counts = a.tensor();
    const bool wanted = a.truth();
    Stored got;
    {
      pybind11::gil_scoped_release no_gil;
      got = cache_append_int4(k, v, scales, tables, lengths, key, value, counts, wanted);
    }
    if (!wanted) Py_RETURN_NONE;
    return Py_BuildValue("(NN)", THPVariable_Wrap(got.key), THPVariable_Wrap(got.value));
  });
}
TFB_PY(py_prompt_mass) {  // q, k, lse, counts, slopes, rounded
  return guarded([&]() -> PyObject* {
    refuse_tracing("prompt_mass");
    Args a(argv, argc, 6, "prompt_mass");
    const Tensor &q = a.tensor(), &k = a.tensor(), &lse = a.tensor(), &counts = a.tensor(), &slopes = a.tensor();
    const int64_t rounded = a.integer();
    return tensor_result([&] { return prompt_mass(q, k, lse, counts, slopes, rounded); });
  });
}
// k, v, mass, positions, tables, lengths, next_positions, k_out, v_out, mass_out, positions_out, out_tables, keep, recent
TFB_PY(py_cache_evict) {
  return guarded([&]() -> PyObject* {
    refuse_tracing("cache_evict");
    Args a(argv, argc, 14, "cache_evict");
    const Tensor &k = a.tensor(), &v = a.tensor(), &mass = a.tensor(), &positions = a.tensor(), &tables = a.tensor(),
                 &lengths = a.tensor(), &next = a.tensor(), &k_out = a.tensor(), &v_out = a.tensor(), &mass_out = a.tensor(),
                 &positions_out = a.tensor(), &out_tables = a.tensor();
    const int64_t keep = a.integer(), recent = a.integer();
    return tensor_result([&] {
      return cache_evict(k, v, mass, positions, tables, lengths, next, k_out, v_out, mass_out, positions_out, out_tables, keep, recent);
    });
  });
}
Int4 int4_of(Args& a) {  // codes, scales, rows, columns, group
  Int4 w;
  w.codes = a.tensor();
  w.scales = a.tensor();
  w.in = a.integer();
  w.out = a.integer();
  w.group = a.integer();
  return w;
}
TFB_PY(py_int4_quantize) {  // weight, group -> (codes, scales)
  return guarded([&]() -> PyObject* {
    refuse_tracing("quantize_int4");
    Args a(argv, argc, 2, "quantize_int4");
    const Tensor& w = a.tensor();
    const int64_t group = a.integer();
    Int4 q;
    {
      pybind11::gil_scoped_release no_gil;
      q = int4_quantize(w, group);
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(q.codes), THPVariable_Wrap(q.scales));
  });
}
TFB_PY(py_int4_expand) {  // a packed weight
  return guarded([&]() -> PyObject* {
    refuse_tracing("Int4Weight.dequantize");
    Args a(argv, argc, 5, "Int4Weight.dequantize");
    const Int4 w = int4_of(a);
    return tensor_result([&] { return int4_expand(w); });
  });
}
TFB_PY(py_int4_linear) {  // x, a packed weight, bias, relu, addend
  return guarded([&]() -> PyObject* {
    refuse_tracing("linear_int4");
    Args a(argv, argc, 9, "linear_int4");
    const Tensor& x = a.tensor();
    const Int4 w = int4_of(a);
    const Tensor& bias = a.tensor();
    const bool relu = a.truth();
    const Tensor& addend = a.tensor();
    return tensor_result([&] { return int4_linear(x, w, bias, relu, addend); });
  });
}
TFB_PY(py_sample) {  // logits, uniforms, and of temperature, top_k, top_p, min_p each: one per row or None, one for all
  return guarded([&]() -> PyObject* {
    refuse_tracing("sample_tokens");
    Args a(argv, argc, 10, "sample_tokens");
    const Tensor &logits = a.tensor(), &uniforms = a.tensor();
    Setting s[4];
    for (Setting& x : s) {
      x.each = a.tensor();
      x.all = a.real();
    }
    return tensor_result([&] { return sample(logits, uniforms, s[0], s[1], s[2], s[3]); });
  });
}
TFB_PY(py_set_grad_mode) {  // accumulating, overwrite, defer, fork
  return guarded([&]() -> PyObject* {
    Args a(argv, argc, 4, "set_grad_mode");
    g_mode.accumulating = a.truth();
    g_mode.overwrite = a.truth();
    g_mode.defer = a.truth();
    g_mode.fork = a.truth();
    Py_RETURN_NONE;
  });
}
TFB_PY(py_take_written) {
  return guarded([&]() -> PyObject* {
    const std::vector<uintptr_t> v = take_written();
    PyObject* list = PyList_New((Py_ssize_t)v.size());
    if (!list) throw python_error();
    for (size_t i = 0; i < v.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, PyLong_FromUnsignedLongLong(v[i]));
    return list;
  });
}
TFB_PY(py_join_weight_grads) {
  return guarded([&]() -> PyObject* {
    join_all();
    Py_RETURN_NONE;
  });
}
TFB_PY(py_gemm_workspace) {  // device index, stream handle
  return guarded([&] {
    Args a(argv, argc, 2, "gemm_workspace");
    const int64_t dev = a.integer(), stream = a.integer();
    return tensor_result([&] {
      return gemm_workspace(c10::Device(c10::kCUDA, (c10::DeviceIndex)dev), reinterpret_cast<cudaStream_t>(stream));
    });
  });
}
TFB_PY(py_set_recorder) {
  return guarded([&]() -> PyObject* {
    if (argc != 1) throw ArgumentError("set_recorder: wrong number of arguments");
    Py_INCREF(argv[0]);
    Py_XDECREF(std::exchange(g_recorder, argv[0]));
    Py_RETURN_NONE;
  });
}
TFB_PY(py_reset_workspaces) {
  return guarded([&]() -> PyObject* {
    reset_workspaces();
    Py_RETURN_NONE;
  });
}

#define TFB_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TFB_METHOD(linear), TFB_METHOD(layernorm), TFB_METHOD(attention), TFB_METHOD(softmax),
                         TFB_METHOD(cross_entropy), TFB_METHOD(lm_loss), TFB_METHOD(embedding), TFB_METHOD(layer),
                         TFB_METHOD(layer_and_activations),
                         TFB_METHOD(paged_attention), TFB_METHOD(cache_append), TFB_METHOD(prompt_mass), TFB_METHOD(cache_evict),
                         TFB_METHOD(paged_attention_int4), TFB_METHOD(cache_append_int4), TFB_METHOD(int4_quantize), TFB_METHOD(int4_expand), TFB_METHOD(int4_linear), TFB_METHOD(sample),
                         TFB_METHOD(set_grad_mode), TFB_METHOD(take_written), TFB_METHOD(join_weight_grads),
                         TFB_METHOD(gemm_workspace), TFB_METHOD(reset_workspaces), TFB_METHOD(set_recorder), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native host path of tritonformer_b200.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
