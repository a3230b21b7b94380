// The serving calls (kvcache, speculative) between torch tensors and the C ABI.
//
// These calls are made once per decoded token, and at small batches the time of
// a call is the host's: their checks, two to three allocations and one
// foreign-function call of up to 20 arguments took 14 to 19 us in Python, the
// kernels 5 to 10.  Here the same checks read the tensors directly.
//
// Every function takes positional arguments (the modules kvcache and
// speculative hold the signatures and their documentation) and raises
// ValueError, NotImplementedError or TallaxError as _lib.check does.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <sstream>
#include <stdexcept>

#include "tallax_hip.h"

namespace {

PyObject* g_error = nullptr;          // _lib.TallaxError
PyObject* g_out_of_memory = nullptr;  // torch.OutOfMemoryError
PyObject* g_workspace = nullptr;      // _lib.workspace_arg
PyObject* g_per_row = nullptr;        // sampling._per_row, of float32

struct ValueError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Unsupported : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python error is already set

template <class... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}

std::string shape_text(at::IntArrayRef d) {
  std::ostringstream s;
  s << "(";
  for (size_t i = 0; i < d.size(); ++i) s << (i ? ", " : "") << d[i];
  s << ")";
  return s.str();
}

// A function body with its C++ exceptions turned into Python ones.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Raised&) {
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Unsupported& e) {
    PyErr_SetString(PyExc_NotImplementedError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_out_of_memory, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void check(int status, const char* what) {
  if (status == 0) return;
  const std::string m = text(what, ": ", tallax_last_error());
  if (status == 2) throw Unsupported(m);
  if (status == 1 || status == 4) throw ValueError(m);
  PyErr_SetString(g_error, text(m, " (status ", status, ")").c_str());
  throw Raised();
}

// A tensor on the card, on the same device as the others of the call.
struct Operands {
  c10::Device device{c10::DeviceType::CPU};
  bool any = false;

  const at::Tensor& need(PyObject* o) {
    if (!THPVariable_Check(o))
      throw ValueError("tallax_amd operands must be torch tensors on a ROCm (cuda) device");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) throw ValueError("tallax_amd operands must be torch tensors on a ROCm (cuda) device");
    if (t.layout() != at::kStrided) throw ValueError("tallax_amd operands must be dense tensors");
    if (any && t.device() != device)
      throw ValueError(text("operands on different devices: ", device, " and ", t.device()));
    device = t.device();
    any = true;
    return t;
  }
  const at::Tensor* may(PyObject* o) { return o == Py_None ? nullptr : &need(o); }
};

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TALLAX_F32;
    case at::kBFloat16: return TALLAX_BF16;
    case at::kInt: return TALLAX_I32;
    default: throw Unsupported(text("dtype ", t.scalar_type(), " is not supported (float32, bfloat16, int32)"));
  }
}

void int_rows(const char* name, const at::Tensor& t, int64_t batch) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != batch || !t.is_contiguous())
    throw ValueError(text(name, " must be a contiguous int32 tensor of shape (", batch, ",)"));
}

template <class T>
T* data(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

struct Cache {
  tallax_kv_cache c;
  at::ScalarType dtype;

  Cache(Operands& on, PyObject* k_o, PyObject* v_o, PyObject* table_o, PyObject* lens_o) {
    const at::Tensor &k = on.need(k_o), &v = on.need(v_o), &table = on.need(table_o), &lens = on.need(lens_o);
    if (k.dim() != 4 || v.sizes() != k.sizes())
      throw ValueError(text("k_pages and v_pages must be 4D [pages, kv_heads, page_size, dim] of one shape, got ",
                            shape_text(k.sizes()), " and ", shape_text(v.sizes())));
    dtype = k.scalar_type();
    if (v.scalar_type() != dtype)
      throw ValueError(text("k_pages ", dtype, " and v_pages ", v.scalar_type(), " must have one dtype"));
    c.dtype = dtype_code(k);
    if (c.dtype == TALLAX_I32) throw Unsupported("a cache holds bfloat16 or float32");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || !table.is_contiguous())
      throw ValueError("block_table must be a contiguous int32 [batch, table_width] tensor");
    c.batch = table.size(0);
    c.table_width = table.size(1);
    int_rows("lens", lens, c.batch);
    c.pages = k.size(0);
    c.kv_heads = k.size(1);
    c.page_size = k.size(2);
    if (k.size(3) > INT32_MAX) throw Unsupported("a cache's dim is at most 256");
    c.dim = static_cast<int32_t>(k.size(3));
    if (c.dim > 1 && (k.stride(3) != 1 || v.stride(3) != 1))
      throw ValueError("the dim elements of a slot must be contiguous");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.k_stride_page = k.stride(0);
    c.k_stride_head = k.stride(1);
    c.k_stride_slot = k.stride(2);
    c.v_stride_page = v.stride(0);
    c.v_stride_head = v.stride(1);
    c.v_stride_slot = v.stride(2);
    c.block_table = static_cast<const int32_t*>(table.data_ptr());
  }

  int64_t capacity() const { return c.table_width * c.page_size; }

  void per_slot(const char* name, const at::Tensor& t, at::ScalarType type) const {
    if (t.scalar_type() != type || t.dim() != 3 || t.size(0) != c.batch || t.size(1) != c.kv_heads ||
        t.size(2) != capacity() || !t.is_contiguous())
      throw ValueError(text(name, " must be a contiguous ", type, " tensor of shape (", c.batch, ", ", c.kv_heads,
                            ", ", capacity(), ")"));
  }
};

bool on_16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

at::Tensor dense_16(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return on_16(c) ? c : c.clone();
}

tallax_stream_t stream_of(const c10::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

struct Held {  // a new reference, dropped at the end
  PyObject* o;
  explicit Held(PyObject* p) : o(p) {
    if (!p) throw Raised();
  }
  ~Held() { Py_DECREF(o); }
  Held(const Held&) = delete;
};

// The caller's workspace, or the device's shared one (_lib.workspace_arg).
struct Workspace {
  void* at = nullptr;
  size_t bytes = 0;
  PyObject* held = nullptr;
  Workspace(PyObject* arg, const c10::Device& device, size_t need) {
    if (need == 0) return;
    Held dev(THPDevice_New(device)), n(PyLong_FromSize_t(need));
    held = PyObject_CallFunctionObjArgs(g_workspace, arg, dev.o, n.o, nullptr);
    if (!held) throw Raised();
    const at::Tensor& t = THPVariable_Unpack(held);
    at = t.data_ptr();
    bytes = static_cast<size_t>(t.numel());
  }
  ~Workspace() { Py_XDECREF(held); }
  Workspace(const Workspace&) = delete;
};

PyObject* tuple_of(std::initializer_list<PyObject*> items) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  bool ok = r != nullptr;
  for (PyObject* o : items) {
    ok = ok && o;
    if (r) PyTuple_SET_ITEM(r, i++, o);
    else Py_XDECREF(o);
  }
  if (!ok) {
    Py_XDECREF(r);
    return nullptr;
  }
  return r;
}

void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw ValueError(text("expected ", want, " arguments, got ", got));
}

// k_pages, v_pages, block_table, lens, k_new, v_new, counts, scores, positions, seen
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 10);
    Operands on;
    const Cache c(on, a[0], a[1], a[2], a[3]);
    const at::Tensor &lens = on.need(a[3]), &k_new = on.need(a[4]), &v_new = on.need(a[5]);
    if (k_new.dim() != 4 || k_new.sizes() != v_new.sizes() || k_new.size(0) != c.c.batch ||
        k_new.size(2) != c.c.kv_heads || k_new.size(3) != c.c.dim)
      throw ValueError(text("k_new and v_new must be [", c.c.batch, ", tokens, ", c.c.kv_heads, ", ", c.c.dim,
                            "], got ", shape_text(k_new.sizes()), " and ", shape_text(v_new.sizes())));
    if (k_new.scalar_type() != c.dtype || v_new.scalar_type() != c.dtype)
      throw ValueError(text("k_new and v_new must be ", c.dtype, ", as the cache"));
    if ((a[7] == Py_None) != (a[8] == Py_None) || (a[7] != Py_None && a[9] == Py_None))
      throw ValueError("scores, positions and seen go together");
    const at::Tensor *counts = on.may(a[6]), *scores = on.may(a[7]), *positions = on.may(a[8]), *seen = nullptr;
    if (scores) {
      seen = &on.need(a[9]);
      c.per_slot("scores", *scores, at::kFloat);
      c.per_slot("positions", *positions, at::kInt);
      int_rows("seen", *seen, c.c.batch);
    }
    if (counts) int_rows("counts", *counts, c.c.batch);
    const c10::DeviceGuard guard(on.device);
    const at::Tensor k = dense_16(k_new), v = dense_16(v_new);
    at::Tensor out = at::empty_like(lens);
    check(tallax_kv_append(&c.c, data<int32_t>(&lens), data<int32_t>(counts), k.data_ptr(), v.data_ptr(), k.size(1),
                           data<float>(scores), data<int32_t>(positions), data<int32_t>(seen), data<int32_t>(&out),
                           stream_of(on.device)),
          "kvcache.append");
    return THPVariable_Wrap(std::move(out));
  });
}

// q, k_pages, v_pages, block_table, lens, scale, counts, scores, out_scores, max_len, workspace
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 11);
    Operands on;
    const Cache c(on, a[1], a[2], a[3], a[4]);
    const at::Tensor &lens = on.need(a[4]), &q_in = on.need(a[0]);
    if (q_in.dim() != 4 || q_in.size(0) != c.c.batch || q_in.size(3) != c.c.dim)
      throw ValueError(text("q must be [", c.c.batch, ", queries, heads, ", c.c.dim, "], got ",
                            shape_text(q_in.sizes())));
    if (q_in.scalar_type() != c.dtype)
      throw ValueError(text("q must be ", c.dtype, ", as the cache, got ", q_in.scalar_type()));
    const int64_t queries = q_in.size(1), heads = q_in.size(2);
    const at::Tensor *counts = on.may(a[6]), *scores = on.may(a[7]), *into = on.may(a[8]);
    if (counts) int_rows("counts", *counts, c.c.batch);
    if (scores) c.per_slot("scores", *scores, at::kFloat);
    if (into) {
      if (!scores) throw ValueError("out_scores without scores");
      c.per_slot("out_scores", *into, at::kFloat);
    }
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt(static_cast<double>(c.c.dim)) : real(a[5]);
    const int64_t max_len = a[9] == Py_None ? c.capacity() : integer(a[9]);
    const int64_t es = q_in.element_size();
    const bool fits = q_in.stride(3) == 1 && on_16(q_in) && q_in.stride(0) * es % 16 == 0 &&
                      q_in.stride(1) * es % 16 == 0 && q_in.stride(2) * es % 16 == 0;
    const c10::DeviceGuard guard(on.device);
    at::Tensor copy;
    if (!fits) copy = q_in.clone(at::MemoryFormat::Contiguous);
    const at::Tensor& q = fits ? q_in : copy;
    at::Tensor out = at::empty({c.c.batch, queries, heads, c.c.dim}, q.options());
    at::Tensor lse = at::empty({c.c.batch, queries, heads}, lens.options().dtype(at::kFloat));
    at::Tensor fresh;
    if (scores && !into) {
      fresh = at::empty_like(*scores);
      into = &fresh;
    }
    const size_t need = tallax_kv_decode_workspace_size(&c.c, queries, heads, max_len, scores != nullptr);
    const Workspace ws(a[10], on.device, need);
    check(tallax_kv_decode(&c.c, q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), queries, heads, scale,
                           data<int32_t>(&lens), data<int32_t>(counts), max_len, data<float>(scores), out.data_ptr(),
                           data<float>(&lse), data<float>(into), ws.at, ws.bytes, stream_of(on.device)),
          "kvcache.decode");
    PyObject *po = THPVariable_Wrap(std::move(out)), *pl = THPVariable_Wrap(std::move(lse));
    if (!scores) return tuple_of({po, pl});
    PyObject* ps = a[8];
    if (ps == Py_None)
      ps = THPVariable_Wrap(std::move(fresh));
    else
      Py_INCREF(ps);
    return tuple_of({po, pl, ps});
  });
}

// k_pages, v_pages, block_table, lens, scores, positions, seen, budget, recent, sinks, workspace
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 11);
    Operands on;
    const Cache c(on, a[0], a[1], a[2], a[3]);
    const at::Tensor &lens = on.need(a[3]), &scores = on.need(a[4]), &positions = on.need(a[5]), &seen = on.need(a[6]);
    c.per_slot("scores", scores, at::kFloat);
    c.per_slot("positions", positions, at::kInt);
    int_rows("seen", seen, c.c.batch);
    const int64_t budget = integer(a[7]), recent = integer(a[8]), sinks = integer(a[9]);
    const c10::DeviceGuard guard(on.device);
    at::Tensor new_lens = at::empty_like(lens), new_scores = at::empty_like(scores),
               new_positions = at::empty_like(positions);
    const size_t need = tallax_kv_evict_workspace_size(&c.c, budget);
    const Workspace ws(a[10], on.device, need);
    check(tallax_kv_evict(&c.c, data<int32_t>(&lens), data<float>(&scores), data<int32_t>(&positions),
                          data<int32_t>(&seen), budget, recent, sinks, data<int32_t>(&new_lens),
                          data<float>(&new_scores), data<int32_t>(&new_positions), ws.at, ws.bytes,
                          stream_of(on.device)),
          "kvcache.evict");
    PyObject *p0 = THPVariable_Wrap(std::move(new_lens)), *p1 = THPVariable_Wrap(std::move(new_scores)),
             *p2 = THPVariable_Wrap(std::move(new_positions));
    return tuple_of({p0, p1, p2});
  });
}

void shaped(const char* name, const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
  if (t.sizes() != shape || t.scalar_type() != type)
    throw ValueError(text(name, " must be a ", type, " tensor of shape ", shape_text(shape), ", got ",
                          t.scalar_type(), " ", shape_text(t.sizes())));
}

// draft_tokens, target_logits, uniforms, noise, draft_probs, temperature, counts, workspace
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 8);
    Operands on;
    const at::Tensor &logits_in = on.need(a[1]), &draft_in = on.need(a[0]), &uniforms_in = on.need(a[2]),
                     &noise_in = on.need(a[3]);
    if (logits_in.dim() != 3 || logits_in.size(1) < 1 || logits_in.size(2) < 1)
      throw ValueError(text("target_logits must be [batch, drafted + 1, vocab], got ", shape_text(logits_in.sizes())));
    const int64_t batch = logits_in.size(0), drafted = logits_in.size(1) - 1, vocab = logits_in.size(2);
    shaped("draft_tokens", draft_in, {batch, drafted}, at::kInt);
    shaped("uniforms", uniforms_in, {batch, drafted}, at::kFloat);
    shaped("noise", noise_in, {batch, vocab}, at::kFloat);
    const int dt = dtype_code(logits_in);
    if (dt == TALLAX_I32) throw Unsupported("verify needs float logits");
    const at::Tensor *probs_in = on.may(a[4]), *counts_in = on.may(a[6]);
    int qdt = TALLAX_F32;
    if (probs_in) {
      if (probs_in->sizes() != at::IntArrayRef({batch, drafted, vocab}))
        throw ValueError(text("draft_probs must be of shape ", shape_text({batch, drafted, vocab}), ", got ",
                              shape_text(probs_in->sizes())));
      qdt = dtype_code(*probs_in);
      if (qdt == TALLAX_I32) throw Unsupported("verify needs float draft probabilities");
    }
    if (counts_in && (counts_in->scalar_type() != at::kInt || counts_in->dim() != 1 || counts_in->size(0) != batch))
      throw ValueError(text("counts must be an int32 tensor of shape (", batch, ",)"));
    const c10::DeviceGuard guard(on.device);
    at::Tensor temperature;
    if (THPVariable_Check(a[5])) {  // what a serving loop passes: its own tensor, used as it is
      const at::Tensor& t = THPVariable_Unpack(a[5]);
      if (t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == batch && t.device() == on.device)
        temperature = t.contiguous();
    }
    if (!temperature.defined()) {
      Held rows(PyLong_FromLongLong(batch)), dev(THPDevice_New(on.device));
      Held t(PyObject_CallFunctionObjArgs(g_per_row, a[5], rows.o, dev.o, nullptr));
      temperature = THPVariable_Unpack(t.o);
    }
    const at::Tensor logits = logits_in.contiguous(), draft = draft_in.contiguous(),
                     uniforms = uniforms_in.contiguous(), noise = noise_in.contiguous();
    const at::Tensor probs = probs_in ? probs_in->contiguous() : at::Tensor(),
                     counts = counts_in ? counts_in->contiguous() : at::Tensor();
    at::Tensor tokens = at::empty({batch, drafted + 1}, draft.options()), accepted = at::empty({batch}, draft.options());
    const size_t need = tallax_verify_workspace_size(batch, drafted, vocab, dt);
    const Workspace ws(a[7], on.device, need);
    check(tallax_verify(data<int32_t>(&draft), logits.data_ptr(), dt, batch, drafted, vocab,
                        counts_in ? data<int32_t>(&counts) : nullptr, data<float>(&temperature),
                        probs_in ? probs.data_ptr() : nullptr, qdt, data<float>(&uniforms), data<float>(&noise),
                        data<int32_t>(&tokens), data<int32_t>(&accepted), ws.at, ws.bytes, stream_of(on.device)),
          "speculative.verify");
    PyObject *p0 = THPVariable_Wrap(std::move(tokens)), *p1 = THPVariable_Wrap(std::move(accepted));
    return tuple_of({p0, p1});
  });
}

// The error classes and what is called back: the workspace's and the per-row parameter's functions.
PyObject* setup(PyObject*, PyObject* args) {
  PyObject** const to[4] = {&g_error, &g_out_of_memory, &g_workspace, &g_per_row};
  PyObject* o[4];
  if (!PyArg_ParseTuple(args, "OOOO", &o[0], &o[1], &o[2], &o[3])) return nullptr;
  for (int i = 0; i < 4; ++i) {
    Py_INCREF(o[i]);
    Py_XDECREF(*to[i]);
    *to[i] = o[i];
  }
  Py_RETURN_NONE;
}

template <class F>
PyCFunction method(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"append", method(append), METH_FASTCALL, nullptr},
                         {"decode", method(decode), METH_FASTCALL, nullptr},
                         {"evict", method(evict), METH_FASTCALL, nullptr},
                         {"verify", method(verify), METH_FASTCALL, nullptr},
                         {"setup", setup, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "serving_ext", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_serving_ext(void) { return PyModule_Create(&module); }
