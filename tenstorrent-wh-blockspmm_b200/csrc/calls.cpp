// Python's way into the decoder-attention entries of the C ABI: the operands of
// a call are torch tensors, looked at here (type, device, shape, strides) and
// passed on.
//
// The other entries are called through ctypes from bsp.py.  These are called
// once a layer and token, on tensors of a few kilobytes: looked at from Python
// and passed through ctypes a call cost the host 8.0 us (rotary, 16 tokens) and
// 11.9 us (append, 31 arguments); from here 4.1 us each, most of it the launch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "bsp.h"

namespace {

PyObject* g_error = nullptr;   // bsp.BspError
PyObject* g_device = nullptr;  // bsp.device
PyObject *s_handle, *s_value, *s_ordinal, *s_cuda_stream, *s_address;

struct Refusal {  // becomes BspError(BSP_ERR_INVALID_ARG, what)
  std::string what;
};
struct PyFailed {};  // a Python error is set

[[noreturn]] void refuse(std::string what) { throw Refusal{std::move(what)}; }

struct Ref {  // an owned reference
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {
    if (!p) throw PyFailed{};
  }
  ~Ref() { Py_DECREF(p); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

void set_error(int status, const char* what) {
  PyObject* e = PyObject_CallFunction(g_error, "is", status, what);
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
}

// A handle of bsp.py: a ctypes c_void_p, or None once it is closed.
void* handle_of(PyObject* owner) {
  const Ref h(PyObject_GetAttr(owner, s_handle));
  if (h.p == Py_None) return nullptr;
  const Ref v(PyObject_GetAttr(h.p, s_value));
  if (v.p == Py_None) return nullptr;
  void* p = PyLong_AsVoidPtr(v.p);
  if (!p && PyErr_Occurred()) throw PyFailed{};
  return p;
}

long number(PyObject* owner, PyObject* name) {
  const Ref v(PyObject_GetAttr(owner, name));
  const long n = PyLong_AsLong(v.p);
  if (n == -1 && PyErr_Occurred()) throw PyFailed{};
  return n;
}

// The opened GPU of a call: the caller's, or the one that holds its tensor.
struct OnGpu {
  bsp_device* dev;
  int ordinal;
};
OnGpu gpu_of(PyObject* dev, int holds) {
  if (dev != Py_None) return {static_cast<bsp_device*>(handle_of(dev)), static_cast<int>(number(dev, s_ordinal))};
  const Ref index(PyLong_FromLong(holds));
  const Ref d(PyObject_CallOneArg(g_device, index.p));
  return {static_cast<bsp_device*>(handle_of(d.p)), holds};
}

// The given stream (an object with cuda_stream, or its number), or the current one.
void* stream_of(PyObject* stream, int ordinal) {
  if (stream == Py_None) return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(ordinal)).stream();
  PyObject* n = PyObject_GetAttr(stream, s_cuda_stream);
  if (!n) {
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) throw PyFailed{};
    PyErr_Clear();
    n = PyNumber_Long(stream);
  }
  const Ref v(n);
  void* p = PyLong_AsVoidPtr(v.p);
  if (!p && PyErr_Occurred()) throw PyFailed{};
  return p;
}

std::string shape_text(c10::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

// A CUDA tensor of one type, on GPU `ordinal` unless that is -1.
const at::Tensor& tensor(PyObject* x, const char* name, at::ScalarType type, int ordinal) {
  if (!THPVariable_Check(x)) refuse(std::string(name) + " must be a torch tensor");
  const at::Tensor& t = THPVariable_Unpack(x);
  if (t.scalar_type() != type || !t.is_cuda())
    refuse(std::string(name) + " must be a " + c10::toString(type) + " cuda tensor, not " +
           c10::toString(t.scalar_type()) + " on " + t.device().str());
  if (ordinal >= 0 && t.device().index() != ordinal)
    refuse(std::string(name) + " is on " + t.device().str() + ", not on GPU " + std::to_string(ordinal));
  return t;
}

// A cache: its description (bsp.KvCache keeps it) and the GPU that its tensors are on.
struct Cache {
  const bsp_kv_cache* desc;
  long ordinal;
};
Cache cache_of(PyObject* x) {
  const Ref address(PyObject_GetAttr(x, s_address));
  const auto* desc = static_cast<const bsp_kv_cache*>(PyLong_AsVoidPtr(address.p));
  if (PyErr_Occurred()) throw PyFailed{};
  if (!desc) refuse("null cache");
  return {desc, number(x, s_ordinal)};
}
const bsp_kv_cache* cache_on(const Cache& c, int at) {
  if (c.ordinal != at) refuse("the cache is on cuda:" + std::to_string(c.ordinal) + ", not on GPU " + std::to_string(at));
  return c.desc;
}

// A [tokens, heads, d] operand, d contiguous.  A dimension of one entry is never
// stepped over: its stride counts as 0.
struct Heads {
  void* p = nullptr;
  int64_t token = 0, head = 0;
};
Heads heads_of(PyObject* x, const char* name, int64_t tokens, int64_t heads, int64_t d, int ordinal,
               at::ScalarType type = at::kBFloat16) {
  const at::Tensor& t = tensor(x, name, type, ordinal);
  const auto s = t.sizes();
  if (s.size() != 3 || s[0] != tokens || s[1] != heads || s[2] != d)
    refuse(std::string(name) + " is " + shape_text(s) + ", expected " + shape_text({tokens, heads, d}));
  void* p = t.data_ptr();
  if (t.is_contiguous()) return {p, heads * d, d};
  if (t.stride(2) != 1 && d > 1) refuse(std::string(name) + ": the values of a head must be contiguous");
  return {p, tokens > 1 ? t.stride(0) : 0, heads > 1 ? t.stride(1) : 0};
}

const int32_t* index_of(PyObject* x, const char* name, int64_t n, int ordinal) {
  const at::Tensor& t = tensor(x, name, at::kInt, ordinal);
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous int32 tensor [" + std::to_string(n) + "], not " +
           shape_text(t.sizes()));
  return t.data_ptr<int32_t>();
}

struct Pages {
  const int32_t* p;
  int64_t stride, width;
};
Pages pages_of(PyObject* x, int64_t n, int ordinal) {
  const at::Tensor& t = tensor(x, "pages", at::kInt, ordinal);
  if (t.dim() != 2 || t.size(0) != n)
    refuse("pages must be an int32 tensor [" + std::to_string(n) + ", width], not " + shape_text(t.sizes()));
  const int64_t width = t.size(1);
  if (t.is_contiguous()) return {t.data_ptr<int32_t>(), width, width};
  if (t.stride(1) != 1 && width > 1) refuse("the rows of pages must be contiguous");
  return {t.data_ptr<int32_t>(), n > 1 ? t.stride(0) : 0, width};
}

struct Table {
  const float* p = nullptr;
  int64_t n_pos = 0;
  int32_t rot = 0;
};
Table table_of(PyObject* x, int ordinal) {
  const at::Tensor& t = tensor(x, "a rotary table", at::kFloat, ordinal);
  if (t.dim() != 3 || t.size(2) != 2 || !t.is_contiguous() || t.size(1) > (1 << 20))
    refuse("a rotary table is a contiguous f32 cuda tensor [positions, rot / 2, 2]");
  return {t.data_ptr<float>(), t.size(0), static_cast<int32_t>(2 * t.size(1))};
}

float* lse_of(PyObject* x, int64_t tokens, int64_t heads, int ordinal) {
  if (x == Py_None) return nullptr;
  const at::Tensor& t = tensor(x, "lse", at::kFloat, ordinal);
  if (t.dim() != 2 || t.size(0) != tokens || t.size(1) != heads || !t.is_contiguous())
    refuse("lse must be a contiguous f32 tensor " + shape_text({tokens, heads}) + ", not " + shape_text(t.sizes()));
  return t.data_ptr<float>();
}

const at::Tensor& with_dims(PyObject* x, const char* name, int64_t dims) {
  if (!THPVariable_Check(x)) refuse(std::string(name) + " must be a torch tensor");
  const at::Tensor& t = THPVariable_Unpack(x);
  if (t.dim() != dims) refuse(std::string(name) + " must have " + std::to_string(dims) + " dimensions");
  if (!t.is_cuda()) refuse(std::string(name) + " must be a cuda tensor");
  return t;
}

int32_t int_of(int64_t n, const char* what) {
  if (n < 0 || n > 0x7FFFFFFF) refuse(std::string(what) + " out of range");
  return static_cast<int32_t>(n);
}

// The body of a call: what it throws becomes a Python error, and so does a status.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t expected, F&& body) {
  try {
    if (got != expected) {
      PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", got, expected);
      return nullptr;
    }
    const bsp_status s = body();
    if (s != BSP_OK) {
      set_error(s, bsp_last_error_string());
      return nullptr;
    }
    Py_RETURN_NONE;
  } catch (const Refusal& r) {
    set_error(BSP_ERR_INVALID_ARG, r.what.c_str());
  } catch (const PyFailed&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <typename F>
bsp_status unlocked(F&& call) {  // without the interpreter's lock: a launch waits when the stream's queue is full
  PyThreadState* t = PyEval_SaveThread();
  const bsp_status s = call();
  PyEval_RestoreThread(t);
  return s;
}

// rope(x, positions, table, layout, transpose, out, dev, stream)
PyObject* py_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&] {
    const at::Tensor& x = with_dims(a[0], "x", 3);
    const bool f32 = x.scalar_type() == at::kFloat;
    const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
    const int64_t tokens = x.size(0), heads = x.size(1), d = x.size(2);
    const int at = x.device().index();
    const Heads in = heads_of(a[0], "x", tokens, heads, d, at, type), out = heads_of(a[5], "out", tokens, heads, d, at, type);
    const int32_t* positions = index_of(a[1], "positions", tokens, at);
    const Table t = table_of(a[2], at);
    const long layout = PyLong_AsLong(a[3]), transpose = PyLong_AsLong(a[4]);
    if (PyErr_Occurred()) throw PyFailed{};
    if (tokens == 0 || heads == 0) return BSP_OK;
    const OnGpu gpu = gpu_of(a[6], at);
    if (gpu.ordinal != at) refuse("x is on " + x.device().str() + ", not on GPU " + std::to_string(gpu.ordinal));
    void* stream = stream_of(a[7], at);
    const int32_t h = int_of(heads, "heads"), dd = int_of(d, "d");
    return unlocked([&] {
      return bsp_rope(gpu.dev, in.p, in.token, in.head, positions, t.p, t.n_pos, tokens, h, dd, t.rot,
                      static_cast<bsp_rope_layout>(layout), transpose != 0, f32 ? BSP_F32 : BSP_BF16, out.p, out.token,
                      out.head, stream);
    });
  });
}

// kv_append(cache, k, v, starts, before, pages, table, layout, q, q_out, k_out, dev, stream)
PyObject* py_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&] {
    const Cache held = cache_of(a[0]);
    const at::Tensor& kt = with_dims(a[1], "k", 3);
    const at::Tensor& bt = with_dims(a[4], "before", 1);
    const int64_t tokens = kt.size(0), seqs = bt.size(0);
    const int at = kt.device().index();
    const bsp_kv_cache* cache = cache_on(held, at);
    const int hk = cache->kv_heads, d = cache->d;
    const Heads k = heads_of(a[1], "k", tokens, hk, d, at), v = heads_of(a[2], "v", tokens, hk, d, at);
    const int32_t* starts = index_of(a[3], "starts", seqs + 1, at);
    const int32_t* before = index_of(a[4], "before", seqs, at);
    const Pages pages = pages_of(a[5], seqs, at);
    const Table t = a[6] == Py_None ? Table{} : table_of(a[6], at);
    const long layout = PyLong_AsLong(a[7]);
    if (PyErr_Occurred()) throw PyFailed{};
    Heads q, q_out, k_out;
    int32_t heads = 0;
    if ((a[8] == Py_None) != (a[9] == Py_None)) refuse("q and q_out come together");
    if (a[8] != Py_None) {
      heads = int_of(with_dims(a[8], "q", 3).size(1), "heads");
      q = heads_of(a[8], "q", tokens, heads, d, at);
      q_out = heads_of(a[9], "q_out", tokens, heads, d, at);
    }
    if (a[10] != Py_None) k_out = heads_of(a[10], "k_out", tokens, hk, d, at);
    if (tokens == 0 || seqs == 0) return BSP_OK;
    const OnGpu gpu = gpu_of(a[11], at);
    if (gpu.ordinal != at) refuse("k is on " + kt.device().str() + ", not on GPU " + std::to_string(gpu.ordinal));
    void* stream = stream_of(a[12], at);
    const int32_t ns = int_of(seqs, "sequences");
    return unlocked([&] {
      return bsp_kv_append(gpu.dev, cache, k.p, k.token, k.head, v.p, v.token, v.head, tokens, ns, starts, before,
                           pages.p, pages.stride, pages.width, t.p, t.n_pos, t.rot, static_cast<bsp_rope_layout>(layout),
                           q.p, q.token, q.head, heads, q_out.p, q_out.token, q_out.head, k_out.p, k_out.token,
                           k_out.head, stream);
    });
  });
}

float scale_of(PyObject* scale) {
  const double s = PyFloat_AsDouble(scale);
  if (s == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return static_cast<float>(s);
}

// prompt(plan, ordinal, q, k, v, o, scale, lse, stream)
PyObject* py_prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const auto* plan = static_cast<const bsp_prompt_plan*>(handle_of(a[0]));
    int64_t info[16];
    const bsp_status s = bsp_prompt_plan_info(plan, info);
    if (s != BSP_OK) return s;
    const int at = static_cast<int>(PyLong_AsLong(a[1]));
    if (PyErr_Occurred()) throw PyFailed{};
    const int64_t tokens = info[2], heads = info[4], d = info[6];
    const Heads q = heads_of(a[2], "q", tokens, heads, d, at), k = heads_of(a[3], "k", info[3], info[5], d, at),
                v = heads_of(a[4], "v", info[3], info[5], d, at), o = heads_of(a[5], "o", tokens, heads, d, at);
    const float scale = scale_of(a[6]);
    float* lse = lse_of(a[7], tokens, heads, at);
    void* stream = stream_of(a[8], at);
    return unlocked([&] {
      return bsp_prompt_execute(plan, q.p, q.token, q.head, k.p, k.token, k.head, v.p, v.token, v.head, scale, o.p,
                                o.token, o.head, lse, stream);
    });
  });
}

// decode(plan, ordinal, cache, q, lens, pages, o, scale, lse, stream)
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&] {
    const auto* plan = static_cast<const bsp_decode_plan*>(handle_of(a[0]));
    int64_t info[16];
    const bsp_status s = bsp_decode_plan_info(plan, info);
    if (s != BSP_OK) return s;
    const int at = static_cast<int>(PyLong_AsLong(a[1]));
    if (PyErr_Occurred()) throw PyFailed{};
    const bsp_kv_cache* cache = cache_on(cache_of(a[2]), at);
    const int64_t seqs = with_dims(a[3], "q", 3).size(0), heads = info[2], d = info[4];
    const Heads q = heads_of(a[3], "q", seqs, heads, d, at), o = heads_of(a[6], "o", seqs, heads, d, at);
    const int32_t* lens = index_of(a[4], "lens", seqs, at);
    const Pages pages = pages_of(a[5], seqs, at);
    const float scale = scale_of(a[7]);
    float* lse = lse_of(a[8], seqs, heads, at);
    void* stream = stream_of(a[9], at);
    const int32_t ns = int_of(seqs, "sequences");
    return unlocked([&] {
      return bsp_decode_execute(plan, cache, q.p, q.token, q.head, ns, lens, pages.p, pages.stride, pages.width, scale,
                                o.p, o.token, o.head, lse, stream);
    });
  });
}

// setup(BspError, device)
PyObject* py_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "setup(BspError, device)");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_XSETREF(g_error, a[0]);
  Py_INCREF(a[1]);
  Py_XSETREF(g_device, a[1]);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F* f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef g_methods[] = {
    {"setup", fast(py_setup), METH_FASTCALL, nullptr},         {"rope", fast(py_rope), METH_FASTCALL, nullptr},
    {"kv_append", fast(py_kv_append), METH_FASTCALL, nullptr}, {"prompt", fast(py_prompt), METH_FASTCALL, nullptr},
    {"decode", fast(py_decode), METH_FASTCALL, nullptr},       {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bsp_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bsp_calls() {
  s_handle = PyUnicode_InternFromString("handle");
  s_value = PyUnicode_InternFromString("value");
  s_ordinal = PyUnicode_InternFromString("ordinal");
  s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
  s_address = PyUnicode_InternFromString("address");
  if (!s_handle || !s_value || !s_ordinal || !s_cuda_stream || !s_address) return nullptr;
  return PyModule_Create(&g_module);
}
