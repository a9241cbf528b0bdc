// The torch side of the 8-bit KV cache's entry points: argument checks, outputs, scratch and
// streams for ops.py, then one call of the C ABI. In C++ because these calls are made per
// layer and step: the same checks in Python took 15 us a call, more than a decode step's
// kernel at small batches; here they take about 2.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <string>
#include <tuple>

#include "nslg_b200.h"

namespace {

struct Error {
  PyObject* type;
  std::string msg;
};
[[noreturn]] void value_error(const std::string& m) { throw Error{PyExc_ValueError, m}; }
[[noreturn]] void type_error(const std::string& m) { throw Error{PyExc_TypeError, m}; }
[[noreturn]] void runtime_error(const std::string& m) { throw Error{PyExc_RuntimeError, m}; }

PyObject* g_status_ptr = nullptr;     // device index -> address of its status word
PyObject* g_native_error = nullptr;   // (function, code, message) -> exception

// ---------------------------------------------------------------- arguments
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + ": a tensor is needed");
  return THPVariable_Unpack(o);
}

const at::Tensor* optional(PyObject* o, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, name);
}

int integer(PyObject* o, const char* name) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Error{nullptr, ""};
  if (v < INT32_MIN || v > INT32_MAX) value_error(std::string(name) + " is out of range");
  return static_cast<int>(v);
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Error{nullptr, ""};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Error{nullptr, ""};
  return v != 0;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return NSLG_DTYPE_BF16;
    case at::kHalf: return NSLG_DTYPE_F16;
    case at::kFloat: return NSLG_DTYPE_F32;
    default:
      type_error(std::string("nanoslg_b200 kernels support bfloat16, float16 and float32, got ") +
                 c10::toString(t));
  }
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

void* data(const at::Tensor* t) { return t ? const_cast<void*>(t->const_data_ptr()) : nullptr; }
template <typename T>
T* data(const at::Tensor* t) {
  return static_cast<T*>(data(t));
}

// All on one CUDA device; returns its index.
template <typename... Ts>
int one_device(const at::Tensor& first, Ts... rest) {
  for (const at::Tensor* t : {&first, static_cast<const at::Tensor*>(rest)...}) {
    if (t == nullptr) continue;
    if (!t->is_cuda()) runtime_error("nanoslg_b200 kernels need CUDA tensors (no CPU path)");
    if (t->get_device() != first.get_device())
      runtime_error("nanoslg_b200 kernels need CUDA tensors of one device, got cuda:" +
                    std::to_string(first.get_device()) + " and cuda:" +
                    std::to_string(t->get_device()));
  }
  return static_cast<int>(first.get_device());
}

// One layer of the cache and a page list.
struct Cache {
  const at::Tensor *k, *v, *sk, *sv, *indptr, *indices, *lpl;
  int64_t pages;
  int hkv, ps, d, batch;
};

Cache cache_args(PyObject* const* a) {
  Cache c{&tensor(a[0], "pool_k"),     &tensor(a[1], "pool_v"),     &tensor(a[2], "scale_k"),
          &tensor(a[3], "scale_v"),    &tensor(a[4], "kv_indptr"),  &tensor(a[5], "kv_indices"),
          &tensor(a[6], "kv_last_page_len"), 0, 0, 0, 0, 0};
  if (c.k->dim() != 4 || c.k->sizes() != c.v->sizes())
    value_error("kv8 pools must be [num_pages, Hkv, page_size, D], K and V alike");
  c.pages = c.k->size(0);
  for (int i = 1; i < 4; ++i)
    if (c.k->size(i) > INT32_MAX) value_error("kv8 pools: a dimension is out of range");
  c.hkv = static_cast<int>(c.k->size(1));
  c.ps = static_cast<int>(c.k->size(2));
  c.d = static_cast<int>(c.k->size(3));
  for (const at::Tensor* t : {c.k, c.v}) {
    if (t->scalar_type() != at::kFloat8_e4m3fn)
      type_error(std::string("kv8 pools are float8_e4m3fn, got ") + c10::toString(t->scalar_type()));
    if (!t->is_contiguous()) value_error("kv8 pool layers must be contiguous");
  }
  for (const at::Tensor* t : {c.sk, c.sv})
    if (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != c.pages ||
        t->size(1) != c.hkv || !t->is_contiguous())
      value_error("kv8 scales must be contiguous float32 [num_pages, Hkv]");
  for (const at::Tensor* t : {c.indptr, c.indices, c.lpl})
    if (t->scalar_type() != at::kInt || !t->is_contiguous())
      value_error("CSR arrays must be contiguous int32");
  const int64_t batch = c.indptr->numel() - 1;
  if (batch < 0 || batch > INT32_MAX || c.lpl->numel() < batch)
    value_error("kv_indptr needs batch + 1 entries and kv_last_page_len batch");
  c.batch = static_cast<int>(batch);
  return c;
}

// [..., H, D] viewed as rows with one row stride.
struct Rows {
  int64_t n, stride;
  int heads;
};
Rows rows_of(const at::Tensor& x, const char* name, const Cache& c) {
  const int64_t dim = x.dim();
  if (dim < 3 || x.size(dim - 1) != c.d || c.hkv <= 0 || x.size(dim - 2) % c.hkv ||
      x.size(dim - 2) <= 0 || x.size(dim - 2) > INT32_MAX)
    value_error(std::string(name) + ": " + shape_of(x) + " does not go with " +
                std::to_string(c.hkv) + " kv heads of " + std::to_string(c.d));
  Rows r{1, x.size(dim - 1) * x.size(dim - 2), static_cast<int>(x.size(dim - 2))};
  if ((x.stride(dim - 1) != 1 && c.d != 1) || (x.stride(dim - 2) != c.d && r.heads != 1))
    value_error(std::string(name) + ": heads and head_dim must be contiguous");
  // the leading dims must collapse into one row index; size-1 dims carry no stride
  bool first = true;
  int64_t expect = 0;
  for (int64_t i = dim - 3; i >= 0; --i) {
    r.n *= x.size(i);
    if (x.size(i) == 1) continue;
    if (first) {
      r.stride = expect = x.stride(i);
      first = false;
    } else if (x.stride(i) != expect) {
      value_error(std::string(name) + ": leading dims do not form one row stride");
    }
    expect *= x.size(i);
  }
  return r;
}

Rows out_rows(const at::Tensor& out, const at::Tensor& q, const Rows& rq, const Cache& c) {
  const Rows r = rows_of(out, "out", c);
  if (r.n != rq.n || r.heads != rq.heads || out.scalar_type() != q.scalar_type())
    value_error("out must have q's rows, heads, head_dim and dtype");
  return r;
}

void index_args(const at::Tensor& qo_indptr, const at::Tensor* q_row_start, int batch) {
  for (auto [t, n] : {std::pair{&qo_indptr, batch + 1}, std::pair{q_row_start, batch}})
    if (t != nullptr && (t->scalar_type() != at::kInt || !t->is_contiguous() || t->numel() != n))
      value_error("qo_indptr (batch + 1) and q_row_start (batch) must be contiguous int32");
}

// ---------------------------------------------------------------- device state
uint32_t* status_word(int device) {
  static auto* words = new std::map<int, uint32_t*>;      // never freed: outlives the context
  auto it = words->find(device);
  if (it != words->end()) return it->second;
  PyObject* r = PyObject_CallFunction(g_status_ptr, "i", device);
  if (r == nullptr) throw Error{nullptr, ""};
  auto* p = static_cast<uint32_t*>(PyLong_AsVoidPtr(r));
  Py_DECREF(r);
  (*words)[device] = p;
  return p;
}

void check(const char* fn, int rc) {
  if (rc == NSLG_OK) return;
  PyObject* e = PyObject_CallFunction(g_native_error, "sis", fn, rc, nslg_last_error());
  if (e != nullptr) {
    PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(e)), e);
    Py_DECREF(e);
  }
  throw Error{nullptr, ""};
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType t, int device) {
  return at::detail::empty_cuda(shape, t, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)),
                                std::nullopt);
}

// Scratch that starts zeroed and that every call leaves with its counts at zero: one per
// stream (calls on two streams may overlap) and one per graph capture (so may the replays of
// two graphs; its zeroing is captured, once a graph). It is allocated on the stream that uses
// it, so a regrown one is reused only behind its readers.
at::Tensor& workspace(int device, cudaStream_t stream, int64_t bytes) {
  struct Entry {
    uint64_t capture = 0;
    at::Tensor buf;
  };
  static auto* all = new std::map<std::tuple<int, cudaStream_t, bool>, Entry>;
  uint64_t id = 0;
  check("nslg_stream_capture_id", nslg_stream_capture_id(stream, &id));
  Entry& e = (*all)[{device, stream, id != 0}];
  if (!e.buf.defined() || e.capture != id || e.buf.numel() < bytes) {
    e.buf = empty({std::max<int64_t>(bytes, 1 << 20)}, at::kByte, device);
    e.buf.zero_();
    e.capture = id;
  }
  return e.buf;
}

// ---------------------------------------------------------------- the operators
// rope_kv8_append(q, k, v, cos, sin, <cache: 7>, qo_indptr, max_qo_len, q_row_start, q_out, rotate)
PyObject* append(PyObject* const* a) {
  const at::Tensor* q = optional(a[0], "q");
  const at::Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  const Cache c = cache_args(a + 5);
  const at::Tensor& qo = tensor(a[12], "qo_indptr");
  const int most = integer(a[13], "max_qo_len");
  const at::Tensor* start = optional(a[14], "q_row_start");
  const at::Tensor* given = optional(a[15], "q_out");
  const bool rotate = truth(a[16]);
  const int dt = dtype_code(k.scalar_type());
  index_args(qo, start, c.batch);
  const Rows rk = rows_of(k, "k", c), rv = rows_of(v, "v", c);
  if (rk.n != rv.n || k.scalar_type() != v.scalar_type() || rk.heads != c.hkv || rv.heads != c.hkv)
    value_error("k and v must have the same rows and type and the cache's kv heads");
  Rows rq{rk.n, 0, c.hkv};
  if (q != nullptr) {
    rq = rows_of(*q, "q", c);
    if (rq.n != rk.n || q->scalar_type() != k.scalar_type())
      value_error("q must match k in row count and dtype");
    if (given != nullptr && (given->scalar_type() != q->scalar_type() || !given->is_contiguous() ||
                             given->numel() != rq.n * rq.heads * c.d))
      value_error("q_out must be contiguous [rows, Hq, D] of q's dtype");
  } else if (given != nullptr) {
    value_error("q_out given without q");
  }
  const at::Tensor *cos = nullptr, *sin = nullptr;
  int64_t table = 0;
  if (rotate) {
    cos = optional(a[3], "cos");
    sin = optional(a[4], "sin");
    for (const at::Tensor* t : {cos, sin})
      if (t == nullptr || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() != 2 ||
          t->size(1) != c.d)
        value_error("cos/sin tables must be contiguous float32 [rows, D]");
    table = std::min(cos->size(0), sin->size(0));
  }
  const int dev = one_device(k, &v, q, given, cos, sin, c.k, c.v, c.sk, c.sv, c.indptr, c.indices,
                             c.lpl, &qo, start);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out;
  if (q != nullptr) out = given ? *given : empty({rq.n, rq.heads, c.d}, q->scalar_type(), dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev));
  if (rk.n > 0)
    check("nslg_rope_kv8_append",
          nslg_rope_kv8_append(
              dt, c.batch, rq.heads, c.hkv, c.d, c.ps, data(q), rq.stride, data(&k), rk.stride,
              data(&v), rv.stride, rk.n, q != nullptr ? out.mutable_data_ptr() : nullptr,
              data<float>(cos), data<float>(sin), table, data(c.k), data(c.v), data<float>(c.sk),
              data<float>(c.sv), c.pages, data<int32_t>(&qo), data<int32_t>(start), most,
              data<int32_t>(c.indptr), data<int32_t>(c.indices), data<int32_t>(c.lpl),
              status_word(dev), stream));
  if (q == nullptr) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// kv8_gather(<cache: 7>, dtype, out_k, out_v)
PyObject* gather(PyObject* const* a) {
  const Cache c = cache_args(a);
  if (!THPDtype_Check(a[7])) type_error("kv8_gather: dtype must be a torch dtype");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
  const int dt = dtype_code(t);
  const int64_t n = c.indices->numel();
  const at::Tensor* given[2] = {optional(a[8], "out"), optional(a[9], "out")};
  for (const at::Tensor* o : given)
    if (o != nullptr && (o->scalar_type() != t || !o->is_contiguous() || o->dim() != 4 ||
                         o->size(0) != n || o->size(1) != c.ps || o->size(2) != c.hkv ||
                         o->size(3) != c.d))
      value_error("kv8_gather: the outputs must be contiguous [listed pages, page_size, Hkv, D] "
                  "of dtype");
  const int dev = one_device(*c.k, c.v, c.sk, c.sv, c.indptr, c.indices, c.lpl, given[0], given[1]);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out[2];
  for (int i = 0; i < 2; ++i) out[i] = given[i] ? *given[i] : empty({n, c.ps, c.hkv, c.d}, t, dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev));
  check("nslg_kv8_gather",
        nslg_kv8_gather(dt, c.batch, c.hkv, c.d, c.ps, data(c.k), data(c.v), data<float>(c.sk),
                        data<float>(c.sv), c.pages, data<int32_t>(c.indptr),
                        data<int32_t>(c.indices), data<int32_t>(c.lpl), n,
                        out[0].mutable_data_ptr(), out[1].mutable_data_ptr(), status_word(dev),
                        stream));
  PyObject* k = THPVariable_Wrap(out[0]);
  PyObject* v = THPVariable_Wrap(out[1]);
  PyObject* r = k != nullptr && v != nullptr ? PyTuple_Pack(2, k, v) : nullptr;
  Py_XDECREF(k);
  Py_XDECREF(v);
  return r;
}

// paged_decode_kv8(q, <cache: 7>, sm_scale, out)
PyObject* decode(PyObject* const* a) {
  const at::Tensor& q = tensor(a[0], "q");
  const Cache c = cache_args(a + 1);
  const double sm = real(a[8]);
  const at::Tensor* given = optional(a[9], "out");
  const int dt = dtype_code(q.scalar_type());
  const Rows rq = rows_of(q, "q", c);
  if (rq.n != c.batch)
    value_error("paged_decode_kv8: " + std::to_string(rq.n) + " queries for " +
                std::to_string(c.batch) + " sequences");
  Rows ro{rq.n, static_cast<int64_t>(rq.heads) * c.d, rq.heads};
  if (given != nullptr) ro = out_rows(*given, q, rq, c);
  const int dev = one_device(q, given, c.k, c.v, c.sk, c.sv, c.indptr, c.indices, c.lpl);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out = given ? *given : empty({rq.n, rq.heads, c.d}, q.scalar_type(), dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev));
  at::Tensor& ws = workspace(dev, stream,
                             nslg_decode_kv8_workspace_bytes(c.batch, rq.heads, c.hkv, c.d));
  check("nslg_paged_decode_kv8",
        nslg_paged_decode_kv8(dt, c.batch, rq.heads, c.hkv, c.d, c.ps, data(&q), rq.stride,
                              out.mutable_data_ptr(), ro.stride, data(c.k), data(c.v),
                              data<float>(c.sk), data<float>(c.sv), c.pages,
                              data<int32_t>(c.indptr), data<int32_t>(c.indices),
                              data<int32_t>(c.lpl), static_cast<float>(sm), ws.mutable_data_ptr(),
                              ws.numel(), status_word(dev), stream));
  return THPVariable_Wrap(out);
}

// paged_prefill_kv8(q, qo_indptr, max_qo_len, <cache: 7>, sm_scale, causal, q_row_start, out)
PyObject* prefill(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &qo = tensor(a[1], "qo_indptr");
  const int most = integer(a[2], "max_qo_len");
  const Cache c = cache_args(a + 3);
  const double sm = real(a[10]);
  const bool causal = truth(a[11]);
  const at::Tensor *start = optional(a[12], "q_row_start"), *given = optional(a[13], "out");
  const int dt = dtype_code(q.scalar_type());
  index_args(qo, start, c.batch);
  const Rows rq = rows_of(q, "q", c);
  Rows ro{rq.n, static_cast<int64_t>(rq.heads) * c.d, rq.heads};
  if (given != nullptr) ro = out_rows(*given, q, rq, c);
  const int dev = one_device(q, given, &qo, start, c.k, c.v, c.sk, c.sv, c.indptr, c.indices, c.lpl);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out = given ? *given : empty(q.sizes(), q.scalar_type(), dev);
  if (given == nullptr && start != nullptr) out.zero_();
  if (rq.n > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev));
    at::Tensor& ws = workspace(
        dev, stream, nslg_prefill_kv8_workspace_bytes(rq.heads, c.hkv, c.d, std::max(most, 0)));
    check("nslg_paged_prefill_kv8",
          nslg_paged_prefill_kv8(dt, c.batch, rq.heads, c.hkv, c.d, c.ps, data(&q), rq.stride, rq.n,
                                 out.mutable_data_ptr(), ro.stride, data<int32_t>(&qo),
                                 data<int32_t>(start), most, data(c.k), data(c.v),
                                 data<float>(c.sk), data<float>(c.sv), c.pages,
                                 data<int32_t>(c.indptr), data<int32_t>(c.indices),
                                 data<int32_t>(c.lpl), static_cast<float>(sm), causal ? 1 : 0,
                                 ws.mutable_data_ptr(), ws.numel(), status_word(dev), stream));
  }
  return THPVariable_Wrap(out);
}

template <PyObject* (*F)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "%d arguments are needed, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Error& e) {
    if (e.type != nullptr) PyErr_SetString(e.type, e.msg.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "8-bit KV cache: unknown C++ exception");
  }
  return nullptr;
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "setup(status_ptr, native_error)");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  g_status_ptr = args[0];
  g_native_error = args[1];
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef g_methods[] = {
    {"setup", fast(&setup), METH_FASTCALL, nullptr},
    {"append", fast(&entry<append, 17>), METH_FASTCALL, nullptr},
    {"gather", fast(&entry<gather, 10>), METH_FASTCALL, nullptr},
    {"decode", fast(&entry<decode, 10>), METH_FASTCALL, nullptr},
    {"prefill", fast(&entry<prefill, 14>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv8", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8() { return PyModule_Create(&g_module); }
