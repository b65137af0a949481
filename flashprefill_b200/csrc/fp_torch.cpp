// Tensor plumbing of the paged-cache entry points: checks, strides, workspace and stream, then the C ABI of
// libflashprefill_b200.so (include/flashprefill_b200.h), whose functions are handed over by address at load time.
//
// These calls run once for each layer of each token, and the small ones take 1.5 to 5 us on the GPU; the same plumbing in
// Python through ctypes took 20 to 34 us a call, so it bound every call below 200 MB of cache; this takes 3 to 4.  It is plain CPython
// (vectorcall) over torch's C++ tensors.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <string>

#include "../../include/flashprefill_b200.h"

namespace {

decltype(&fpb_kv_cache_write) g_write;
decltype(&fpb_kv_cache_read) g_read;
decltype(&fpb_paged_decode) g_decode;
decltype(&fpb_paged_decode_workspace_bytes) g_workspace_bytes;
decltype(&fpb_last_error) g_last_error;
PyObject* g_library_error;  // FlashPrefillError

#define REFUSE(cond, E, ...)                                          \
  do {                                                                \
    if (cond) throw E(c10::str(__VA_ARGS__));                         \
  } while (0)

struct Value : std::runtime_error { using std::runtime_error::runtime_error; };
struct Type : std::runtime_error { using std::runtime_error::runtime_error; };
struct Library : std::runtime_error { using std::runtime_error::runtime_error; };

bool given(PyObject* o) { return o != nullptr && o != Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name, int64_t ndim, const at::Device* device) {
  REFUSE(o == nullptr || !THPVariable_Check(o), Type, name, " must be a torch.Tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  REFUSE(t.dim() != ndim, Value, name, " must have ", ndim, " dimensions, got shape ", t.sizes());
  REFUSE(!t.is_cuda(), Value, name, " must be a CUDA tensor (flashprefill_b200 has no CPU path), got ", t.device());
  REFUSE(device && t.device() != *device, Value, name, " is on ", t.device(), ", expected ", *device);
  return t;
}

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return FPB_BF16;
  if (t.scalar_type() == at::kHalf) return FPB_FP16;
  throw Type(c10::str("flashprefill_b200 supports bfloat16 and float16 inputs (got ", t.scalar_type(), ")"));
}

// The kernels address 16-byte pieces of rows of 128 contiguous elements.
bool rows_ok(const at::Tensor& t) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.stride(i) % 8) return false;
  return true;
}

// An input as it is, or a copy where its rows are not aligned.
at::Tensor input(PyObject* o, const char* name, int64_t ndim, const at::Device* device) {
  const at::Tensor& t = tensor(o, name, ndim, device);
  dtype_code(t);
  if (t.numel() == 0 || rows_ok(t)) return t;
  at::NoGradGuard no_grad;
  return t.clone(at::MemoryFormat::Contiguous);
}

// A tensor that a kernel writes must not have two indices for one element through a stride of 0.
void written(const at::Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    REFUSE(t.stride(i) == 0 && t.size(i) > 1, Value, name, " is written to and must not be an expanded tensor (strides ",
           t.strides(), ")");
}

int as_int(int64_t x, const char* what) {
  REFUSE(x > INT32_MAX, Value, what, " (", x, ") is too large");
  return (int)x;
}

struct Cache {
  const at::Tensor *k, *v;
  float *k_scale = nullptr, *v_scale = nullptr;
  const int64_t *strides, *scale_strides = nullptr;
  int dtype, pages, page_size, heads;
};

Cache cache_args(PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso, const at::Tensor& rows, const at::Device& device,
                 int64_t heads, bool write) {
  Cache c;
  const at::Tensor& k = tensor(ko, "k_cache", 4, &device);
  const at::Tensor& v = tensor(vo, "v_cache", 4, &device);
  REFUSE(v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != k.scalar_type(), Value,
         "k_cache and v_cache must share shape, strides and dtype");
  REFUSE(heads >= 0 && k.size(2) != heads, Value, "the cache has ", k.size(2), " KV heads, expected ", heads);
  REFUSE(k.size(3) != 128 || k.stride(3) != 1, Value,
         "the cache's last dimension must be 128 contiguous elements, got shape ", k.sizes(), ", strides ", k.strides());
  if (write) written(k, "k_cache");
  c.k = &k;
  c.v = &v;
  c.strides = k.strides().data();
  c.pages = as_int(k.size(0), "pages");
  c.page_size = as_int(k.size(1), "page_size");
  c.heads = as_int(k.size(2), "KV heads");
  const bool codes = k.scalar_type() == at::kFloat8_e4m3fn;
  REFUSE(!codes && k.scalar_type() != rows.scalar_type(), Type, "the cache must be ", rows.scalar_type(),
         " or torch.float8_e4m3fn, got ", k.scalar_type());
  REFUSE(!codes && (given(kso) || given(vso)), Value, "a 16-bit cache takes no scales");
  REFUSE(codes && !(given(kso) && given(vso)), Value, "an e4m3 cache needs k_scale and v_scale");
  c.dtype = codes ? FPB_E4M3 : dtype_code(k);
  if (codes) {
    const at::Tensor& ks = tensor(kso, "k_scale", 3, &device);
    const at::Tensor& vs = tensor(vso, "v_scale", 3, &device);
    REFUSE(ks.sizes() != k.sizes().slice(0, 3) || vs.sizes() != ks.sizes(), Value, "k_scale and v_scale must have shape ",
           k.sizes().slice(0, 3));
    REFUSE(ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat, Type, "k_scale and v_scale must be float32");
    REFUSE(ks.strides() != vs.strides(), Value, "k_scale and v_scale must share strides");
    if (write) written(ks, "k_scale");
    c.k_scale = ks.data_ptr<float>();
    c.v_scale = vs.data_ptr<float>();
    c.scale_strides = ks.strides().data();
  }
  return c;
}

struct Table {
  const int32_t *pages, *lens;
  int64_t stride;
  int width;
};

Table table_args(PyObject* po, PyObject* lo, int64_t batch, const at::Device& device) {
  const at::Tensor& p = tensor(po, "page_table", 2, &device);
  const at::Tensor& l = tensor(lo, "seq_lens", 1, &device);
  REFUSE(p.scalar_type() != at::kInt || l.scalar_type() != at::kInt, Type, "page_table and seq_lens must be int32");
  REFUSE(p.size(0) != batch || l.size(0) != batch, Value, "page_table ", p.sizes(), " and seq_lens ", l.sizes(), " must have ",
         batch, " rows");
  REFUSE((p.size(1) > 1 && p.stride(1) != 1) || (batch > 1 && l.stride(0) != 1), Value,
         "the last dimension of page_table and of seq_lens must be contiguous");
  return {p.data_ptr<int32_t>(), l.data_ptr<int32_t>(), p.stride(0), as_int(p.size(1), "page_table width")};
}

void check(int rc) {
  if (rc == FPB_OK) return;
  const std::string msg = std::string("flashprefill_b200: ") + g_last_error();
  if (rc == FPB_EINVAL) throw Value(msg);
  throw Library(msg);
}

// Runs f() -> return code on the tensors' device and its current stream, without the interpreter lock.
template <typename F>
void launch(const at::Device& device, F&& f) {
  c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(stream);
  Py_END_ALLOW_THREADS
  check(rc);
}

// kv_cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale)
void write_(PyObject* const* a) {
  const at::Tensor k = input(a[0], "k", 3, nullptr);
  const at::Device device = k.device();
  const at::Tensor v = input(a[1], "v", 3, &device);
  REFUSE(v.sizes() != k.sizes(), Value, "v shape ", v.sizes(), " must equal k shape ", k.sizes());
  REFUSE(v.scalar_type() != k.scalar_type(), Type, "k and v must share one dtype");
  const Cache c = cache_args(a[2], a[3], a[5], a[6], k, device, k.size(1), true);
  REFUSE(c.k->data_ptr() == c.v->data_ptr(), Value, "k_cache and v_cache must not be the same memory");
  REFUSE(c.k_scale && c.k_scale == c.v_scale, Value, "k_scale and v_scale must not be the same memory");
  const at::Tensor& s = tensor(a[4], "slots", 1, &device);
  REFUSE(s.scalar_type() != at::kLong && s.scalar_type() != at::kInt, Type, "slots must be int64 or int32, got ", s.scalar_type());
  REFUSE(s.size(0) != k.size(0), Value, "slots must have one entry for each of the ", k.size(0), " rows, got ", s.size(0));
  const at::Tensor slots = s.contiguous();
  const int tokens = as_int(k.size(0), "rows"), dim = as_int(k.size(2), "head_dim");
  launch(device, [&](void* stream) {
    return g_write(k.data_ptr(), v.data_ptr(), dtype_code(k), tokens, c.heads, dim, k.strides().data(), v.strides().data(),
                   c.k->data_ptr(), c.v->data_ptr(), c.dtype, c.pages, c.page_size, c.strides, c.k_scale, c.v_scale,
                   c.scale_strides, slots.data_ptr(), (int)slots.element_size(), stream);
  });
}

// kv_cache_read(k_cache, v_cache, page_table, seq_lens, k, v, k_scale, v_scale)
void read_(PyObject* const* a) {
  const at::Tensor& k = tensor(a[4], "k", 4, nullptr);
  const at::Device device = k.device();
  const at::Tensor& v = tensor(a[5], "v", 4, &device);
  dtype_code(k);
  for (const at::Tensor* t : {&k, &v}) {
    written(*t, t == &k ? "k" : "v");
    REFUSE(t->numel() && !rows_ok(*t), Value, t == &k ? "k" : "v", " must have a contiguous last dimension and 16-byte aligned rows");
  }
  REFUSE(v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type(), Value, "k and v must share shape and dtype");
  REFUSE(k.numel() && k.data_ptr() == v.data_ptr(), Value, "k and v must not be the same memory");
  const Cache c = cache_args(a[0], a[1], a[6], a[7], k, device, k.size(2), false);
  const Table t = table_args(a[2], a[3], k.size(0), device);
  if (k.size(0) == 0 || k.size(1) == 0 || t.width == 0) return;
  const int batch = as_int(k.size(0), "batch"), len = as_int(k.size(1), "length"), dim = as_int(k.size(3), "head_dim");
  launch(device, [&](void* stream) {
    return g_read(c.k->data_ptr(), c.v->data_ptr(), c.dtype, c.pages, c.page_size, c.heads, dim, c.strides, c.k_scale, c.v_scale,
                  c.scale_strides, t.pages, t.stride, t.width, t.lens, batch, k.data_ptr(), v.data_ptr(), dtype_code(k), len,
                  k.strides().data(), v.strides().data(), stream);
  });
}

// paged_decode(q, k_cache, v_cache, page_table, seq_lens, out, lse, k_scale, v_scale, sm_scale, workspace)
void decode_(PyObject* const* a) {
  const at::Tensor q = input(a[0], "q", 3, nullptr);
  const at::Device device = q.device();
  const at::Tensor& out = tensor(a[5], "out", 3, &device);
  REFUSE(out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type(), Value,
         "out must be a tensor with q's shape, dtype and device");
  REFUSE(out.stride(2) != 1, Value, "out's last dimension must be contiguous");
  written(out, "out");
  const Cache c = cache_args(a[1], a[2], a[7], a[8], q, device, -1, false);
  const int64_t batch = q.size(0), heads = q.size(1);
  REFUSE(c.heads == 0 || heads % c.heads, Value, "num_q_heads (", heads, ") must be a multiple of num_kv_heads (", c.heads, ")");
  const Table t = table_args(a[3], a[4], batch, device);
  float* lse = nullptr;
  if (given(a[6])) {
    const at::Tensor& l = tensor(a[6], "lse", 2, &device);
    REFUSE(l.size(0) != batch || l.size(1) != heads || l.scalar_type() != at::kFloat || !l.is_contiguous(), Value,
           "lse must be a contiguous float32 tensor of shape (", batch, ", ", heads, ")");
    lse = l.data_ptr<float>();
  }
  double scale = 1.0 / std::sqrt(128.0);
  if (given(a[9])) {
    scale = PyFloat_AsDouble(a[9]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  }
  if (batch == 0 || heads == 0) return;
  const int B = as_int(batch, "batch"), Hq = as_int(heads, "num_q_heads"), dim = as_int(q.size(2), "head_dim");
  at::Tensor ws;
  if (given(a[10])) {
    ws = tensor(a[10], "workspace", 1, &device);
    REFUSE(!ws.is_contiguous(), Value, "workspace must be contiguous");
  } else if (const size_t n = g_workspace_bytes(B, Hq, c.heads, c.dtype, t.width, c.page_size)) {
    ws = at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(device));
  }
  launch(device, [&](void* stream) {
    return g_decode(q.data_ptr(), dtype_code(q), B, Hq, c.heads, dim, q.strides().data(), c.k->data_ptr(), c.v->data_ptr(),
                    c.dtype, c.pages, c.page_size, c.strides, c.k_scale, c.v_scale, c.scale_strides, t.pages, t.stride, t.width,
                    t.lens, out.data_ptr(), out.strides().data(), lse, (float)scale, ws.defined() ? ws.data_ptr() : nullptr,
                    ws.defined() ? ws.nbytes() : 0, stream);
  });
}

template <void (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    F(args);
  } catch (const Value& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  } catch (const Type& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
    return nullptr;
  } catch (const Library& e) {
    PyErr_SetString(g_library_error ? g_library_error : PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// bind(write, read, decode, workspace_bytes, last_error, FlashPrefillError): addresses of the library's functions
PyObject* bind(PyObject*, PyObject* args) {
  Py_ssize_t w, r, d, b, e;
  PyObject* error;
  if (!PyArg_ParseTuple(args, "nnnnnO", &w, &r, &d, &b, &e, &error)) return nullptr;
  g_write = reinterpret_cast<decltype(g_write)>(w);
  g_read = reinterpret_cast<decltype(g_read)>(r);
  g_decode = reinterpret_cast<decltype(g_decode)>(d);
  g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(b);
  g_last_error = reinterpret_cast<decltype(g_last_error)>(e);
  Py_INCREF(error);
  g_library_error = error;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef g_methods[] = {
    {"kv_cache_write", fast<entry<write_, 7>>(), METH_FASTCALL, nullptr},
    {"kv_cache_read", fast<entry<read_, 8>>(), METH_FASTCALL, nullptr},
    {"paged_decode", fast<entry<decode_, 11>>(), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fp_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__fp_torch() {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "built_for", FPB_BUILT_FOR) < 0) Py_CLEAR(m);  // torch.__version__
  return m;
}
