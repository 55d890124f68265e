// _fkv_py: the per-call path of flexkv_amd.c_ext.transfer_kv_blocks,
// transfer_kv_blocks_kv_ptrs and the functions on a 4-bit cache as a CPython
// extension (vectorcall, no argument tuple).  It unpacks the torch tensors in C++,
// checks them, takes the current torch stream and calls the C-ABI entry with the GIL
// released, the work that csrc/bindings.cpp:25-55 does for the reference through
// pybind11.
//
// The C-ABI functions are not linked: c_ext hands over their addresses in the
// library it already loaded (bind()), so both routes drive one copy of the
// library's state.  When a check fails the functions return False without
// raising, and the Python wrapper then names the argument and the reason; a
// failed transfer raises RuntimeError with the library's last error.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>

#include "flexkv_hip.h"

namespace {

using TransferFn = int (*)(int, int, int, const int64_t*, void* const*, int64_t, int64_t,
                           const int64_t*, void*, int64_t, int64_t, int64_t, int64_t, int64_t,
                           void*, int, int, int, int);
using TransferKvPtrsFn = int (*)(int, int, int, const int64_t*, void* const*, int64_t,
                                 const int64_t*, void*, int64_t, int64_t, int64_t, int64_t,
                                 int64_t, void*, int, int, int, int);
using LastErrorFn = const char* (*)();

TransferFn g_transfer = nullptr;
TransferKvPtrsFn g_transfer_kv_ptrs = nullptr;
LastErrorFn g_last_error = nullptr;
int g_mode_kernel = 0;
int g_mode_ce = 1;
int g_device_visible = -1;   // unknown until the first call that needs the current stream

// an int64 host tensor, contiguous (the id and pointer tables)
bool int64_host(PyObject* o, const at::Tensor** out) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kLong || !t.device().is_cpu() || !t.is_contiguous()) return false;
  *out = &t;
  return true;
}

bool as_i64(PyObject* o, int64_t* v) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) return false;
  *v = x;
  return true;
}

// an argument the C-ABI takes as int
bool as_int(PyObject* o, int* v) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) return false;
  if (x < INT_MIN || x > INT_MAX) {
    PyErr_Format(PyExc_OverflowError, "%ld does not fit a C int", x);
    return false;
  }
  *v = static_cast<int>(x);
  return true;
}

// block and layer counts the C-ABI takes as int
bool count_fits(int64_t n, const char* what) {
  if (n <= INT_MAX) return true;
  PyErr_Format(PyExc_RuntimeError, "%lld %s in one call; at most %d", static_cast<long long>(n),
               what, INT_MAX);
  return false;
}

// a numpy scalar bool (numpy 1.x names its type numpy.bool_, 2.x numpy.bool)
bool is_numpy_bool(PyObject* o) {
  const char* n = Py_TYPE(o)->tp_name;
  return std::strcmp(n, "numpy.bool_") == 0 || std::strcmp(n, "numpy.bool") == 0;
}

// use_ce_transfer: a bool (Python or numpy) picks the copy engines or the
// kernel, an integer is a mode
bool as_mode(PyObject* o, int* mode) {
  if (PyBool_Check(o) || is_numpy_bool(o)) {
    const int r = PyObject_IsTrue(o);
    if (r < 0) return false;
    *mode = r ? g_mode_ce : g_mode_kernel;
    return true;
  }
  int64_t v = 0;
  if (!as_i64(o, &v)) return false;
  *mode = static_cast<int>(v);
  return true;
}

bool as_flag(PyObject* o, int* v) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) return false;
  *v = r;
  return true;
}

// The stream argument: None -> the current torch stream of the current device.
// Returns 0 with *ok false (no Python error) when no device is visible.
bool stream_of(PyObject* o, void** s, bool* ok) {
  *ok = true;
  if (o != Py_None) {
    *s = PyLong_AsVoidPtr(o);
    return !(*s == nullptr && PyErr_Occurred());
  }
  if (g_device_visible < 0) g_device_visible = c10::hip::device_count() > 0 ? 1 : 0;
  if (!g_device_visible) {
    *ok = false;
    return true;
  }
  try {
    *s = c10::hip::getCurrentHIPStream().stream();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return false;
  }
  return true;
}

PyObject* finish(int rc) {
  if (rc == 0) Py_RETURN_NONE;
  const char* msg = g_last_error ? g_last_error() : nullptr;
  if (msg && *msg)
    PyErr_SetString(PyExc_RuntimeError, msg);
  else
    PyErr_Format(PyExc_RuntimeError, "transfer failed (%d)", rc);
  return nullptr;
}

PyObject* not_bound() {
  PyErr_SetString(PyExc_RuntimeError, "_fkv_py.bind() has not been called");
  return nullptr;
}

// transfer_kv_blocks(gpu_block_ids, gpu_layer_ptrs, gpu_kv_stride, gpu_block_stride,
//                    cpu_block_ids, cpu_tensor, cpu_kv_stride, cpu_layer_stride,
//                    cpu_block_stride, chunk, start_layer, transfer_sms,
//                    is_host_to_device, use_ce_transfer, is_mla, stream)
PyObject* transfer_kv_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!g_transfer) return not_bound();
  if (n != 16) {
    PyErr_Format(PyExc_TypeError, "transfer_kv_blocks takes 16 arguments (%zd given)", n);
    return nullptr;
  }
  const at::Tensor *gids, *ptrs, *cids;
  if (!int64_host(a[0], &gids) || !int64_host(a[1], &ptrs) || !int64_host(a[4], &cids) ||
      !THPVariable_Check(a[5]))
    Py_RETURN_FALSE;
  const at::Tensor& cpu = THPVariable_Unpack(a[5]);
  const int64_t nb = gids->numel();
  if (cids->numel() != nb) Py_RETURN_FALSE;
  int64_t gkv, gblk, ckv, clay, cblk, chunk;
  int start, sms, h2d, mla, mode;
  if (!as_i64(a[2], &gkv) || !as_i64(a[3], &gblk) || !as_i64(a[6], &ckv) ||
      !as_i64(a[7], &clay) || !as_i64(a[8], &cblk) || !as_i64(a[9], &chunk) ||
      !as_int(a[10], &start) || !as_int(a[11], &sms) || !as_flag(a[12], &h2d) ||
      !as_mode(a[13], &mode) || !as_flag(a[14], &mla) || !count_fits(nb, "block ids") ||
      !count_fits(ptrs->numel(), "layer pointers"))
    return nullptr;
  void* stream = nullptr;
  bool ok = true;
  if (!stream_of(a[15], &stream, &ok)) return nullptr;
  if (!ok) Py_RETURN_FALSE;
  const int64_t* g = static_cast<const int64_t*>(gids->data_ptr());
  void* const* p = static_cast<void* const*>(ptrs->data_ptr());
  const int64_t* c = static_cast<const int64_t*>(cids->data_ptr());
  void* host = cpu.data_ptr();
  const int nl = static_cast<int>(ptrs->numel());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_transfer(static_cast<int>(nb), start, nl, g, p, gkv, gblk, c, host, ckv, clay, cblk, 0,
                  chunk, stream, sms, h2d, mode, mla);
  Py_END_ALLOW_THREADS
  return finish(rc);
}

// transfer_kv_blocks_kv_ptrs(gpu_block_ids, gpu_kv_ptrs, gpu_block_stride,
//                            cpu_block_ids, cpu_tensor, cpu_kv_stride, cpu_layer_stride,
//                            cpu_block_stride, chunk, start_layer, transfer_sms,
//                            is_host_to_device, use_ce_transfer, is_mla, stream)
PyObject* transfer_kv_blocks_kv_ptrs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!g_transfer_kv_ptrs) return not_bound();
  if (n != 15) {
    PyErr_Format(PyExc_TypeError, "transfer_kv_blocks_kv_ptrs takes 15 arguments (%zd given)", n);
    return nullptr;
  }
  const at::Tensor *gids, *ptrs, *cids;
  if (!int64_host(a[0], &gids) || !int64_host(a[1], &ptrs) || !int64_host(a[3], &cids) ||
      !THPVariable_Check(a[4]))
    Py_RETURN_FALSE;
  const at::Tensor& cpu = THPVariable_Unpack(a[4]);
  const int64_t nb = gids->numel();
  int64_t gblk, ckv, clay, cblk, chunk;
  int start, sms, h2d, mla, mode;
  if (!as_i64(a[2], &gblk) || !as_i64(a[5], &ckv) || !as_i64(a[6], &clay) ||
      !as_i64(a[7], &cblk) || !as_i64(a[8], &chunk) || !as_int(a[9], &start) ||
      !as_int(a[10], &sms) || !as_flag(a[11], &h2d) || !as_mode(a[12], &mode) ||
      !as_flag(a[13], &mla) || !count_fits(nb, "block ids") ||
      !count_fits(ptrs->numel(), "layer pointers"))
    return nullptr;
  const int kv = mla ? 1 : 2;
  if (cids->numel() != nb || ptrs->numel() % kv) Py_RETURN_FALSE;
  void* stream = nullptr;
  bool ok = true;
  if (!stream_of(a[14], &stream, &ok)) return nullptr;
  if (!ok) Py_RETURN_FALSE;
  const int64_t* g = static_cast<const int64_t*>(gids->data_ptr());
  void* const* p = static_cast<void* const*>(ptrs->data_ptr());
  const int64_t* c = static_cast<const int64_t*>(cids->data_ptr());
  void* host = cpu.data_ptr();
  const int nl = static_cast<int>(ptrs->numel() / kv);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_transfer_kv_ptrs(static_cast<int>(nb), start, nl, g, p, gblk, c, host, ckv, clay, cblk,
                          0, chunk, stream, sms, h2d, mode, mla);
  Py_END_ALLOW_THREADS
  return finish(rc);
}

// The functions on a 4-bit cache.  Each returns False, doing nothing, where an
// argument is not plainly what it takes or lies on another device than the
// current one; the Python wrapper then makes the call over ctypes, or names what
// is wrong.
decltype(&fkv_quantize_kv_blocks) g_quantize_blocks = nullptr;
decltype(&fkv_dequantize_kv_blocks) g_dequantize_blocks = nullptr;
decltype(&fkv_quantize_kv_tokens) g_quantize_tokens = nullptr;
decltype(&fkv_mx4_attention_workspace) g_attention_workspace = nullptr;
decltype(&fkv_mx4_attention) g_attention = nullptr;

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? FKV_DTYPE_BF16 : t == at::kHalf ? FKV_DTYPE_FP16
         : t == at::kFloat  ? FKV_DTYPE_FP32 : -1;
}

// a tensor on the current device that no gradient is asked for
bool here(PyObject* o, const at::Tensor** out) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != c10::hip::current_device()) return false;
  if (t.requires_grad() && c10::GradMode::is_enabled()) return false;
  *out = &t;
  return true;
}

// one layer's view [K|V, block, chunk bytes]; its tokens per block, or 0
int tokens_of_layer(const at::Tensor& mx, int64_t halves, int64_t heads, int64_t dim) {
  if (mx.scalar_type() != at::kByte || mx.dim() != 3 || mx.stride(2) != 1 ||
      mx.size(0) != halves || heads < 1 || heads > 1024 || dim < 32 || dim % 32 || dim > 1024)
    return 0;
  const int64_t token = heads * (dim / 32) * 17, tokens = mx.size(2) / token;
  return mx.size(2) % token || tokens % 16 || tokens > 4096 ? 0 : static_cast<int>(tokens);
}

// (to_mx, gpu_block_ids, gpu_layer_ptrs, gpu_kv_stride, gpu_block_stride,
//            mx_block_ids, mx_tensor, mx_kv_stride, mx_layer_stride, mx_block_stride,
//            tokens_per_block, num_heads, head_size, dtype code, start_layer, is_mla)
PyObject* mx4_blocks_of(PyObject* const* a) {
  const at::Tensor *gids, *ptrs, *mids;
  if (!int64_host(a[1], &gids) || !int64_host(a[2], &ptrs) || !int64_host(a[5], &mids) ||
      !THPVariable_Check(a[6]) || !PyLong_Check(a[13]))
    Py_RETURN_FALSE;
  const at::Tensor& mx = THPVariable_Unpack(a[6]);
  const int64_t nb = gids->numel();
  if (mids->numel() != nb) Py_RETURN_FALSE;
  int64_t gkv, gblk, mkv, mlay, mblk;
  int to_mx, tokens, heads, dim, dtype, start, mla;
  if (!as_flag(a[0], &to_mx) || !as_i64(a[3], &gkv) || !as_i64(a[4], &gblk) ||
      !as_i64(a[7], &mkv) || !as_i64(a[8], &mlay) || !as_i64(a[9], &mblk) ||
      !as_int(a[10], &tokens) || !as_int(a[11], &heads) || !as_int(a[12], &dim) ||
      !as_int(a[13], &dtype) || !as_int(a[14], &start) || !as_flag(a[15], &mla) ||
      !count_fits(nb, "block ids") || !count_fits(ptrs->numel(), "layer pointers"))
    return nullptr;
  void* stream = nullptr;
  bool ok = true;
  if (!stream_of(Py_None, &stream, &ok)) return nullptr;
  if (!ok) Py_RETURN_FALSE;
  const int64_t* g = static_cast<const int64_t*>(gids->data_ptr());
  void* const* p = static_cast<void* const*>(ptrs->data_ptr());
  const int64_t* m = static_cast<const int64_t*>(mids->data_ptr());
  void* cache = mx.data_ptr();
  const int nl = static_cast<int>(ptrs->numel());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = to_mx ? g_quantize_blocks(static_cast<int>(nb), start, nl, g, p, gkv, gblk, m, cache, mkv,
                                 mlay, mblk, tokens, heads, dim, dtype, stream, mla)
             : g_dequantize_blocks(static_cast<int>(nb), start, nl, g, p, gkv, gblk, m, cache, mkv,
                                   mlay, mblk, tokens, heads, dim, dtype, stream, mla);
  Py_END_ALLOW_THREADS
  return finish(rc);
}

// (key, value, mx_layer, slots)
PyObject* mx4_tokens_of(PyObject* const* a) {
  const at::Tensor *key, *value = nullptr, *mx, *slots;
  if (!here(a[0], &key) || (a[1] != Py_None && !here(a[1], &value)) || !here(a[2], &mx) ||
      !here(a[3], &slots))
    Py_RETURN_FALSE;
  const int dtype = dtype_code(key->scalar_type());
  if (dtype < 0 || key->dim() != 3 || key->stride(2) != 1) Py_RETURN_FALSE;
  if (value && (value->sizes() != key->sizes() || value->scalar_type() != key->scalar_type() ||
                value->stride(2) != 1))
    Py_RETURN_FALSE;
  const int64_t n = key->size(0), heads = key->size(1), dim = key->size(2);
  const int tokens = tokens_of_layer(*mx, value ? 2 : 1, heads, dim);
  const bool wide = slots->scalar_type() == at::kLong;
  if (!tokens || n > INT_MAX || (!wide && slots->scalar_type() != at::kInt) || slots->dim() != 1 ||
      slots->size(0) != n || !slots->is_contiguous())
    Py_RETURN_FALSE;
  const int64_t es = key->element_size();
  void* stream = c10::hip::getCurrentHIPStream().stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_quantize_tokens(
      static_cast<int>(n), key->data_ptr(), key->stride(0) * es, key->stride(1) * es,
      value ? value->data_ptr() : nullptr, value ? value->stride(0) * es : 0,
      value ? value->stride(1) * es : 0, slots->data_ptr(), wide, mx->data_ptr(), mx->stride(0),
      mx->stride(1), mx->size(1), tokens, static_cast<int>(heads), static_cast<int>(dim), dtype,
      stream);
  Py_END_ALLOW_THREADS
  return finish(rc);
}

// whether the bytes from a tensor's first element to its last meet another's
bool ranges_meet(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return static_cast<const char*>(x.data_ptr()) < end(y) &&
         static_cast<const char*>(y.data_ptr()) < end(x);
}

// (query, mx_layer, num_kv_heads, block_table, seq_lens, query_starts, scale, causal, out,
//  lse)
PyObject* mx4_attention_of(PyObject* const* a) {
  const at::Tensor *query, *mx, *table, *lens, *starts = nullptr, *given = nullptr, *lse = nullptr;
  if (!here(a[0], &query) || !here(a[1], &mx) || !PyLong_Check(a[2]) || !here(a[3], &table) ||
      !here(a[4], &lens) || (a[5] != Py_None && !here(a[5], &starts)) ||
      (a[6] != Py_None && !PyFloat_Check(a[6])) || (a[8] != Py_None && !here(a[8], &given)) ||
      (a[9] != Py_None && !here(a[9], &lse)))
    Py_RETURN_FALSE;
  int kv_heads, causal;
  if (!as_int(a[2], &kv_heads) || !as_flag(a[7], &causal)) return nullptr;
  const at::ScalarType type = query->scalar_type(), index = lens->scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || query->dim() != 3 || query->stride(2) != 1 ||
      kv_heads < 1)
    Py_RETURN_FALSE;
  const int64_t rows = query->size(0), heads = query->size(1), dim = query->size(2);
  if (heads < 1 || heads % kv_heads || rows > INT_MAX) Py_RETURN_FALSE;
  const int tokens = tokens_of_layer(*mx, 2, kv_heads, dim);
  if (!tokens || (index != at::kInt && index != at::kLong) || table->scalar_type() != index ||
      (starts && starts->scalar_type() != index) || lens->dim() != 1 || !lens->is_contiguous())
    Py_RETURN_FALSE;
  const int64_t batch = lens->size(0);
  if (table->dim() != 2 || table->size(0) != batch || table->size(1) > INT_MAX ||
      (table->size(1) > 1 && table->stride(1) != 1) || batch > INT_MAX)
    Py_RETURN_FALSE;
  if (starts ? starts->dim() != 1 || starts->size(0) != batch + 1 || !starts->is_contiguous()
             : rows < batch)
    Py_RETURN_FALSE;
  if (given && (given->sizes() != query->sizes() || given->scalar_type() != type ||
                given->stride(2) != 1 || ranges_meet(*given, *query)))
    Py_RETURN_FALSE;
  if (lse && (lse->dim() != 2 || lse->size(0) != rows || lse->size(1) != heads ||
              lse->scalar_type() != at::kFloat))
    Py_RETURN_FALSE;
  const at::Tensor out = given ? *given : at::empty({rows, heads, dim}, query->options());
  const int64_t es = query->element_size();
  fkv_mx4_attention_args c{};
  c.query = query->data_ptr(), c.out = out.data_ptr();
  c.lse = lse ? static_cast<float*>(lse->data_ptr()) : nullptr;
  c.query_row_stride_bytes = query->stride(0) * es;
  c.query_head_stride_bytes = query->stride(1) * es;
  c.out_row_stride_bytes = out.stride(0) * es, c.out_head_stride_bytes = out.stride(1) * es;
  c.lse_row_stride = lse ? lse->stride(0) : 0, c.lse_head_stride = lse ? lse->stride(1) : 0;
  c.mx_ptr = mx->data_ptr();
  c.mx_kv_stride_bytes = mx->stride(0), c.mx_block_stride_bytes = mx->stride(1);
  c.num_mx_blocks = mx->size(1);
  c.block_table = table->data_ptr(), c.seq_lens = lens->data_ptr();
  c.query_starts = starts ? starts->data_ptr() : nullptr;
  c.table_row_stride = table->stride(0);
  c.index_is_64bit = index == at::kLong;
  c.table_width = static_cast<int>(table->size(1));
  c.batch = static_cast<int>(batch), c.num_queries = static_cast<int>(rows);
  c.tokens_per_block = tokens, c.num_heads = kv_heads;
  c.group_size = static_cast<int>(heads / kv_heads), c.head_size = static_cast<int>(dim);
  c.dtype = dtype_code(type), c.causal = causal;
  c.scale = static_cast<float>(a[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(dim))
                                               : PyFloat_AS_DOUBLE(a[6]));
  size_t need = 0;
  int rc = g_attention_workspace(&c, &need);
  at::Tensor workspace;
  if (!rc && need) {
    // the allocator orders its reuse on the current stream
    workspace = at::empty({static_cast<int64_t>(need)}, mx->options());
    c.workspace = workspace.data_ptr(), c.workspace_bytes = need;
  }
  if (!rc) {
    void* stream = c10::hip::getCurrentHIPStream().stream();
    Py_BEGIN_ALLOW_THREADS
    rc = g_attention(&c, stream);
    Py_END_ALLOW_THREADS
  }
  PyObject* done = finish(rc);
  if (!done) return nullptr;
  Py_DECREF(done);
  return THPVariable_Wrap(out);
}

// torch's errors (an allocation that fails, a tensor without strides) as Python's
template <PyObject* (*call)(PyObject* const*)>
PyObject* checked(const char* name, PyObject* const* a, Py_ssize_t n, Py_ssize_t takes) {
  if (!g_attention) return not_bound();
  if (n != takes) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, takes, n);
    return nullptr;
  }
  try {
    return call(a);
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
PyObject* mx4_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked<mx4_blocks_of>("mx4_blocks", a, n, 16);
}
PyObject* mx4_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked<mx4_tokens_of>("mx4_tokens", a, n, 4);
}
PyObject* mx4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked<mx4_attention_of>("mx4_attention", a, n, 10);
}

// bind_mx4(quantize_blocks, dequantize_blocks, quantize_tokens, attention_workspace,
//          attention): addresses of the C-ABI functions in the loaded library
PyObject* bind_mx4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind_mx4 takes 5 arguments");
    return nullptr;
  }
  void* f[5];
  for (int i = 0; i < 5; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function address");
      return nullptr;
    }
  }
  g_quantize_blocks = reinterpret_cast<decltype(g_quantize_blocks)>(f[0]);
  g_dequantize_blocks = reinterpret_cast<decltype(g_dequantize_blocks)>(f[1]);
  g_quantize_tokens = reinterpret_cast<decltype(g_quantize_tokens)>(f[2]);
  g_attention_workspace = reinterpret_cast<decltype(g_attention_workspace)>(f[3]);
  g_attention = reinterpret_cast<decltype(g_attention)>(f[4]);
  Py_RETURN_NONE;
}

// bind(transfer, transfer_kv_ptrs, last_error, mode_kernel, mode_ce): addresses
// of the C-ABI functions in the loaded library and the two mode values.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes 5 arguments");
    return nullptr;
  }
  void* f[3];
  for (int i = 0; i < 3; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function address");
      return nullptr;
    }
  }
  int64_t mk = 0, mc = 0;
  if (!as_i64(a[3], &mk) || !as_i64(a[4], &mc)) return nullptr;
  g_transfer = reinterpret_cast<TransferFn>(f[0]);
  g_transfer_kv_ptrs = reinterpret_cast<TransferKvPtrsFn>(f[1]);
  g_last_error = reinterpret_cast<LastErrorFn>(f[2]);
  g_mode_kernel = static_cast<int>(mk);
  g_mode_ce = static_cast<int>(mc);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"transfer_kv_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(
                               &transfer_kv_blocks)),
     METH_FASTCALL, "Checked per-call path of c_ext.transfer_kv_blocks (16 positional)."},
    {"transfer_kv_blocks_kv_ptrs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(
                                       &transfer_kv_blocks_kv_ptrs)),
     METH_FASTCALL, "Checked per-call path of c_ext.transfer_kv_blocks_kv_ptrs (15 positional)."},
    {"mx4_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&mx4_blocks)),
     METH_FASTCALL, "Per-call path of c_ext.(de)quantize_kv_blocks (16 positional)."},
    {"mx4_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&mx4_tokens)),
     METH_FASTCALL, "Per-call path of c_ext.quantize_kv_tokens (4 positional)."},
    {"mx4_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&mx4_attention)),
     METH_FASTCALL, "Per-call path of c_ext.mx4_attention (10 positional)."},
    {"bind_mx4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind_mx4)),
     METH_FASTCALL, "Hand over the addresses of the functions on a 4-bit cache."},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL,
     "Hand over the C-ABI function addresses and mode values."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fkv_py", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fkv_py() { return PyModule_Create(&kModule); }
