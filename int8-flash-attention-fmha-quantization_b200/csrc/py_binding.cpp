// Native Python binding of the C ABI (include/fmha_i8_c.h): reads the descriptor objects, tensor addresses and the
// stream straight from the Python arguments and calls the library with the GIL released.
//
// Why it exists: a forward call on a short sequence keeps the GPU busy for 5-7 us, and building the same call from
// ctypes arrays and torch.cuda.current_stream() costs about 8 us of Python per call (measured on the B200 host: two
// descriptor arrays 1.1 us, five addresses 1.3 us, the stream object 3.6 us, the foreign call 1.5 us), so the host was
// what bounded it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cstdint>
#include <initializer_list>
#include <utility>

#include "../../include/fmha_i8_c.h"

namespace {

PyObject *s_q_amax, *s_k_amax, *s_v_amax, *s_o_amax, *s_s_max;
PyObject *s_batch_num, *s_seq_len, *s_seq_len_q, *s_seq_len_k, *s_head_num, *s_head_dim;
PyObject *s_data_ptr, *s_ctypes, *s_data, *s_cuda_stream;
PyObject *s_max_seq_q, *s_max_seq_k, *s_head_num_kv, *s_dtype, *s_shape, *s_stride, *s_get_device;

// torch's raw-stream getters (device index -> stream handle, and the current device index), once torch's CUDA state is
// initialised; until then the Python-level slow path, which initialises it.
PyObject *g_raw_stream, *g_get_device, *g_slow_stream;

// torch's element types, in the order of Type, and its function for the current device index, once torch is imported.
enum Type { kInt8 = FMHA_I8_TYPE_I8, kBf16 = FMHA_I8_TYPE_BF16, kFp16 = FMHA_I8_TYPE_FP16, kFp32 = FMHA_I8_TYPE_FP32, kInt32, kInt64, kFp64, kTypes };
const char* const g_type_names[kTypes] = {"int8", "bfloat16", "float16", "float32", "int32", "int64", "float64"};
PyObject* g_types[kTypes];
PyObject* g_slow_device;

bool get_float(PyObject* obj, PyObject* name, float* out) {
  PyObject* v = PyObject_GetAttr(obj, name);
  if (!v) return false;
  const double d = PyFloat_AsDouble(v);
  Py_DECREF(v);
  if (d == -1.0 && PyErr_Occurred()) return false;
  *out = static_cast<float>(d);
  return true;
}
bool get_int(PyObject* obj, PyObject* name, int* out) {
  PyObject* v = PyObject_GetAttr(obj, name);
  if (!v) return false;
  PyObject* i = PyNumber_Index(v);
  Py_DECREF(v);
  if (!i) return false;
  *out = static_cast<int>(PyLong_AsUnsignedLongLongMask(i));
  Py_DECREF(i);
  return true;
}
// Whatever int() takes.
bool as_int(PyObject* v, int* out) {
  PyObject* i = PyNumber_Long(v);
  if (!i) return false;
  *out = static_cast<int>(PyLong_AsUnsignedLongLongMask(i));
  Py_DECREF(i);
  return true;
}
bool as_address(PyObject* v, void** out) {
  const unsigned long long a = PyLong_AsUnsignedLongLongMask(v);
  if (a == static_cast<unsigned long long>(-1) && PyErr_Occurred()) return false;
  *out = reinterpret_cast<void*>(static_cast<uintptr_t>(a));
  return true;
}

// Device or host address of None, an int, a torch tensor or a numpy array.
bool get_ptr(PyObject* x, void** out) {
  if (x == Py_None) { *out = nullptr; return true; }
  if (PyLong_Check(x)) return as_address(x, out);
  PyObject* r = PyObject_CallMethodNoArgs(x, s_data_ptr);
  if (!r && PyErr_ExceptionMatches(PyExc_AttributeError)) {
    PyErr_Clear();
    PyObject* c = PyObject_GetAttr(x, s_ctypes);
    if (c) {
      r = PyObject_GetAttr(c, s_data);
      Py_DECREF(c);
    } else {
      PyErr_Clear();
      PyErr_Format(PyExc_TypeError, "cannot take the address of %R", reinterpret_cast<PyObject*>(Py_TYPE(x)));
    }
  }
  if (!r) return false;
  const bool ok = as_address(r, out);
  Py_DECREF(r);
  return ok;
}

bool get_stream(PyObject* s, void** out) {
  PyObject* r;
  if (s == Py_None) {
    if (g_raw_stream) {
      PyObject* dev = PyObject_CallNoArgs(g_get_device);
      if (!dev) return false;
      r = PyObject_CallOneArg(g_raw_stream, dev);
      Py_DECREF(dev);
    } else {
      r = PyObject_CallNoArgs(g_slow_stream);
    }
  } else if (PyLong_Check(s)) {
    return as_address(s, out);
  } else {
    r = PyObject_GetAttr(s, s_cuda_stream);
  }
  if (!r) return false;
  const bool ok = as_address(r, out);
  Py_DECREF(r);
  return ok;
}

bool get_param(PyObject* p, float (&a)[5]) {
  return get_float(p, s_q_amax, &a[0]) && get_float(p, s_k_amax, &a[1]) && get_float(p, s_v_amax, &a[2]) && get_float(p, s_o_amax, &a[3]) &&
         get_float(p, s_s_max, &a[4]);
}
bool get_desc4(PyObject* d, int (&a)[4]) {
  return get_int(d, s_batch_num, &a[0]) && get_int(d, s_seq_len, &a[1]) && get_int(d, s_head_num, &a[2]) && get_int(d, s_head_dim, &a[3]);
}
bool get_desc5(PyObject* d, int (&a)[5]) {
  return get_int(d, s_batch_num, &a[0]) && get_int(d, s_seq_len_q, &a[1]) && get_int(d, s_seq_len_k, &a[2]) && get_int(d, s_head_num, &a[3]) &&
         get_int(d, s_head_dim, &a[4]);
}
bool want(Py_ssize_t got, Py_ssize_t n) {
  if (got == n) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", n, got);
  return false;
}

// infer(stream, param, desc, q, k, v, mask, o, flags) -> status
PyObject* py_infer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void *stream, *t[5];
  float amax[5];
  int desc[4], flags, st;
  if (!want(n, 9) || !get_stream(a[0], &stream) || !get_param(a[1], amax) || !get_desc4(a[2], desc) || !as_int(a[8], &flags)) return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!get_ptr(a[3 + i], &t[i])) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer(stream, amax, desc, t[0], t[1], t[2], t[3], t[4], static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// infer_slice(stream, param, desc, q, k, v, mask, o, bh_begin, bh_count, flags) -> status
PyObject* py_infer_slice(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void *stream, *t[5];
  float amax[5];
  int desc[4], begin, count, flags, st;
  if (!want(n, 11) || !get_stream(a[0], &stream) || !get_param(a[1], amax) || !get_desc4(a[2], desc) || !as_int(a[8], &begin) ||
      !as_int(a[9], &count) || !as_int(a[10], &flags))
    return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!get_ptr(a[3 + i], &t[i])) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer_slice(stream, amax, desc, t[0], t[1], t[2], t[3], t[4], begin, count, static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// bh_count == None: all heads from bh_begin on
bool get_slice(PyObject* begin, PyObject* count, const int (&desc)[5], int* b, int* c) {
  if (!as_int(begin, b)) return false;
  if (count == Py_None) {
    *c = static_cast<int>(static_cast<long long>(desc[0]) * desc[3] - *b);
    return true;
  }
  return as_int(count, c);
}

// infer_cross(stream, param, desc_x, q, k, v, mask, o, bh_begin, bh_count, flags) -> status
PyObject* py_infer_cross(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void *stream, *t[5];
  float amax[5];
  int desc[5], begin, count, flags, st;
  if (!want(n, 11) || !get_stream(a[0], &stream) || !get_param(a[1], amax) || !get_desc5(a[2], desc) || !get_slice(a[8], a[9], desc, &begin, &count) ||
      !as_int(a[10], &flags))
    return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!get_ptr(a[3 + i], &t[i])) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer_cross(stream, amax, desc, t[0], t[1], t[2], t[3], t[4], begin, count, static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// infer_policy(stream, param, desc_x, q, k, v, mask, o, bh_begin, bh_count, flags, policy, row_scratch) -> status
PyObject* py_infer_policy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void *stream, *t[5], *scratch;
  float amax[5];
  int desc[5], begin, count, flags, policy, st;
  if (!want(n, 13) || !get_stream(a[0], &stream) || !get_param(a[1], amax) || !get_desc5(a[2], desc) || !get_slice(a[8], a[9], desc, &begin, &count) ||
      !as_int(a[10], &flags) || !as_int(a[11], &policy) || !get_ptr(a[12], &scratch))
    return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!get_ptr(a[3 + i], &t[i])) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer_policy(stream, amax, desc, t[0], t[1], t[2], t[3], t[4], begin, count, static_cast<unsigned>(flags), policy,
                                  static_cast<float*>(scratch));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// infer_host(param, desc, q, k, v, mask, o, bh_begin, bh_count, flags) -> status; bh_begin None: the whole problem
PyObject* py_infer_host(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* t[5];
  float amax[5];
  int desc[4], begin = 0, count = 0, flags, st;
  if (!want(n, 10) || !get_param(a[0], amax) || !get_desc4(a[1], desc) || !as_int(a[9], &flags)) return nullptr;
  const bool whole = a[7] == Py_None;
  if (!whole && (!as_int(a[7], &begin) || !as_int(a[8], &count))) return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!get_ptr(a[2 + i], &t[i])) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = whole ? fmha_i8_sm100_infer_host(amax, desc, t[0], t[1], t[2], t[3], t[4], static_cast<unsigned>(flags))
             : fmha_i8_sm100_infer_host_slice(amax, desc, t[0], t[1], t[2], t[3], t[4], begin, count, static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// quantize(stream, x, n, out, amax_out, no_alloc) -> status
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void *stream, *x, *out, *amax;
  int st;
  if (!want(n, 6) || !get_stream(a[0], &stream) || !get_ptr(a[1], &x) || !get_ptr(a[3], &out) || !get_ptr(a[4], &amax)) return nullptr;
  const long long count = PyLong_AsLongLong(a[2]);
  if (count == -1 && PyErr_Occurred()) return nullptr;
  const int no_alloc = PyObject_IsTrue(a[5]);
  if (no_alloc < 0) return nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = (no_alloc ? fmha_i8_sm100_quantize_f32_noalloc : fmha_i8_sm100_quantize_f32)(stream, static_cast<const float*>(x), count,
                                                                                    static_cast<int8_t*>(out), static_cast<float*>(amax));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// What a serving call reads of a torch tensor.
struct Tensor {
  const char* name;
  void* ptr;
  int type, dims;
  long long size[4], stride[4];
};
bool load_torch() {
  if (g_slow_device) return true;
  PyObject* torch = PyImport_ImportModule("torch");
  if (!torch) return false;
  for (int i = 0; i < kTypes; ++i) {
    PyObject* t = PyObject_GetAttrString(torch, g_type_names[i]);
    if (!t) { Py_DECREF(torch); return false; }
    Py_XSETREF(g_types[i], t);
  }
  PyObject* cuda = PyObject_GetAttrString(torch, "cuda");
  Py_DECREF(torch);
  if (!cuda) return false;
  g_slow_device = PyObject_GetAttrString(cuda, "current_device");
  Py_DECREF(cuda);
  return g_slow_device != nullptr;
}
bool bad(const char* name, const char* what) {
  PyErr_Format(PyExc_ValueError, "%s: %s", name, what);
  return false;
}
bool read_tuple(PyObject* t, int n, long long* out) {
  for (int i = 0; i < n; ++i) {
    out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(t, i));
    if (out[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}
// The tensor's memory, sizes and strides; its type has to be one of `types` (bits).
bool get_tensor(PyObject* x, const char* name, unsigned types, int dims, Tensor* t) {
  t->name = name;
  PyObject* type = PyObject_GetAttr(x, s_dtype);
  if (!type) {
    PyErr_Clear();
    PyErr_Format(PyExc_TypeError, "%s: expected a torch tensor, got %R", name, reinterpret_cast<PyObject*>(Py_TYPE(x)));
    return false;
  }
  t->type = 0;
  while (t->type < kTypes && g_types[t->type] != type) ++t->type;
  Py_DECREF(type);
  if (t->type == kTypes || !((types >> t->type) & 1u)) return bad(name, "wrong element type");
  PyObject* shape = PyObject_GetAttr(x, s_shape);
  if (!shape || !PyTuple_Check(shape)) { Py_XDECREF(shape); return PyErr_Occurred() ? false : bad(name, "no shape"); }
  t->dims = static_cast<int>(PyTuple_GET_SIZE(shape));
  const bool fits = t->dims == dims;
  const bool ok = fits && read_tuple(shape, dims, t->size);
  Py_DECREF(shape);
  if (!fits) { PyErr_Format(PyExc_ValueError, "%s: %d dimensions, expected %d", name, t->dims, dims); return false; }
  if (!ok) return false;
  PyObject* stride = PyObject_CallMethodNoArgs(x, s_stride);
  if (!stride || !PyTuple_Check(stride)) { Py_XDECREF(stride); return PyErr_Occurred() ? false : bad(name, "no strides"); }
  const bool read = read_tuple(stride, dims, t->stride);
  Py_DECREF(stride);
  return read && get_ptr(x, &t->ptr);
}
// Dimensions from `first` on lie densely one in the other; one of size 1 may have any stride, and so may all of a tensor without elements.
bool dense_from(const Tensor& t, int first) {
  for (int i = 0; i < t.dims; ++i)
    if (t.size[i] == 0) return true;
  long long want = 1;
  for (int i = t.dims - 1; i >= first; --i) {
    if (t.size[i] != 1 && t.stride[i] != want) return bad(t.name, "the last dimensions have to be contiguous");
    want *= t.size[i];
  }
  return true;
}
bool has_sizes(const Tensor& t, int first, std::initializer_list<long long> sizes) {
  int i = first;
  for (const long long n : sizes)
    if (t.size[i++] != n) {
      PyErr_Format(PyExc_ValueError, "%s: dimension %d has %lld elements, expected %lld", t.name, i - 1, t.size[i - 1], n);
      return false;
    }
  return true;
}
// Elements from one index of dimension 0 to the next; a dimension that has no next one counts as dense.
long long outer_stride(const Tensor& t) {
  if (t.size[0] > 1) return t.stride[0];
  long long n = 1;
  for (int i = 1; i < t.dims; ++i) n *= t.size[i];
  return n;
}
// All tensors are on the current CUDA device.
bool on_current_device(std::initializer_list<std::pair<PyObject*, const char*>> tensors) {
  PyObject* now = nullptr;
  long device = -1;
  for (const auto& x : tensors) {
    if (x.first == Py_None) continue;
    PyObject* d = PyObject_CallMethodNoArgs(x.first, s_get_device);
    if (!d) return false;
    const long at = PyLong_AsLong(d);
    Py_DECREF(d);
    if (at == -1 && PyErr_Occurred()) return false;
    if (at < 0) return bad(x.second, "not a CUDA tensor");
    if (!now) {
      now = PyObject_CallNoArgs(g_get_device ? g_get_device : g_slow_device);
      if (!now) return false;
      device = PyLong_AsLong(now);
      Py_DECREF(now);
    }
    if (at != device) { PyErr_Format(PyExc_ValueError, "%s: on device %ld, but the current device is %ld", x.second, at, device); return false; }
  }
  return true;
}
bool get_desc6(PyObject* d, int (&a)[6]) {
  return get_int(d, s_batch_num, &a[0]) && get_int(d, s_max_seq_q, &a[1]) && get_int(d, s_max_seq_k, &a[2]) && get_int(d, s_head_num, &a[3]) &&
         get_int(d, s_head_num_kv, &a[4]) && get_int(d, s_head_dim, &a[5]);
}
constexpr unsigned bit(Type t) { return 1u << t; }
constexpr unsigned kOutTypes = bit(kInt8) | bit(kBf16) | bit(kFp16), kInTypes = bit(kBf16) | bit(kFp16) | bit(kFp32);

// infer_packed(stream, param, desc, q, k, v, cu_seqlens_q, cu_seqlens_k, o, flags) -> status
PyObject* py_infer_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* stream;
  float amax[5];
  int desc[6], flags, st;
  Tensor q, k, v, cu_q, cu_k, o;
  if (!want(n, 10) || !load_torch() || !get_param(a[1], amax) || !get_desc6(a[2], desc) || !get_tensor(a[3], "q", bit(kInt8), 3, &q) ||
      !get_tensor(a[4], "k", bit(kInt8), 3, &k) || !get_tensor(a[5], "v", bit(kInt8), 3, &v) || !get_tensor(a[6], "cu_seqlens_q", bit(kInt32), 1, &cu_q) ||
      !get_tensor(a[7], "cu_seqlens_k", bit(kInt32), 1, &cu_k) || !get_tensor(a[8], "o", kOutTypes, 3, &o) || !as_int(a[9], &flags))
    return nullptr;
  if (!has_sizes(q, 1, {desc[3], desc[5]}) || !has_sizes(k, 1, {desc[4], desc[5]}) || !has_sizes(v, 0, {k.size[0], desc[4], desc[5]}) ||
      !has_sizes(o, 0, {q.size[0], desc[3], desc[5]}) || !has_sizes(cu_q, 0, {desc[0] + 1LL}) || !has_sizes(cu_k, 0, {desc[0] + 1LL}) || !dense_from(q, 1) ||
      !dense_from(k, 1) || !dense_from(v, 1) || !dense_from(o, 1) || !dense_from(cu_q, 0) || !dense_from(cu_k, 0) ||
      !on_current_device({{a[3], "q"}, {a[4], "k"}, {a[5], "v"}, {a[6], "cu_seqlens_q"}, {a[7], "cu_seqlens_k"}, {a[8], "o"}}) || !get_stream(a[0], &stream))
    return nullptr;
  if (q.size[0] == 0) return PyLong_FromLong(0);      // no tokens, and no memory
  const long long tokens[2] = {q.size[0], k.size[0]}, strides[4] = {outer_stride(q), outer_stride(k), outer_stride(v), outer_stride(o)};
  alignas(16) static char nothing[16];                // no keys: an address that is not read
  const void *kp = k.ptr ? k.ptr : nothing, *vp = v.ptr ? v.ptr : nothing;
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer_packed(stream, amax, desc, q.ptr, kp, vp, static_cast<const int*>(cu_q.ptr), static_cast<const int*>(cu_k.ptr), o.ptr, o.type, tokens,
                                  strides, static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// infer_paged(stream, param, desc, q, k_cache, v_cache, page_table, seqlens_k, cu_seqlens_q, o, flags) -> status
PyObject* py_infer_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* stream;
  float amax[5];
  int desc[6], flags, st;
  Tensor q, k, v, table, lens, cu_q, o;
  if (!want(n, 11) || !load_torch() || !get_param(a[1], amax) || !get_desc6(a[2], desc) || !get_tensor(a[3], "q", bit(kInt8), 3, &q) ||
      !get_tensor(a[4], "k_cache", bit(kInt8), 4, &k) || !get_tensor(a[5], "v_cache", bit(kInt8), 4, &v) || !get_tensor(a[6], "page_table", bit(kInt32), 2, &table) ||
      !get_tensor(a[7], "seqlens_k", bit(kInt32), 1, &lens) || !get_tensor(a[8], "cu_seqlens_q", bit(kInt32), 1, &cu_q) || !get_tensor(a[9], "o", kOutTypes, 3, &o) ||
      !as_int(a[10], &flags))
    return nullptr;
  if (!has_sizes(q, 1, {desc[3], desc[5]}) || !has_sizes(k, 1, {desc[4], k.size[2], desc[5]}) || !has_sizes(v, 0, {k.size[0], desc[4], k.size[2], desc[5]}) ||
      !has_sizes(o, 0, {q.size[0], desc[3], desc[5]}) || !has_sizes(table, 0, {desc[0]}) || !has_sizes(lens, 0, {desc[0]}) || !has_sizes(cu_q, 0, {desc[0] + 1LL}) ||
      !dense_from(q, 1) || !dense_from(k, 1) || !dense_from(v, 1) || !dense_from(o, 1) || !dense_from(table, 1) || !dense_from(lens, 0) || !dense_from(cu_q, 0))
    return nullptr;
  if (outer_stride(k) != outer_stride(v)) return bad("v_cache", "its pages have to be as far apart as those of k_cache"), nullptr;
  if (!on_current_device({{a[3], "q"}, {a[4], "k_cache"}, {a[5], "v_cache"}, {a[6], "page_table"}, {a[7], "seqlens_k"}, {a[8], "cu_seqlens_q"}, {a[9], "o"}}) ||
      !get_stream(a[0], &stream))
    return nullptr;
  if (q.size[0] == 0) return PyLong_FromLong(0);
  const long long strides[2] = {outer_stride(q), outer_stride(o)}, cache[5] = {k.size[0], k.size[2], outer_stride(k), table.size[1], outer_stride(table)};
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_infer_paged(stream, amax, desc, q.ptr, k.ptr, v.ptr, static_cast<const int*>(table.ptr), static_cast<const int*>(lens.ptr),
                                 static_cast<const int*>(cu_q.ptr), o.ptr, o.type, q.size[0], strides, cache, static_cast<unsigned>(flags));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// rope_table(stream, inv_freq, table, magnitude) -> status
PyObject* py_rope_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* stream;
  Tensor freq, table;
  int st;
  if (!want(n, 4) || !load_torch() || !get_tensor(a[1], "inv_freq", bit(kFp64), 1, &freq) || !get_tensor(a[2], "table", bit(kFp32), 3, &table)) return nullptr;
  const double magnitude = PyFloat_AsDouble(a[3]);
  if (magnitude == -1.0 && PyErr_Occurred()) return nullptr;
  if (!has_sizes(table, 0, {2}) || !has_sizes(table, 2, {2 * freq.size[0]}) || !dense_from(freq, 0) || !dense_from(table, 0) ||
      !on_current_device({{a[1], "inv_freq"}, {a[2], "table"}}) || !get_stream(a[0], &stream))
    return nullptr;
  if (freq.size[0] == 0 || table.size[1] == 0) return PyLong_FromLong(0);
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_rope_table(stream, static_cast<const double*>(freq.ptr), static_cast<int>(freq.size[0]), table.size[1], magnitude,
                                static_cast<float*>(table.ptr));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// rope_append(stream, param, q, k, v, positions, table or None, q_out, k_out, v_out, slots or None, interleaved) -> status
PyObject* py_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* stream;
  float amax[5];
  Tensor q, k, v, positions, table{}, q_out, k_out, v_out, slots{};
  int st;
  if (!want(n, 12) || !load_torch() || !get_param(a[1], amax) || !get_tensor(a[2], "q", kInTypes, 3, &q) || !get_tensor(a[3], "k", kInTypes, 3, &k) ||
      !get_tensor(a[4], "v", kInTypes, 3, &v) || !get_tensor(a[5], "positions", bit(kInt32), 1, &positions))
    return nullptr;
  const bool turned = a[6] != Py_None, paged = a[10] != Py_None;
  const int dims = paged ? 4 : 3;
  if ((turned && !get_tensor(a[6], "table", bit(kFp32), 3, &table)) || !get_tensor(a[7], "q_out", bit(kInt8), 3, &q_out) ||
      !get_tensor(a[8], "k_out", bit(kInt8), dims, &k_out) || !get_tensor(a[9], "v_out", bit(kInt8), dims, &v_out) ||
      (paged && !get_tensor(a[10], "slots", bit(kInt64), 1, &slots)))
    return nullptr;
  const int interleaved = PyObject_IsTrue(a[11]);
  if (interleaved < 0) return nullptr;
  if (k.type != q.type || v.type != q.type) return bad("k, v", "their element type has to be that of q"), nullptr;
  const long long T = q.size[0], H = q.size[1], Hkv = k.size[1], D = q.size[2];
  if (!has_sizes(k, 0, {T, Hkv, D}) || !has_sizes(v, 0, {T, Hkv, D}) || !has_sizes(positions, 0, {T}) || !has_sizes(q_out, 0, {T, H, D}) ||
      (turned && !has_sizes(table, 0, {2})) || (paged && !has_sizes(slots, 0, {T})))
    return nullptr;
  if (paged ? !has_sizes(k_out, 1, {Hkv, k_out.size[2], D}) || !has_sizes(v_out, 0, {k_out.size[0], Hkv, k_out.size[2], D})
            : !has_sizes(k_out, 0, {T, Hkv, D}) || !has_sizes(v_out, 0, {T, Hkv, D}))
    return nullptr;
  const int from = paged ? 1 : 0;
  if (!dense_from(q, 1) || !dense_from(k, 1) || !dense_from(v, 1) || !dense_from(positions, 0) || (turned && !dense_from(table, 0)) || !dense_from(q_out, 0) ||
      !dense_from(k_out, from) || !dense_from(v_out, from) || (paged && !dense_from(slots, 0)))
    return nullptr;
  if (paged && outer_stride(k_out) != outer_stride(v_out)) return bad("v_out", "its pages have to be as far apart as those of k_out"), nullptr;
  if (!on_current_device({{a[2], "q"}, {a[3], "k"}, {a[4], "v"}, {a[5], "positions"}, {a[6], "table"}, {a[7], "q_out"}, {a[8], "k_out"}, {a[9], "v_out"}, {a[10], "slots"}}) ||
      !get_stream(a[0], &stream))
    return nullptr;
  if (T == 0) return PyLong_FromLong(0);
  const long long rot = turned ? table.size[2] : 0;
  const long long shape[5] = {T, H, Hkv, D, rot}, strides[3] = {outer_stride(q), outer_stride(k), outer_stride(v)}, cache[3] = {k_out.size[0], paged ? k_out.size[2] : 0, outer_stride(k_out)};
  Py_BEGIN_ALLOW_THREADS
  st = fmha_i8_sm100_rope_quantize_append(stream, amax, shape, q.ptr, k.ptr, v.ptr, q.type, strides, static_cast<const int*>(positions.ptr),
                                          static_cast<const float*>(table.ptr), turned ? table.size[1] : 0, interleaved, static_cast<int8_t*>(q_out.ptr), static_cast<int8_t*>(k_out.ptr),
                                          static_cast<int8_t*>(v_out.ptr), static_cast<const long long*>(slots.ptr), cache);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// set_stream_source(slow) before first use; set_raw_stream(raw_stream, get_device) once torch's CUDA state exists
PyObject* py_set_stream_source(PyObject*, PyObject* slow) {
  Py_INCREF(slow);
  Py_XSETREF(g_slow_stream, slow);
  Py_RETURN_NONE;
}
PyObject* py_set_raw_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 2)) return nullptr;
  Py_INCREF(a[1]);
  Py_XSETREF(g_get_device, a[1]);
  Py_INCREF(a[0]);
  Py_XSETREF(g_raw_stream, a[0]);
  Py_RETURN_NONE;
}

#define FAST(name) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr
PyMethodDef g_methods[] = {
    {"infer", FAST(py_infer)},
    {"infer_slice", FAST(py_infer_slice)},
    {"infer_cross", FAST(py_infer_cross)},
    {"infer_policy", FAST(py_infer_policy)},
    {"infer_host", FAST(py_infer_host)},
    {"quantize", FAST(py_quantize)},
    {"infer_packed", FAST(py_infer_packed)},
    {"infer_paged", FAST(py_infer_paged)},
    {"rope_table", FAST(py_rope_table)},
    {"rope_append", FAST(py_rope_append)},
    {"set_stream_source", py_set_stream_source, METH_O, nullptr},
    {"set_raw_stream", FAST(py_set_raw_stream)},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fmha_i8_py", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fmha_i8_py(void) {
  struct { PyObject** slot; const char* text; } names[] = {
      {&s_q_amax, "q_amax"}, {&s_k_amax, "k_amax"}, {&s_v_amax, "v_amax"}, {&s_o_amax, "o_amax"}, {&s_s_max, "s_max"},
      {&s_batch_num, "batch_num"}, {&s_seq_len, "seq_len"}, {&s_seq_len_q, "seq_len_q"}, {&s_seq_len_k, "seq_len_k"},
      {&s_head_num, "head_num"}, {&s_head_dim, "head_dim"}, {&s_data_ptr, "data_ptr"}, {&s_ctypes, "ctypes"}, {&s_data, "data"},
      {&s_cuda_stream, "cuda_stream"}, {&s_max_seq_q, "max_seq_q"}, {&s_max_seq_k, "max_seq_k"}, {&s_head_num_kv, "head_num_kv"}, {&s_dtype, "dtype"},
      {&s_shape, "shape"}, {&s_stride, "stride"}, {&s_get_device, "get_device"}};
  for (auto& x : names)
    if (!(*x.slot = PyUnicode_InternFromString(x.text))) return nullptr;
  return PyModule_Create(&g_module);
}
