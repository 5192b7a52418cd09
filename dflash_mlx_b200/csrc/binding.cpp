// Python binding of the operators whose host side would otherwise cost more than their kernels: argument checks, output and
// workspace allocation and the call into the C ABI in one C++ function per operator (a few microseconds, against 25 to 30 for
// the same steps in Python).  Tensors come from and go to torch; the computing is behind the function pointers that bind() is
// given, which are those of libdflash_b200.
//
// Every check of the public functions in quantized_kv.py and logprobs.py is made here; a refusal is a ValueError, a status
// of the library the exception class given to bind().
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <sstream>
#include <string>
#include <utility>

#include "../../include/dflash_b200.h"

namespace {

struct Library {
  decltype(&dflash_kv4_write) write;
  decltype(&dflash_kv4_read) read;
  decltype(&dflash_kv4_sdpa_workspace_bytes) sdpa_workspace;
  decltype(&dflash_kv4_sdpa) sdpa;
  decltype(&dflash_token_logprobs) logprobs;
  decltype(&dflash_last_error_string) error;
} lib{};
PyObject* error_class = nullptr;

constexpr int kGroup = 64, kMaxTopK = 32;

struct Refusal { std::string text; };
template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refusal{s.str()};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o, const char* name) {
  PyObject* i = PyNumber_Index(o);
  if (!i) {
    PyErr_Clear();
    refuse(name, " must be an integer");
  }
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(i, &overflow);
  Py_DECREF(i);
  if (overflow) refuse(name, " does not fit 64 bits");
  return v;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a number");
  }
  return v;
}

// All operands on one CUDA device.
struct Device {
  c10::Device dev{c10::kCPU};
  bool any = false;
  void add(const at::Tensor* t) {
    if (!t) return;
    if (!t->is_cuda()) refuse("dflash_mlx_b200 ops take CUDA tensors (there is no CPU path)");
    if (!any) {
      dev = t->device();
      any = true;
    } else if (t->device() != dev) {
      refuse("all operands must live on the same CUDA device");
    }
  }
};

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return DFLASH_BF16;
    case at::kHalf: return DFLASH_F16;
    case at::kFloat: return DFLASH_F32;
    default: refuse("unsupported dtype ", t);
  }
}

struct Side {
  dflash_kv4_cache c;
  int64_t B, Hk, cap, D;
  at::ScalarType type;
  bool same(const Side& o) const { return B == o.B && Hk == o.Hk && cap == o.cap && D == o.D && type == o.type; }
};

Side side(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& biases, const char* name) {
  if (codes.dim() != 4 || (codes.scalar_type() != at::kInt && codes.scalar_type() != at::kUInt32))
    refuse(name, " codes must be int32 [B, Hk, capacity, D/8], got ", codes.scalar_type(), " ", codes.sizes());
  Side s;
  s.B = codes.size(0); s.Hk = codes.size(1); s.cap = codes.size(2); s.D = codes.size(3) * 8;
  if (s.D != 128 && s.D != 256) refuse(name, ": D=", s.D, " is not supported (need 128 or 256)");
  if (s.B > INT_MAX || s.Hk > INT_MAX || s.cap > INT_MAX) refuse(name, ": sizes beyond 31 bits");
  const int64_t want[4] = {s.B, s.Hk, s.cap, s.D / kGroup};
  for (const at::Tensor* t : {&scales, &biases})
    if (t->sizes() != at::IntArrayRef(want, 4))
      refuse(name, t == &scales ? " scales" : " biases", " must be [B, Hk, capacity, D/64] = ",
             at::IntArrayRef(want, 4), ", got ", t->sizes());
  s.type = scales.scalar_type();
  if ((s.type != at::kBFloat16 && s.type != at::kHalf) || biases.scalar_type() != s.type)
    refuse(name, " scales and biases must share bfloat16 or float16");
  for (const at::Tensor* t : {&codes, &scales, &biases})
    if (t->stride(3) != 1 || (t->stride(2) != t->size(3) && s.cap > 1)) refuse(name, ": the positions of a cache must be contiguous");
  // the stride of a dimension of one element is never used
  auto st = [](const at::Tensor& t, int d) { return t.size(d) > 1 ? (long long)t.stride(d) : 0ll; };
  s.c = dflash_kv4_cache{(uint32_t*)codes.data_ptr(), scales.data_ptr(), biases.data_ptr(), st(codes, 0), st(codes, 1),
                         st(scales, 0), st(scales, 1), st(biases, 0), st(biases, 1)};
  return s;
}

struct Cache { Side k, v; };
Cache cache(PyObject* const* a, Device* d) {   // six arguments: key codes, scales, biases, value codes, scales, biases
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) t[i] = &tensor(a[i], "cache arrays");
  if (d) for (const at::Tensor* x : t) d->add(x);
  Cache c{side(*t[0], *t[1], *t[2], "key cache"), side(*t[3], *t[4], *t[5], "value cache")};
  if (!c.k.same(c.v)) refuse("the key cache and the value cache differ in shape or type");
  return c;
}

// A cache that is written: no place of it may belong to two sequences, heads or sides, whose blocks would race for it.
void check_apart(PyObject* const* a) {
  for (int i = 0; i < 6; ++i) {
    const at::Tensor& x = THPVariable_Unpack(a[i]);
    if (x.numel() == 0) return;
    const int64_t block = x.size(2) * x.size(3);   // one head's positions, contiguous
    int64_t n[2] = {x.size(0), x.size(1)}, s[2] = {x.stride(0), x.stride(1)};
    for (int d = 0; d < 2; ++d) if (n[d] == 1) s[d] = 0;
    if (s[0] > s[1]) { std::swap(s[0], s[1]); std::swap(n[0], n[1]); }
    if ((n[0] > 1 && s[0] < block) || (n[1] > 1 && s[1] < (n[0] - 1) * s[0] + block))
      refuse("a cache that is written must not repeat or overlap its sequences or heads");
    for (int j = 0; j < i; ++j)
      if (THPVariable_Unpack(a[j]).data_ptr() == x.data_ptr()) refuse("the arrays of a cache that is written must not be one another");
  }
}

// Contiguous rows of D on 16-byte boundaries; anything else is copied.
struct Rows {
  at::Tensor t;
  long long strides[3];
  explicit Rows(const at::Tensor& x) : t(x) {
    bool ok = t.stride(3) == 1 && (uintptr_t)t.data_ptr() % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
    if (!ok) t = t.clone(at::MemoryFormat::Contiguous);   // contiguous() would keep a contiguous tensor where it is
    for (int i = 0; i < 3; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
  }
};

const int* per_sequence(const at::Tensor& t, int64_t B, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != B || !t.is_contiguous())
    refuse(name, " must be a contiguous int32 tensor [B] = [", B, "]");
  return t.data_ptr<int>();
}

bool ok(int status, const char* what) {
  if (status >= 0) return true;
  PyErr_Format(error_class, "%s: status %d: %s", what, status, lib.error());
  return false;
}

// torch's errors and refusals become Python exceptions; none leaves an entry.
#define BEGIN_CHECKED HANDLE_TH_ERRORS try {
#define END_CHECKED                                             \
  } catch (const Refusal& r) {                                  \
    PyErr_SetString(PyExc_ValueError, r.text.c_str());          \
    return nullptr;                                             \
  }                                                             \
  END_HANDLE_TH_ERRORS

#define NEED_ARGS(n)                                                                    \
  if (!error_class) { PyErr_SetString(PyExc_RuntimeError, "bind() first"); return nullptr; } \
  if (nargs != (n)) { PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", (n), nargs); return nullptr; }

PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 7) { PyErr_SetString(PyExc_TypeError, "bind(error class, six addresses)"); return nullptr; }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i + 1]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib = Library{(decltype(lib.write))p[0], (decltype(lib.read))p[1], (decltype(lib.sdpa_workspace))p[2], (decltype(lib.sdpa))p[3],
                (decltype(lib.logprobs))p[4], (decltype(lib.error))p[5]};
  Py_INCREF(a[0]);
  error_class = a[0];
  Py_RETURN_NONE;
}

PyObject* py_check_cache(PyObject*, PyObject* const* a, Py_ssize_t nargs) {   // the six arrays, on any device; whether they are written
  BEGIN_CHECKED
  const bool written = nargs == 7 && PyObject_IsTrue(a[6]) == 1;
  if (nargs == 7) nargs = 6;
  NEED_ARGS(6)
  cache(a, nullptr);
  if (written) check_apart(a);
  Py_RETURN_NONE;
  END_CHECKED
}

// keys, values, six cache arrays, offsets, counts or None
PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  BEGIN_CHECKED
  NEED_ARGS(10)
  const at::Tensor &keys = tensor(a[0], "keys"), &values = tensor(a[1], "values"), &offsets = tensor(a[8], "offsets");
  const at::Tensor* counts = maybe_tensor(a[9], "counts");
  Device d;
  d.add(&keys); d.add(&values);
  const Cache c = cache(a + 2, &d);
  d.add(&offsets); d.add(counts);
  const Side& k = c.k;
  check_apart(a + 2);
  if (keys.dim() != 4 || keys.sizes() != values.sizes() || keys.size(0) != k.B || keys.size(1) != k.Hk || keys.size(3) != k.D)
    refuse("keys and values must be [B, Hk, T, D] = [", k.B, ", ", k.Hk, ", T, ", k.D, "], got ", keys.sizes(), " and ", values.sizes());
  if (keys.scalar_type() != k.type || values.scalar_type() != k.type) refuse("keys and values must have the cache's dtype ", k.type);
  if (keys.size(2) > INT_MAX) refuse("T beyond 31 bits");
  const int* off = per_sequence(offsets, k.B, "offsets");
  const int* cnt = counts ? per_sequence(*counts, k.B, "counts") : nullptr;
  const c10::cuda::CUDAGuard guard(d.dev);
  const Rows x(keys), y(values);
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = lib.write(x.t.data_ptr(), x.strides, y.t.data_ptr(), y.strides, &c.k.c, &c.v.c, off, cnt, (int)k.B, (int)k.Hk,
                 (int)keys.size(2), (int)k.D, (int)k.cap, dtype_code(k.type), stream);
  Py_END_ALLOW_THREADS
  if (!ok(st, "dflash_kv4_write")) return nullptr;
  Py_RETURN_NONE;
  END_CHECKED
}

// six cache arrays, start (int or tensor), length
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  BEGIN_CHECKED
  NEED_ARGS(8)
  Device d;
  const Cache c = cache(a, &d);
  const Side& k = c.k;
  const int* starts = nullptr;
  int64_t start = 0;
  if (THPVariable_Check(a[6])) {
    const at::Tensor& t = THPVariable_Unpack(a[6]);
    d.add(&t);
    starts = per_sequence(t, k.B, "start");
  } else {
    start = integer(a[6], "start");
    if (start < INT_MIN || start > INT_MAX) refuse("start=", start, " does not fit 32 bits");
  }
  const int64_t length = integer(a[7], "length");
  if (length < 0) refuse("length=", length, " is negative");
  if (length > INT_MAX) refuse("length=", length, " does not fit 32 bits");
  const c10::cuda::CUDAGuard guard(d.dev);
  const auto opt = at::TensorOptions().dtype(k.type).device(d.dev);
  at::Tensor x = at::empty({k.B, k.Hk, length, k.D}, opt), y = at::empty({k.B, k.Hk, length, k.D}, opt);
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = lib.read(&c.k.c, &c.v.c, x.data_ptr(), y.data_ptr(), starts, (int)start, (int)k.B, (int)k.Hk, (int)length, (int)k.D, (int)k.cap,
                dtype_code(k.type), stream);
  Py_END_ALLOW_THREADS
  if (!ok(st, "dflash_kv4_read")) return nullptr;
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(x)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(y)));
  return r;
  END_CHECKED
}

// queries, six cache arrays, scale, lengths (int or tensor), mask or None, max_length or None, num_splits
PyObject* py_sdpa(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  BEGIN_CHECKED
  NEED_ARGS(12)
  const at::Tensor& queries = tensor(a[0], "queries");
  const at::Tensor* mask = maybe_tensor(a[9], "mask");
  Device d;
  d.add(&queries);
  const Cache c = cache(a + 1, &d);
  const Side& k = c.k;
  const double scale = number(a[7], "scale");
  if (!std::isfinite((float)scale)) refuse("scale must be finite, got ", scale);
  if (queries.dim() != 4 || queries.size(0) != k.B || queries.size(3) != k.D || queries.size(1) < 1 || k.Hk < 1 || queries.size(1) % k.Hk)
    refuse("queries must be [B, Hq, T, D] = [", k.B, ", n*", k.Hk, ", T, ", k.D, "], got ", queries.sizes());
  if (queries.scalar_type() != k.type) refuse("queries must have the cache's dtype ", k.type);
  const int64_t Hq = queries.size(1), T = queries.size(2);
  if (T > INT_MAX || Hq > INT_MAX) refuse("queries: sizes beyond 31 bits");
  const int* lengths = nullptr;
  int64_t n_max;
  if (THPVariable_Check(a[8])) {
    const at::Tensor& t = THPVariable_Unpack(a[8]);
    d.add(&t);
    lengths = per_sequence(t, k.B, "lengths");
    n_max = a[10] == Py_None ? k.cap : integer(a[10], "max_length");
  } else {
    n_max = integer(a[8], "lengths");
    if (a[10] != Py_None && integer(a[10], "max_length") != n_max) refuse("max_length goes with lengths on the device");
  }
  if (n_max < 0 || n_max > k.cap) refuse("length ", n_max, " outside 0..", k.cap);
  d.add(mask);
  int kind = 0;
  long long ms[4] = {0, 0, 0, 0};
  at::Tensor m;
  if (mask) {
    kind = mask->scalar_type() == at::kBool ? 1 : mask->scalar_type() == k.type ? 2 : mask->scalar_type() == at::kFloat ? 3 : 0;
    if (!kind) refuse("mask must be bool, ", k.type, " or float32, got ", mask->scalar_type());
    m = mask->expand({k.B, Hq, T, n_max});
    for (int i = 0; i < 4; ++i) ms[i] = m.stride(i);
  }
  const int64_t splits = integer(a[11], "num_splits");
  if (splits < 0 || splits > 1024) refuse("num_splits=", splits, " outside 0..1024");
  const c10::cuda::CUDAGuard guard(d.dev);
  at::Tensor out = at::empty({k.B, Hq, T, k.D}, queries.options());
  if (out.numel() > 0 && n_max == 0) out.zero_();
  if (out.numel() > 0 && n_max > 0) {
    const Rows q(queries);
    const size_t need = lib.sdpa_workspace((int)k.B, (int)Hq, (int)k.Hk, (int)T, (int)k.D, (int)n_max, (int)splits);
    at::Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(d.dev));
    void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = lib.sdpa(q.t.data_ptr(), q.strides, &c.k.c, &c.v.c, mask ? m.data_ptr() : nullptr, kind, ms, out.data_ptr(), lengths, (int)k.B,
                  (int)Hq, (int)k.Hk, (int)T, (int)k.D, (int)k.cap, (int)n_max, (float)scale, dtype_code(k.type), (int)splits,
                  need ? ws.data_ptr() : nullptr, need, stream);
    Py_END_ALLOW_THREADS
    if (!ok(st, "dflash_kv4_sdpa")) return nullptr;
  }
  return THPVariable_Wrap(std::move(out));
  END_CHECKED
}

// logits, tokens, top_k, temperature, suppress or None
PyObject* py_logprobs(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  BEGIN_CHECKED
  NEED_ARGS(5)
  const at::Tensor &logits = tensor(a[0], "logits"), &tokens = tensor(a[1], "tokens");
  const at::Tensor* suppress = maybe_tensor(a[4], "suppress");
  Device d;
  d.add(&logits); d.add(&tokens); d.add(suppress);
  if (logits.dim() < 1) refuse("logits must be [..., V]");
  const int64_t V = logits.size(-1);
  const auto rows = logits.sizes().slice(0, logits.dim() - 1);
  if (tokens.sizes() != rows) refuse("tokens must have logits' leading shape ", rows, ", got ", tokens.sizes());
  if (tokens.scalar_type() != at::kInt && tokens.scalar_type() != at::kLong) refuse("tokens must be int32 or int64, got ", tokens.scalar_type());
  const int code = dtype_code(logits.scalar_type());
  const int64_t k = integer(a[2], "top_k");
  if (V < 1 || k < 0 || k > kMaxTopK || k > V) refuse("top_k=", k, " outside 0..min(", kMaxTopK, ", V=", V, ")");
  const double temperature = number(a[3], "temperature");
  if (!(temperature >= 1e-30 && temperature <= 1e38)) refuse("temperature outside 1e-30..1e38, got ", temperature);
  if (suppress && (suppress->scalar_type() != at::kBool || suppress->dim() != 1 || suppress->size(0) != V))
    refuse("suppress must be a bool tensor [V] = [", V, "]");
  const c10::cuda::CUDAGuard guard(d.dev);
  at::Tensor x = logits, ids = tokens, sup;
  if (x.dim() != 2) x = x.reshape({-1, V});
  if (x.stride(1) != 1 || (x.size(0) > 1 && x.stride(0) < V)) x = x.contiguous();
  const int64_t R = x.size(0);
  if (R > INT_MAX || V > INT_MAX) refuse("logits: sizes beyond 31 bits");
  if (ids.scalar_type() == at::kLong) ids = ids.clamp(-1, V).to(at::kInt);   // ids beyond int32 must not wrap into the vocabulary
  ids = ids.reshape({-1}).contiguous();
  if (suppress) sup = suppress->contiguous();
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(d.dev);
  auto shape = rows.vec();
  at::Tensor lp = at::empty(shape, f32), entropy = at::empty(shape, f32);
  shape.push_back(k);
  at::Tensor tops = at::empty(shape, f32), top_ids = at::empty(shape, f32.dtype(at::kInt));
  void* stream = c10::cuda::getCurrentCUDAStream(d.dev.index()).stream();
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = lib.logprobs(x.data_ptr(), R > 1 ? x.stride(0) : V, ids.data_ptr<int>(), suppress ? (const uint8_t*)sup.data_ptr() : nullptr,
                    (float)temperature, lp.data_ptr<float>(), entropy.data_ptr<float>(), k ? tops.data_ptr<float>() : nullptr,
                    k ? top_ids.data_ptr<int>() : nullptr, (int)R, (int)V, (int)k, code, stream);
  Py_END_ALLOW_THREADS
  if (!ok(st, "dflash_token_logprobs")) return nullptr;
  PyObject* r = PyTuple_New(4);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(lp)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(entropy)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(tops)));
  PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(top_ids)));
  return r;
  END_CHECKED
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)py_bind, METH_FASTCALL, "bind(error class, addresses of the library's functions)"},
    {"check_cache", (PyCFunction)(void*)py_check_cache, METH_FASTCALL, "refuses a cache that the kernels cannot address"},
    {"kv4_write", (PyCFunction)(void*)py_write, METH_FASTCALL, "quantized_kv.quantized_kv_write"},
    {"kv4_read", (PyCFunction)(void*)py_read, METH_FASTCALL, "quantized_kv.quantized_kv_read"},
    {"kv4_sdpa", (PyCFunction)(void*)py_sdpa, METH_FASTCALL, "quantized_kv.quantized_kv_sdpa"},
    {"token_logprobs", (PyCFunction)(void*)py_logprobs, METH_FASTCALL, "logprobs.token_logprobs"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
