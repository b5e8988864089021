// Python binding of the 4-bit cache and page calls (metalbench_b200/kv4.py).
//
// These calls are made once a layer in every decode step, and the smallest of
// them run for a few microseconds on the GPU; checking seven tensors and
// passing twenty arguments through ctypes takes longer than that (13 to 17 us a
// call, against 5 to 8 here). So the checks, the allocations and the call
// itself are made here, on torch's tensors, with the entry points of libmb200
// (include/mb200.h) underneath. Every function returns its tensors, or the
// entry point's negative code as an int, which the Python side turns into its
// MbError; a wrong argument raises TypeError or ValueError.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

#include "../../include/mb200.h"

namespace {

constexpr int64_t DH = 128, PAGE_HEAD = 8704;

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const char* name, const char* what) {
  PyErr_Format(type, "%s: %s", name, what);
  throw Refused();
}

// The tensor behind an argument, of the given type, on CUDA device dev (-1: any).
const at::Tensor& tensor(PyObject* o, const char* name, at::ScalarType type, const char* type_name, int dev) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
    throw Refused();
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != type) {
    PyErr_Format(PyExc_TypeError, "%s: dtype %s is not %s", name, c10::toString(t.scalar_type()), type_name);
    throw Refused();
  }
  if (!t.is_cuda()) refuse(PyExc_ValueError, name, "expected a CUDA tensor (no CPU fallback)");
  if (dev >= 0 && t.get_device() != dev) {
    PyErr_Format(PyExc_ValueError, "%s: expected a tensor on cuda:%d, got one on cuda:%d", name, dev,
                 (int)t.get_device());
    throw Refused();
  }
  return t;
}

[[noreturn]] void bad_shape(const char* name, const char* want, const at::Tensor& t) {
  std::string got = "(", st = "(";
  for (int64_t i = 0; i < t.dim(); ++i) {
    got += (i ? ", " : "") + std::to_string(t.size(i));
    st += (i ? ", " : "") + std::to_string(t.stride(i));
  }
  PyErr_Format(PyExc_ValueError, "%s: expected %s, got shape %s) with strides %s)", name, want, got.c_str(), st.c_str());
  throw Refused();
}

bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A contiguous int32 [n].
int* rows(PyObject* o, const char* name, int dev, int64_t n) {
  const at::Tensor& t = tensor(o, name, at::kInt, "int32", dev);
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    bad_shape(name, ("a contiguous int32 tensor of shape (" + std::to_string(n) + ",)").c_str(), t);
  return t.data_ptr<int>();
}

struct Table {
  int64_t B, M;
  int* p;
};
Table table(PyObject* o, const char* name, int dev) {
  const at::Tensor& t = tensor(o, name, at::kInt, "int32", dev);
  if (t.dim() != 2 || t.size(1) == 0 || !t.is_contiguous() || t.numel() > (1ll << 31) - 1)
    bad_shape(name, "a contiguous block table [B, max_pages >= 1]", t);
  return {t.size(0), t.size(1), t.data_ptr<int>()};
}

struct Cache {
  int64_t P, H;
  int dev;
  uint8_t* p;
};
Cache cache(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name, at::kByte, "uint8", -1);
  if (t.dim() != 3 || t.size(2) != PAGE_HEAD || t.numel() == 0 || !t.is_contiguous() || !aligned(t))
    bad_shape(name, "a contiguous, 16-byte aligned cache [num_pages, n_kv_heads, 8704]", t);
  return {t.size(0), t.size(1), (int)t.get_device(), t.data_ptr<uint8_t>()};
}

// Device and stream of a call; libmb200 is set up on the device first.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  int dev;
  explicit On(int d) : dev(d) {
    static bool ready[64] = {};
    if (c10::cuda::current_device() != d) guard.set_index(d);
    if (d < 64 && ready[d]) return;
    PyObject* m = PyImport_ImportModule("metalbench_b200.ops");
    PyObject* r = m ? PyObject_CallMethod(m, "init", "i", d) : nullptr;
    Py_XDECREF(m);
    Py_XDECREF(r);
    if (!r) throw Refused();
    if (d < 64) ready[d] = true;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
};

// A tensor for results; what `empty` does behind its dispatcher (1 us a call).
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::Tensor(at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}
// Scratch memory of a call on the current stream, given back when the call has
// been launched: the allocator hands it out again in stream order (in a capture:
// it stays the graph's).
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

template <typename F>
int without_gil(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f();
  Py_END_ALLOW_THREADS;
  return rc;
}

#define ENTER(want)                                                                                   \
  HANDLE_TH_ERRORS                                                                                    \
  try {                                                                                               \
    if (n != want) {                                                                                  \
      PyErr_Format(PyExc_TypeError, "%s: expected %d arguments, got %d", __func__, want, (int)n);     \
      return nullptr;                                                                                 \
    }
#define LEAVE                 \
  }                           \
  catch (const Refused&) {    \
    return nullptr;           \
  }                           \
  END_HANDLE_TH_ERRORS

const uint16_t* b16(const at::Tensor& t) { return static_cast<const uint16_t*>(t.data_ptr()); }

// ---- storing and reading back ---------------------------------------------------
struct Tokens {
  const uint16_t* p;
  int64_t S, sb, ss, sh;
};
Tokens tokens(PyObject* o, const char* name, int dev, int64_t B, int64_t H) {
  const at::Tensor& t = tensor(o, name, at::kBFloat16, "bfloat16", dev);
  if (t.dim() != 4 || t.size(0) != B || t.size(2) != H || t.size(3) != DH)
    bad_shape(name, ("[" + std::to_string(B) + ", S, " + std::to_string(H) + ", 128]").c_str(), t);
  // a stride that is never taken may be anything
  const int64_t S = t.size(1), sb = B > 1 ? t.stride(0) : 0, ss = S > 1 ? t.stride(1) : 0, sh = H > 1 ? t.stride(2) : 0;
  if (t.numel() && (t.stride(3) != 1 || (sb | ss | sh) % 8 || !aligned(t)))
    bad_shape(name, "the head dim contiguous and 16-byte aligned, the other strides multiples of 8 elements", t);
  return {b16(t), S, sb, ss, sh};
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(7)
  const Cache c = cache(a[2], "kv4_append(cache)");
  const Table t = table(a[3], "kv4_append(block_table)", c.dev);
  const Tokens k = tokens(a[0], "kv4_append(k)", c.dev, t.B, c.H), v = tokens(a[1], "kv4_append(v)", c.dev, t.B, c.H);
  if (k.S != v.S) refuse(PyExc_ValueError, "kv4_append", "k and v shapes differ");
  const int* start = rows(a[4], "kv4_append(start_pos)", c.dev, t.B);
  const int* len = a[5] == Py_None ? nullptr : rows(a[5], "kv4_append(new_len)", c.dev, t.B);
  const int* most = a[6] == Py_None ? nullptr : rows(a[6], "kv4_append(kv_len)", c.dev, t.B);
  On on(c.dev);
  void* s = on.stream();
  return PyLong_FromLong(without_gil([&] {
    return mb_kv4_append_bf16(k.p, v.p, k.sb, k.ss, k.sh, v.sb, v.ss, v.sh, c.p, (int)c.P, (int)c.H, t.p, (int)t.M,
                              start, len, most, (int)t.B, (int)k.S, s);
  }));
  LEAVE
}

PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(5)
  const Cache c = cache(a[0], "kv4_gather(cache)");
  const Table t = table(a[1], "kv4_gather(block_table)", c.dev);
  const int* start = rows(a[2], "kv4_gather(start_pos)", c.dev, t.B);
  const int64_t S = PyLong_AsLongLong(a[3]);
  if (S == -1 && PyErr_Occurred()) return nullptr;
  if (S < 0 || S > (1ll << 31) - 1) refuse(PyExc_ValueError, "kv4_gather", "length out of range");
  const int* len = rows(a[4], "kv4_gather(kv_len)", c.dev, t.B);
  On on(c.dev);
  at::Tensor k = empty({t.B, S, c.H, DH}, at::kFloat, c.dev), v = empty({t.B, S, c.H, DH}, at::kFloat, c.dev);
  void* s = on.stream();
  const int rc = without_gil([&] {
    return mb_kv4_gather_f32(c.p, (int)c.P, (int)c.H, t.p, (int)t.M, start, len, (int)t.B, (int)S, k.data_ptr<float>(),
                             v.data_ptr<float>(), s);
  });
  if (rc) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  LEAVE
}

// ---- attention ------------------------------------------------------------------
struct Rows {
  int64_t S, H, ld;
};
// [B, S, heads, 128] or [B, heads, 128]: heads contiguous, positions evenly spaced.
Rows query(const at::Tensor& t, const char* name, int64_t B, int64_t H) {
  const bool four = t.dim() == 4;
  if ((t.dim() != 3 && !four) || t.size(0) != B || t.size(-1) != DH || t.size(-2) == 0 || t.size(-2) % H)
    bad_shape(name, ("[" + std::to_string(B) + ", S, heads (a multiple of " + std::to_string(H) + "), 128]").c_str(), t);
  const int64_t S = four ? t.size(1) : 1, heads = t.size(-2), sb = t.stride(0), ss = four ? t.stride(1) : 0;
  const int64_t ld = S > 1 ? ss : B > 1 ? sb : heads * DH;
  if (t.numel() && (t.stride(-1) != 1 || (heads > 1 && t.stride(-2) != DH) || (S > 1 && B > 1 && sb != S * ss) ||
                    ld < heads * DH || ld % 8 || !aligned(t)))
    bad_shape(name, "heads contiguous, positions evenly spaced (a multiple of 8 elements) and 16-byte aligned", t);
  return {S, heads, ld};
}

PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(8)
  const Cache c = cache(a[1], "attention_kv4(cache)");
  const Table t = table(a[2], "attention_kv4(block_table)", c.dev);
  const at::Tensor& q = tensor(a[0], "attention_kv4(q)", at::kBFloat16, "bfloat16", c.dev);
  const Rows r = query(q, "attention_kv4(q)", t.B, c.H);
  const int* len = rows(a[3], "attention_kv4(kv_len)", c.dev, t.B);
  const int* start = a[4] == Py_None ? nullptr : rows(a[4], "attention_kv4(start_pos)", c.dev, t.B);
  double scale = 1.0 / std::sqrt((double)DH);
  if (a[5] != Py_None && (scale = PyFloat_AsDouble(a[5])) == -1.0 && PyErr_Occurred()) return nullptr;
  int64_t most = t.M * 64;
  if (a[7] != Py_None) {
    const int64_t m = PyLong_AsLongLong(a[7]);
    if (m == -1 && PyErr_Occurred()) return nullptr;
    if (m < 1 || m > most) refuse(PyExc_ValueError, "attention_kv4", "max_kv_len must be in [1, 64 block table columns]");
    most = m;
  }
  if (most > (1ll << 30)) refuse(PyExc_ValueError, "attention_kv4", "the block table is too wide");
  On on(c.dev);
  at::Tensor out;
  int64_t ldo = r.H * DH;
  if (a[6] == Py_None) {
    out = empty(q.sizes(), at::kBFloat16, c.dev);
  } else {
    out = tensor(a[6], "attention_kv4(out)", at::kBFloat16, "bfloat16", c.dev);
    if (out.sizes() != q.sizes()) bad_shape("attention_kv4(out)", "q's shape", out);
    ldo = query(out, "attention_kv4(out)", t.B, c.H).ld;
  }
  const size_t nb = mb_attention_kv4_workspace_bytes((int)t.B, (int)r.S, (int)r.H, (int)c.H, (int)most);
  const c10::DataPtr ws = scratch(nb);
  void* s = on.stream();
  const int rc = without_gil([&] {
    return mb_attention_kv4_bf16(b16(q), r.ld, c.p, (int)c.P, t.p, (int)t.M, len, (int)most, start, (int)t.B, (int)r.S, (int)r.H,
                                 (int)c.H, (int)DH, (float)scale, static_cast<uint16_t*>(out.data_ptr()), ldo,
                                 ws.get(), nb, s);
  });
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  LEAVE
}

// ---- pages ------------------------------------------------------------------------
struct Pages {
  Table t;
  int64_t P;
  int dev;
  int *len, *refs;
};
Pages pages(PyObject* tb, PyObject* len, PyObject* refs, const char* name) {
  Pages p;
  p.dev = (int)tensor(tb, name, at::kInt, "int32", -1).get_device();
  p.t = table(tb, name, p.dev);
  const at::Tensor& r = tensor(refs, name, at::kInt, "int32", p.dev);
  if (r.dim() != 1 || !r.is_contiguous() || r.numel() > (1ll << 31) - 1) bad_shape(name, "page_refs [num_pages]", r);
  p.P = r.size(0);
  p.refs = r.data_ptr<int>();
  p.len = rows(len, name, p.dev, p.t.B);
  return p;
}

struct Pools {
  std::vector<void*> ptr;
  std::vector<int64_t> bytes;
};
Pools pools(PyObject* o, const char* name, const Pages& p) {
  Pools r;
  if (THPVariable_Check(o)) refuse(PyExc_TypeError, name, "pools: expected a list of page tensors, got a tensor");
  PyObject* seq = PySequence_Fast(o, "pools: expected a list of page tensors");
  if (!seq) throw Refused();
  struct Drop {
    PyObject* o;
    ~Drop() { Py_DECREF(o); }
  } drop{seq};
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* x = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(x)) refuse(PyExc_TypeError, name, "a pool must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(x);
    if (!t.is_cuda() || t.get_device() != p.dev || t.dim() < 1 || t.size(0) != p.P || !t.is_contiguous())
      bad_shape(name, ("a contiguous pool of " + std::to_string(p.P) + " pages on cuda:" + std::to_string(p.dev)).c_str(), t);
    const int64_t size = p.P ? (int64_t)t.nbytes() / p.P : 16;
    if (size == 0 || size % 16 || !aligned(t))
      bad_shape(name, "a pool whose pages are a multiple of 16 bytes and 16-byte aligned", t);
    uint8_t* at = static_cast<uint8_t*>(t.data_ptr());
    for (size_t k = 0; k < r.ptr.size(); ++k) {
      uint8_t* q = static_cast<uint8_t*>(r.ptr[k]);
      if (p.P && at < q + p.P * r.bytes[k] && q < at + t.nbytes())
        refuse(PyExc_ValueError, name, "the same pool twice, or pools that overlap");
    }
    r.ptr.push_back(at);
    r.bytes.push_back(size);
  }
  return r;
}

c10::DataPtr workspace(const Pages& p, size_t* nb) {
  *nb = mb_kv_pages_workspace_bytes((int)p.t.B, (int)p.t.M, (int)p.P);
  return scratch(*nb);
}

PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(4)
  const Pages p = pages(a[0], a[1], a[2], "kv_pages_extend");
  const int* add = rows(a[3], "kv_pages_extend(new_len)", p.dev, p.t.B);
  On on(p.dev);
  at::Tensor start = empty({p.t.B}, at::kInt, p.dev), status = empty({1}, at::kInt, p.dev);
  size_t nb;
  const c10::DataPtr ws = workspace(p, &nb);
  void* s = on.stream();
  const int rc = without_gil([&] {
    return mb_kv_pages_extend(p.t.p, p.len, p.refs, (int)p.t.B, (int)p.t.M, (int)p.P, add, start.data_ptr<int>(),
                              status.data_ptr<int>(), ws.get(), nb, s);
  });
  if (rc) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(start), THPVariable_Wrap(status));
  LEAVE
}

PyObject* fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(5)
  const Pages p = pages(a[1], a[2], a[3], "kv_pages_fork");
  const int* parent = rows(a[4], "kv_pages_fork(parent)", p.dev, p.t.B);
  const Pools pl = pools(a[0], "kv_pages_fork(pools)", p);
  On on(p.dev);
  at::Tensor status = empty({1}, at::kInt, p.dev);
  size_t nb;
  const c10::DataPtr ws = workspace(p, &nb);
  void* s = on.stream();
  const int rc = without_gil([&] {
    return mb_kv_pages_fork(pl.ptr.data(), pl.bytes.data(), (int)pl.ptr.size(), p.t.p, p.len, p.refs, (int)p.t.B,
                            (int)p.t.M, (int)p.P, parent, status.data_ptr<int>(), ws.get(), nb, s);
  });
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(status);
  LEAVE
}

PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
  ENTER(4)
  const Pages p = pages(a[1], a[2], a[3], "kv_pages_compact");
  const Pools pl = pools(a[0], "kv_pages_compact(pools)", p);
  On on(p.dev);
  at::Tensor remap = empty({p.P}, at::kInt, p.dev), live = empty({1}, at::kInt, p.dev);
  size_t nb;
  const c10::DataPtr ws = workspace(p, &nb);
  void* s = on.stream();
  const int rc = without_gil([&] {
    return mb_kv_pages_compact(pl.ptr.data(), pl.bytes.data(), (int)pl.ptr.size(), p.t.p, p.len, p.refs, (int)p.t.B,
                               (int)p.t.M, (int)p.P, remap.data_ptr<int>(), live.data_ptr<int>(), ws.get(), nb, s);
  });
  if (rc) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(remap), THPVariable_Wrap(live));
  LEAVE
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(append), FAST(gather), FAST(attention), FAST(extend), FAST(fork), FAST(compact),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv4() { return PyModule_Create(&module); }
