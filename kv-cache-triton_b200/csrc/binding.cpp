// Python entry of the operators that branch and trim the cache: tensors to
// kv4_tensor descriptors, outputs and workspace from torch's allocator, the
// current stream of the tensors' device, and the C ABI call, without a Python
// frame for each step (a call through ctypes spends about 40 us on the host for
// ten tensors, this one under 10).
//
// Each function takes what its Python wrapper was given and returns its result;
// None when the arguments are not plainly right (the wrapper then checks them
// one by one and raises), or the status when the library refused.
#include <Python.h>

#include <algorithm>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "kvint4.h"

namespace {

struct NotPlain {};   // the wrapper has to look
struct Status { int rc; };

const at::Tensor &tensor(PyObject *o) {
  if (!THPVariable_Check(o)) throw NotPlain{};
  return THPVariable_Unpack(o);
}
const at::Tensor *maybe(PyObject *o) { return o == Py_None ? nullptr : &tensor(o); }

int64_t whole(PyObject *o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw NotPlain{};
  }
  return v;
}

void need(bool ok) {
  if (!ok) throw NotPlain{};
}
void ok(int rc) {
  if (rc) throw Status{rc};
}

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return KV4_F32;
    case at::kHalf: return KV4_F16;
    case at::kBFloat16: return KV4_BF16;
    case at::kByte:
    case at::kBool: return KV4_U8;
    default: throw NotPlain{};
  }
}

bool is_float(at::ScalarType t) {
  return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
}

kv4_tensor desc(const at::Tensor &t) {
  kv4_tensor d{};
  const int64_t n = t.dim();
  need(n >= 1 && n <= 4);
  const auto sizes = t.sizes(), strides = t.strides();
  for (int64_t i = 0; i < n; ++i) {
    d.shape[4 - n + i] = sizes[i];
    d.stride[4 - n + i] = strides[i];
  }
  for (int64_t i = 3 - n; i >= 0; --i) {
    d.shape[i] = 1;
    d.stride[i] = d.stride[i + 1] * d.shape[i + 1];
  }
  d.dtype = code(t.scalar_type());
  d.data = t.data_ptr();
  return d;
}

void on_device(const at::Tensor &t, const at::Tensor &like) {
  need(t.is_cuda() && t.get_device() == like.get_device());
}

// a written tensor: no expanded view
void written(const at::Tensor &t) {
  for (int64_t i = 0; i < t.dim(); ++i) need(t.size(i) <= 1 || t.stride(i) != 0);
}

// Whether two tensors share a byte (views of one buffer may interleave without
// that).  Distances between two elements are sums of step * x, low <= x <= high;
// the largest steps are tried first, as far as the smaller ones can make up for them.
struct Overlap {
  struct Step { int64_t by, low, high, least, most; };
  Step s[8];
  int n = 0, left = 20000;  // places looked at; strides that nest in no way may need more, and pass
  int64_t a_size, b_size;

  void add(const at::Tensor &t, int64_t sign) {
    for (int64_t i = 0; i < t.dim(); ++i) {
      const int64_t by = t.stride(i) * t.element_size(), high = t.size(i) - 1;
      if (high == 0 || by == 0) continue;
      int k = 0;
      while (k < n && s[k].by != by) ++k;
      if (k == n) s[n++] = Step{by, 0, 0, 0, 0};
      (sign > 0 ? s[k].high : s[k].low) += sign * high;
    }
  }
  bool reach(int i, int64_t at) {
    if (--left < 0) return false;
    if (i == n) return -a_size < at && at < b_size;
    const Step &k = s[i];
    const int64_t by = k.by, to = k.most - at, from = at - k.least;
    const int64_t first = std::max(k.low, -(from >= 0 ? from / by : -((-from + by - 1) / by)));
    const int64_t last = std::min(k.high, to >= 0 ? to / by : -((-to + by - 1) / by));
    for (int64_t x = first; x <= last; ++x)
      if (reach(i + 1, at + by * x)) return true;
    return false;
  }
  bool operator()(const at::Tensor &a, const at::Tensor &b) {
    const auto pa = reinterpret_cast<uintptr_t>(a.data_ptr()), pb = reinterpret_cast<uintptr_t>(b.data_ptr());
    a_size = a.element_size();
    b_size = b.element_size();
    add(a, 1);
    add(b, -1);
    std::sort(s, s + n, [](const Step &x, const Step &y) { return x.by > y.by; });
    int64_t least = 1 - a_size, most = b_size - 1;  // where the elements overlap
    for (int k = n - 1; k >= 0; --k) {
      s[k].least = least;
      s[k].most = most;
      least -= s[k].by * s[k].high;
      most -= s[k].by * s[k].low;
    }
    return reach(0, static_cast<int64_t>(pa - pb));
  }
};
// a tensor and its extent, which tells most of them apart
struct View {
  const at::Tensor *t = nullptr;
  uintptr_t from = 0, to = 0;
  View() = default;
  View(const at::Tensor &x) : t(&x) {
    if (x.numel() == 0) return;
    from = reinterpret_cast<uintptr_t>(x.data_ptr());
    int64_t last = 0;
    const auto sizes = x.sizes(), strides = x.strides();
    for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
    to = from + (last + 1) * x.element_size();
  }
};
bool overlap(const View &a, const View &b) {
  return a.from < b.to && b.from < a.to && Overlap{}(*a.t, *b.t);
}
void apart(const View &a, const View &b) { need(!overlap(a, b)); }

// four tensors of packed K/V rows, [B, Hkv, tokens, ...]
struct Rows {
  const at::Tensor *t[4];
  kv4_tensor d[4];
  View v[4];
  explicit Rows(PyObject *const *a, const at::Tensor *like = nullptr) {
    for (int i = 0; i < 4; ++i) {
      t[i] = &tensor(a[i]);
      need(t[i]->dim() == 4);
      on_device(*t[i], like ? *like : *t[0]);
      need(i & 1 ? is_float(t[i]->scalar_type()) : t[i]->scalar_type() == at::kByte);
    }
    need(t[0]->sizes() == t[2]->sizes() && t[1]->sizes() == t[3]->sizes());
    need(t[1]->scalar_type() == t[3]->scalar_type());
    for (int i = 0; i < 3; ++i) need(t[0]->size(i) == t[1]->size(i));
    for (int i = 0; i < 4; ++i) {
      d[i] = desc(*t[i]);
      v[i] = View(*t[i]);
    }
  }
  bool unit_columns() const {
    for (const at::Tensor *x : t)
      if (x->size(3) > 1 && x->stride(3) != 1) return false;
    return true;
  }
};

// the shape checks every attention call shares
void check_query(const at::Tensor &q, const Rows &c, int64_t n_q, int64_t n_kv, int64_t group) {
  need(group > 0 && n_q > 0 && n_kv > 0 && n_q % n_kv == 0);
  need(q.dim() == 4 && is_float(q.scalar_type()) && q.size(1) == n_q);
  need(c.t[0]->size(0) == q.size(0) && c.t[0]->size(1) == n_kv);
  const int64_t groups = (q.size(3) + group - 1) / group;
  need(c.t[0]->size(3) >= groups * ((group + 1) / 2) && c.t[1]->size(3) >= groups);
}

void check_int32(const at::Tensor &t, const at::Tensor &like) {
  need(t.scalar_type() == at::kInt && t.is_contiguous());
  on_device(t, like);
}

void apart(const View &a, const Rows &rows) {
  for (const View &v : rows.v) apart(a, v);
}
bool same_view(const at::Tensor &a, const at::Tensor &b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// a contiguous tensor on the current device (the guard's), from the caching
// allocator without a pass through the dispatcher (an eviction makes six: 13 -> 11 us a call)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(),
                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

at::Tensor scratch(int64_t bytes) {
  ok(bytes < 0 ? static_cast<int>(-bytes) : 0);
  return fresh({bytes}, at::kByte);
}

void *stream_of(const at::Tensor &t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

PyObject *tree(PyObject *const *a) {
  const at::Tensor &q = tensor(a[0]);
  need(q.is_cuda());
  const Rows cache(a + 1, &q), draft(a + 5, &q);
  const at::Tensor &mask = tensor(a[9]);
  const int64_t n_q = whole(a[10]), n_kv = whole(a[11]), group = whole(a[12]);
  const at::Tensor *lens = maybe(a[13]), *lse = maybe(a[15]);
  check_query(q, cache, n_q, n_kv, group);
  const int64_t b = q.size(0), n = q.size(2);
  for (int i = 0; i < 2; ++i) {
    need(draft.t[i]->size(0) == b && draft.t[i]->size(1) == n_kv && draft.t[i]->size(2) == n &&
         draft.t[i]->size(3) == cache.t[i]->size(3) &&
         draft.t[i]->scalar_type() == cache.t[i]->scalar_type());
  }
  need(mask.scalar_type() == at::kBool && (mask.dim() == 2 || mask.dim() == 3));
  need(mask.size(-1) == n && mask.size(-2) == n && (mask.dim() == 2 || mask.size(0) == b));
  on_device(mask, q);
  if (lens) {
    check_int32(*lens, q);
    need(lens->dim() == 1 && lens->size(0) == b);
  }
  kv4_tensor dl{};
  if (lse) {
    need(lse->scalar_type() == at::kFloat && lse->dim() == 3 && lse->size(0) == b &&
         lse->size(1) == n_q && lse->size(2) == n);
    on_device(*lse, q);
    dl = desc(lse->unsqueeze(-1));
    written(*lse);
    const View v(*lse);
    apart(v, q);
    apart(v, mask);
    if (lens) apart(v, *lens);
    apart(v, cache);
    apart(v, draft);
  }
  const c10::cuda::CUDAGuard guard(q.get_device());
  at::Tensor out;
  if (a[14] == Py_None) {
    out = fresh(q.sizes(), q.scalar_type());
  } else {
    out = tensor(a[14]);
    need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
    on_device(out, q);
    written(out);
    const View v(out);
    if (!same_view(out, q)) apart(v, q);
    apart(v, mask);
    if (lens) apart(v, *lens);
    if (lse) apart(v, *lse);
    apart(v, cache);
    apart(v, draft);
  }
  if (q.numel() == 0) return THPVariable_Wrap(out);
  const kv4_tensor dq = desc(q), dm = desc(mask), dout = desc(out);
  const kv4_tensor *c = cache.d, *f = draft.d;
  const at::Tensor ws = scratch(kv4_tree_workspace(&dq, c, c + 1, c + 2, c + 3, f, f + 1, f + 2, f + 3,
                                                   static_cast<int>(group)));
  ok(kv4_tree_attention(&dq, c, c + 1, c + 2, c + 3, f, f + 1, f + 2, f + 3, &dm,
                        lens ? lens->data_ptr<int32_t>() : nullptr, &dout, lse ? &dl : nullptr,
                        static_cast<int>(group), 0.0f, ws.data_ptr(),
                        static_cast<size_t>(ws.numel()), stream_of(q)));
  return THPVariable_Wrap(out);
}

PyObject *commit(PyObject *const *a) {
  const Rows cache(a), draft(a + 4, cache.t[0]);
  const at::Tensor &k = *cache.t[0], &path = tensor(a[8]), &accepted = tensor(a[9]),
                   &lens = tensor(a[10]);
  need(cache.unit_columns() && draft.unit_columns());
  for (int i = 0; i < 4; ++i)
    need(draft.t[i]->size(0) == cache.t[i]->size(0) && draft.t[i]->size(1) == cache.t[i]->size(1) &&
         draft.t[i]->size(3) == cache.t[i]->size(3) &&
         draft.t[i]->scalar_type() == cache.t[i]->scalar_type());
  const int64_t b = k.size(0);
  check_int32(path, k);
  check_int32(accepted, k);
  check_int32(lens, k);
  need(path.dim() == 2 && path.size(0) == b && accepted.dim() == 1 && accepted.size(0) == b &&
       lens.dim() == 1 && lens.size(0) == b);
  const View read[3] = {path, accepted, lens};
  for (int i = 0; i < 4; ++i) {
    written(*cache.t[i]);
    apart(cache.v[i], draft);
    for (const View &v : read) apart(cache.v[i], v);
  }
  const c10::cuda::CUDAGuard guard(k.get_device());
  at::Tensor out;
  if (a[11] == Py_None) {
    out = fresh(lens.sizes(), lens.scalar_type());
  } else {
    out = tensor(a[11]);
    check_int32(out, k);
    need(out.dim() == 1 && out.size(0) == b);
    const View to(out);
    for (const View &v : read) apart(to, v);
    apart(to, cache);
    apart(to, draft);
  }
  const kv4_tensor *c = cache.d, *f = draft.d;
  ok(kv4_commit_rows(c, c + 1, c + 2, c + 3, f, f + 1, f + 2, f + 3, path.data_ptr<int32_t>(),
                     path.stride(0), path.size(1), accepted.data_ptr<int32_t>(),
                     lens.data_ptr<int32_t>(), out.data_ptr<int32_t>(), stream_of(k)));
  return THPVariable_Wrap(out);
}

PyObject *scored(PyObject *const *a) {
  const at::Tensor &q = tensor(a[0]);
  need(q.is_cuda());
  const Rows cache(a + 1, &q);
  const at::Tensor &mass = tensor(a[5]);
  const int64_t n_q = whole(a[6]), n_kv = whole(a[7]), group = whole(a[8]);
  const int causal = PyObject_IsTrue(a[9]);
  const double decay = PyFloat_AsDouble(a[10]);
  if (causal < 0 || (decay == -1.0 && PyErr_Occurred())) {
    PyErr_Clear();
    throw NotPlain{};
  }
  check_query(q, cache, n_q, n_kv, group);
  auto check_mass = [&](const at::Tensor &m) {
    need(m.scalar_type() == at::kFloat && m.dim() == 3);
    for (int i = 0; i < 3; ++i) need(m.size(i) == cache.t[0]->size(i));
    on_device(m, q);
  };
  check_mass(mass);
  const at::Tensor &to = a[11] == Py_None ? mass : tensor(a[11]);
  check_mass(to);
  written(to);
  const View tv(to);
  if (!same_view(to, mass)) apart(tv, mass);
  apart(tv, q);
  apart(tv, cache);
  const c10::cuda::CUDAGuard guard(q.get_device());
  at::Tensor out;
  if (a[12] == Py_None) {
    out = fresh(q.sizes(), q.scalar_type());
  } else {
    out = tensor(a[12]);
    need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
    on_device(out, q);
    written(out);
    const View v(out);
    for (const at::Tensor *t : {&q, &mass, &to}) apart(v, *t);
    apart(v, cache);
  }
  const kv4_tensor dq = desc(q), din = desc(mass), dto = desc(to), dout = desc(out);
  const kv4_tensor *c = cache.d;
  const at::Tensor ws = scratch(kv4_scored_workspace(&dq, c, c + 1, c + 2, c + 3,
                                                     static_cast<int>(group), causal));
  ok(kv4_scored_attention(&dq, c, c + 1, c + 2, c + 3, &din, &dto, &dout, static_cast<int>(group),
                          causal, static_cast<float>(decay), 0.0f, ws.data_ptr(),
                          static_cast<size_t>(ws.numel()), stream_of(q)));
  PyObject *r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(to));
  return r;
}

PyObject *evict(PyObject *const *a) {
  const Rows cache(a);
  const at::Tensor &k = *cache.t[0], &mass = tensor(a[4]);
  const int64_t keep = whole(a[5]), recent = whole(a[6]), sinks = whole(a[7]);
  const int64_t b = k.size(0), h = k.size(1), s = k.size(2);
  need(recent >= 0 && sinks >= 0 && recent + sinks <= keep && keep <= s && cache.unit_columns());
  need(mass.scalar_type() == at::kFloat && mass.dim() == 3 && mass.size(0) == b &&
       mass.size(1) == h && mass.size(2) == s);
  on_device(mass, k);
  const c10::cuda::CUDAGuard guard(k.get_device());
  at::Tensor out[5];
  if (a[8] == Py_None) {
    for (int i = 0; i < 4; ++i)
      out[i] = fresh({b, h, keep, cache.t[i]->size(3)}, cache.t[i]->scalar_type());
    out[4] = fresh({b, h, keep}, at::kFloat);
  } else {
    need(PyTuple_Check(a[8]) && PyTuple_GET_SIZE(a[8]) == 5);
    for (int i = 0; i < 5; ++i) {
      out[i] = tensor(PyTuple_GET_ITEM(a[8], i));
      const at::Tensor &like = i < 4 ? *cache.t[i] : mass;
      need(out[i].dim() == like.dim() && out[i].scalar_type() == like.scalar_type() &&
           out[i].size(0) == b && out[i].size(1) == h && out[i].size(2) == keep);
      if (i < 4)
        need(out[i].size(3) == like.size(3) && (like.size(3) <= 1 || out[i].stride(3) == 1));
      on_device(out[i], k);
      written(out[i]);
      const View v(out[i]);
      apart(v, cache);
      apart(v, mass);
      for (int j = 0; j < i; ++j) apart(v, out[j]);
    }
  }
  const at::Tensor index = fresh({b, h, keep}, at::kInt);
  kv4_tensor o[5];
  for (int i = 0; i < 5; ++i) o[i] = desc(out[i]);
  const kv4_tensor dm = desc(mass), *c = cache.d;
  ok(kv4_evict(c, c + 1, c + 2, c + 3, &dm, o, o + 1, o + 2, o + 3, o + 4,
               index.data_ptr<int32_t>(), recent, sinks, stream_of(k)));
  PyObject *r = PyTuple_New(6);
  if (!r) return nullptr;
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(out[i]));
  PyTuple_SET_ITEM(r, 5, THPVariable_Wrap(index));
  return r;
}

PyObject *overlaps(PyObject *const *a) { return PyBool_FromLong(overlap(View(tensor(a[0])), View(tensor(a[1])))); }

// No exception leaves a C entry: what the arguments lack is None, what the
// library refuses is its status, anything else (out of memory, ...) a Python error.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments", N);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const NotPlain &) {
    Py_RETURN_NONE;
  } catch (const Status &s) {
    return PyLong_FromLong(s.rc);
  } catch (const c10::OutOfMemoryError &e) {
    PyObject *torch = PyImport_ImportModule("torch");
    PyObject *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject *(*F)(PyObject *const *), int N>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<F, N>)), METH_FASTCALL,
          nullptr};
}

PyMethodDef methods[] = {method<tree, 16>("tree"), method<commit, 12>("commit"),
                         method<scored, 13>("scored"), method<evict, 9>("evict"),
                         method<overlaps, 2>("overlap"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module_def); }
