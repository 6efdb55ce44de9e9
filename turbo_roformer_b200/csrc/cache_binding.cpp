// The Python side of the frame cache (frame_cache.py): checks of tensors, allocation of results and the calls of
// libtrcuda's C ABI (include/trcuda.h), as one extension module.
//
// A push of a few frames takes three calls whose kernels run 3 to 6 us. Reading shapes, types, devices and strides of
// up to nine tensors through Python attributes, and some twenty arguments through ctypes, took 11 to 16 us per call;
// the same here takes 4 to 8 us, the launches included. The library itself stays free of torch types: the module gets the
// addresses of its entry points from the ctypes binding (bind).
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <string>

#include "../../include/trcuda.h"

namespace {

using PlanFn = decltype(&trc_cache_plan);
using AppendFn = decltype(&trc_cache_append);
using WorkspaceFn = decltype(&trc_cache_workspace);
using AttentionFn = decltype(&trc_cache_attention);
PlanFn g_plan = nullptr;
AppendFn g_append = nullptr;
WorkspaceFn g_workspace = nullptr;
AttentionFn g_attention = nullptr;

constexpr int64_t kDim = 64;

// A failed check: becomes Python's ValueError. A failed library call: becomes TRCError through its code.
struct Refused {
  std::string what;
};
struct Failed {
  int64_t rc;
};
void need(bool ok, const char* what) {
  if (!ok) throw Refused{what};
}
void need(bool ok, const char* name, const char* what) {
  if (!ok) throw Refused{std::string(name) + what};
}

// Arguments by position; None where one may be missing.
struct Args {
  PyObject* const* v;
  const at::Tensor& tensor(int i, const char* name) const {
    need(THPVariable_Check(v[i]), name, " must be a tensor");
    return THPVariable_Unpack(v[i]);
  }
  bool none(int i) const { return v[i] == Py_None; }
  int64_t integer(int i, const char* name, int64_t low, int64_t high) const {
    const int64_t x = PyLong_AsLongLong(v[i]);
    if (x == -1 && PyErr_Occurred()) throw python_error();
    need(x >= low && x <= high, name, " out of range");
    return x;
  }
};
constexpr int64_t kInt = INT32_MAX;

// The operators have no backward pass: a result without history in place of a gradient would be silent.
const at::Tensor& plain(const at::Tensor& t, const char* name) {
  need(!(c10::GradMode::is_enabled() && t.requires_grad()), name,
       " requires grad, and the frame cache has no backward pass: call it under torch.no_grad()");
  return t;
}

// Tells autograd that a tensor has new contents.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const int32_t* ints(const at::Tensor& t, int device, int64_t ndim, const char* name) {
  need(t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == device && t.dim() == ndim && t.is_contiguous(), name,
       ndim == 1 ? " must be a contiguous 1-d int32 tensor on the first tensor's device"
                 : " must be a contiguous 2-d int32 tensor on the first tensor's device");
  return t.const_data_ptr<int32_t>();
}

int* status_of(const Args& a, int i, int device) {
  if (a.none(i)) return nullptr;
  const at::Tensor& t = a.tensor(i, "status");
  need(t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == device && t.numel() == 1,
       "status must be an int32 tensor of one element on the first tensor's device");
  return t.data_ptr<int32_t>();
}

int precision_of(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1;
}

struct Pools {
  int64_t pages, heads, page;
};
Pools pools_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& like) {
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == kDim &&
           (k.size(2) == 16 || k.size(2) == 32 || k.size(2) == 64 || k.size(2) == 128),
       "pools must be (pages, cache heads, 16 | 32 | 64 | 128, 64), k and v alike");
  need(k.scalar_type() == like.scalar_type() && v.scalar_type() == like.scalar_type() && k.is_cuda() && v.is_cuda() &&
           k.get_device() == like.get_device() && v.get_device() == like.get_device(),
       "pools must have the other tensors' type and device");
  need(k.is_contiguous() && v.is_contiguous(), "pools must be contiguous");
  need(k.size(0) <= kInt && k.size(1) <= kInt, "pools too large");
  return {k.size(0), k.size(1), k.size(2)};
}

// Elements between rows of a (rows, heads, 64) tensor whose rows are contiguous.
int64_t row_stride(const at::Tensor& t, int64_t rows, int64_t heads, const at::Tensor& like, const char* name) {
  need(t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == kDim &&
           t.scalar_type() == like.scalar_type() && t.is_cuda() && t.get_device() == like.get_device(),
       name, " must be (rows, heads, 64) of the other tensors' type and device");
  need(t.stride(2) == 1 && (heads == 1 || t.stride(1) == kDim), name, ": a row's heads must be contiguous");
  return rows > 1 ? t.stride(0) : heads * kDim;
}

float* gates_of(const at::Tensor& t, int64_t rows, int64_t heads, int device) {
  need(t.dim() == 2 && t.size(0) == rows && t.size(1) == heads && t.scalar_type() == at::kFloat && t.is_cuda() &&
           t.get_device() == device && t.is_contiguous(),
       "gates must be a contiguous (rows, heads) float32 tensor on the first tensor's device");
  return t.data_ptr<float>();
}

// The device is made current for a call (it is put back only where another one was).
struct OnDevice {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit OnDevice(int device) {
    if (c10::cuda::current_device() != device) guard.set_index(device);
    stream = c10::cuda::getCurrentCUDAStream(device).stream();
  }
};

PyObject* steal_tuple(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
  return t;
}
PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// plan(cached, new, table, free_pages, page, max_rows, out | None) -> (cu, total, slots, positions, counts)
PyObject* plan(const Args& a) {
  const at::Tensor& cached = a.tensor(0, "cached");
  need(cached.is_cuda(), "cached must be a CUDA tensor");
  const int device = cached.get_device();
  const int32_t* c = ints(cached, device, 1, "cached");
  const at::Tensor& fresh = a.tensor(1, "new");
  const int32_t* n_new = ints(fresh, device, 1, "new");
  const at::Tensor& table = a.tensor(2, "table");
  ints(table, device, 2, "table");
  const at::Tensor& free_pages = a.tensor(3, "free_pages");
  const int32_t* f = ints(free_pages, device, 1, "free_pages");
  const int64_t n = cached.size(0), columns = table.size(1);
  need(fresh.size(0) == n && table.size(0) == n, "cached, new and table must agree in the number of sequences");
  const int64_t page = a.integer(4, "page", 0, kInt);
  need(page == 16 || page == 32 || page == 64 || page == 128, "page must be 16, 32, 64 or 128");
  const int64_t rows = a.integer(5, "max_rows", 0, kInt);
  need(n <= kInt && columns <= kInt && free_pages.size(0) <= kInt, "plan: too many sequences, columns or pages");
  OnDevice on(device);
  at::Tensor out[5];
  const int64_t sizes[5] = {n + 1, n, rows, rows, 2};
  const char* names[5] = {"cu", "total", "slots", "positions", "counts"};
  int32_t* p[5];
  const bool given = !a.none(6);
  if (given) {
    need(PyTuple_Check(a.v[6]) && PyTuple_GET_SIZE(a.v[6]) == 5, "out must be a CachePlan");
    for (int i = 0; i < 5; ++i) {
      PyObject* o = PyTuple_GET_ITEM(a.v[6], i);
      need(THPVariable_Check(o), names[i], " must be a tensor");
      out[i] = THPVariable_Unpack(o);
      ints(out[i], device, 1, names[i]);
      p[i] = out[i].data_ptr<int32_t>();
      need(out[i].size(0) == sizes[i], names[i], " has the wrong number of elements");
    }
  } else {
    // one allocation for all five, each on a 16-byte boundary
    int64_t at_element = 0, starts[5];
    for (int i = 0; i < 5; ++i) {
      starts[i] = at_element;
      at_element += (sizes[i] + 3) & ~int64_t(3);
    }
    const at::Tensor all = at::empty({at_element}, cached.options());
    for (int i = 0; i < 5; ++i) {
      out[i] = at::detail::make_tensor<at::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
      out[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
      out[i].unsafeGetTensorImpl()->set_storage_offset(starts[i]);
      p[i] = out[i].data_ptr<int32_t>();
    }
  }
  const int rc = g_plan(c, n_new, (int)n, (int)page, f, (int)free_pages.size(0), table.data_ptr<int32_t>(),
                        (int)columns, (int)rows, p[0], p[1], p[2], p[3], p[4], on.stream);
  if (rc) throw Failed{rc};
  written(table);
  if (given) {
    for (const at::Tensor& o : out) written(o);
    return same(a.v[6]);
  }
  return steal_tuple({wrap(out[0]), wrap(out[1]), wrap(out[2]), wrap(out[3]), wrap(out[4])});
}

// append(qkv, positions, slots, k, v, heads, kv_heads, freqs | None, q | None, gates | True | None, status | None)
// -> (q, gates | None)
PyObject* append(const Args& a) {
  const at::Tensor& qkv = plain(a.tensor(0, "qkv"), "qkv");
  const int prec = precision_of(qkv);
  need(qkv.is_cuda() && qkv.dim() == 3 && prec >= 0, "qkv must be a (rows, bands, width) fp16 or bf16 CUDA tensor");
  const int device = qkv.get_device();
  const int64_t rows = qkv.size(0), bands = qkv.size(1), width = qkv.size(2);
  const at::Tensor& k = plain(a.tensor(3, "k_pages"), "k_pages");
  const at::Tensor& v = plain(a.tensor(4, "v_pages"), "v_pages");
  const int64_t heads = a.integer(5, "heads", 1, 4096), kv = a.integer(6, "kv_heads", 1, 4096);
  need(heads % kv == 0, "kv_heads must divide heads");
  const Pools pool = pools_of(k, v, qkv);
  need(bands >= 1 && pool.heads == bands * kv, "the pools must have bands * kv_heads cache heads");
  const bool new_gates = a.v[9] == Py_True, wanted = new_gates || !(a.none(9) || a.v[9] == Py_False);
  need(width >= (heads + 2 * kv) * kDim + (wanted ? heads : 0), "qkv rows too short");
  need(qkv.stride(2) == 1, "qkv: a band's elements must be contiguous");
  const at::Tensor& positions = a.tensor(1, "positions");
  const int32_t* pos = ints(positions, device, 1, "positions");
  const at::Tensor& slots = a.tensor(2, "slots");
  const int32_t* slot = ints(slots, device, 1, "slots");
  need(positions.size(0) >= rows && slots.size(0) >= rows, "positions and slots must cover the rows");
  need(rows <= kInt, "too many rows");
  const float* fr = nullptr;
  if (!a.none(7)) {
    const at::Tensor& freqs = plain(a.tensor(7, "freqs"), "freqs");
    need(freqs.scalar_type() == at::kFloat && freqs.is_cuda() && freqs.get_device() == device && freqs.dim() == 1 &&
             freqs.size(0) == kDim / 2 && freqs.is_contiguous(),
         "freqs must be 32 float32 on the first tensor's device");
    fr = freqs.const_data_ptr<float>();
  }
  int* status = status_of(a, 10, device);
  OnDevice on(device);
  const bool new_q = a.none(8);
  const at::Tensor q = new_q ? at::empty({rows, bands * heads, kDim}, qkv.options()) : plain(a.tensor(8, "q"), "q");
  const int64_t q_stride = row_stride(q, rows, bands * heads, qkv, "q");
  at::Tensor gates;
  float* g = nullptr;
  if (wanted) {
    gates = new_gates ? at::empty({rows, bands * heads}, qkv.options().dtype(at::kFloat))
                      : plain(a.tensor(9, "gates"), "gates");
    g = gates_of(gates, rows, bands * heads, device);
  }
  if (rows) {
    // strides of dimensions of one element say nothing
    const int rc = g_append(prec, qkv.const_data_ptr(), rows > 1 ? qkv.stride(0) : 0, bands > 1 ? qkv.stride(1) : 0,
                            (int)rows, (int)bands, (int)heads, (int)kv, pos, slot, fr, (int)pool.page, (int)pool.pages,
                            q.data_ptr(), q_stride, k.data_ptr(), v.data_ptr(), g, status, on.stream);
    if (rc) throw Failed{rc};
    written(k);
    written(v);
    if (!new_q) written(q);
    if (wanted && !new_gates) written(gates);
  }
  return steal_tuple({new_q ? wrap(q) : same(a.v[8]),
                      !wanted     ? same(Py_None)
                      : new_gates ? wrap(gates)
                                  : same(a.v[9])});
}

// attention(q, k, v, table, cu, total, max_new, max_total, causal, window, scale, gates | None, out | None,
// status | None) -> out
PyObject* attention(const Args& a) {
  const at::Tensor& q = plain(a.tensor(0, "q"), "q");
  const int prec = precision_of(q);
  need(q.is_cuda() && q.dim() == 3 && prec >= 0, "q must be a (rows, heads, 64) fp16 or bf16 CUDA tensor");
  const int device = q.get_device();
  const int64_t rows = q.size(0), heads = q.size(1);
  const at::Tensor& k = plain(a.tensor(1, "k_pages"), "k_pages");
  const at::Tensor& v = plain(a.tensor(2, "v_pages"), "v_pages");
  const Pools pool = pools_of(k, v, q);
  need(q.size(2) == kDim && heads >= 1 && heads <= kInt && pool.heads >= 1 && heads % pool.heads == 0,
       "q must have 64 elements per head, and the cache heads must divide its heads");
  const at::Tensor& table = a.tensor(3, "table");
  const int32_t* t = ints(table, device, 2, "table");
  const at::Tensor& cu = a.tensor(4, "cu");
  const int32_t* c = ints(cu, device, 1, "cu");
  const at::Tensor& total = a.tensor(5, "total");
  const int32_t* tot = ints(total, device, 1, "total");
  const int64_t n = table.size(0), columns = table.size(1);
  need(total.size(0) == n && cu.size(0) == n + 1, "table, cu and total must agree in the number of sequences");
  need(n <= kInt && columns <= kInt && rows <= kInt, "attention: too many sequences, columns or rows");
  const int64_t max_new = a.integer(6, "max_new", -kInt, kInt), max_total = a.integer(7, "max_total", -kInt, kInt);
  const int causal = PyObject_IsTrue(a.v[8]);
  if (causal < 0) throw python_error();
  const int64_t window = a.integer(9, "window", -kInt, kInt);
  const double scale = PyFloat_AsDouble(a.v[10]);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  const int64_t q_stride = row_stride(q, rows, heads, q, "q");
  const float* g = a.none(11) ? nullptr : gates_of(plain(a.tensor(11, "gates"), "gates"), rows, heads, device);
  int* status = status_of(a, 13, device);
  OnDevice on(device);
  const bool new_out = a.none(12);
  const at::Tensor out = new_out ? at::empty({rows, heads, kDim}, q.options()) : plain(a.tensor(12, "out"), "out");
  const int64_t out_stride = row_stride(out, rows, heads, q, "out");
  if (rows) {
    at::Tensor held;  // of the current stream's pool: free for later work on it
    int64_t bytes = 0;
    if (max_total > TRC_CACHE_MAX_WHOLE) {
      bytes = g_workspace((int)max_new, (int)heads, (int)pool.heads);
      if (bytes < 0) throw Failed{bytes};
      held = at::empty({bytes}, q.options().dtype(at::kByte));
    }
    const int rc = g_attention(prec, q.const_data_ptr(), q_stride, k.const_data_ptr(), v.const_data_ptr(), t,
                               (int)columns, c, tot, (int)n, (int)rows, (int)max_new, (int)max_total, (int)heads,
                               (int)pool.heads, (int)pool.page, (int)pool.pages, causal, (int)window, (float)scale, g,
                               out.data_ptr(), out_stride, bytes ? held.data_ptr() : nullptr, bytes, status, on.stream);
    if (rc) throw Failed{rc};
    if (!new_out) written(out);
  }
  return new_out ? wrap(out) : same(a.v[12]);
}

PyObject* g_failed = nullptr;  // called with a library error code: raises

template <PyObject* (*F)(const Args&), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  if (!g_plan) {
    PyErr_SetString(PyExc_RuntimeError, "not bound to the library");
    return nullptr;
  }
  try {
    return F(Args{args});
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.what.c_str());
  } catch (const Failed& f) {
    PyObject* r = PyObject_CallFunction(g_failed, "L", (long long)f.rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "library call failed");
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

// bind(plan, append, workspace, attention, failed): the library's entry points as addresses
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p, ap, w, at;
  PyObject* failed;
  if (!PyArg_ParseTuple(args, "KKKKO", &p, &ap, &w, &at, &failed)) return nullptr;
  g_append = reinterpret_cast<AppendFn>(ap);
  g_workspace = reinterpret_cast<WorkspaceFn>(w);
  g_attention = reinterpret_cast<AttentionFn>(at);
  Py_INCREF(failed);
  Py_XSETREF(g_failed, failed);
  g_plan = reinterpret_cast<PlanFn>(p);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<plan, 7>)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<append, 11>)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<attention, 14>)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_cache_binding", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__cache_binding() { return PyModule_Create(&g_module); }
