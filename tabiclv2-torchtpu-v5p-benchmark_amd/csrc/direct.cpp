// The host side of the paged cache's small calls as a Python module: argument checks, outputs and the call of the C entry
// points in one step. A call of few rows is over in 5 to 10 us on the GPU; the same steps in Python take 12 to 17 us of a host
// core, here 4 to 6 (most of it the launch).
//
// Every function answers None where an argument is anything but the ordinary case (another device than the current one, strides
// that need a copy, a wrong shape or dtype, a refusal by the library): the caller then goes on in Python, which copies,
// switches the device or raises. Callers have made sure that the tensors are plain GPU tensors without gradients.
#include <Python.h>

#include <cstring>

#include <ATen/ATen.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tabicl_attn.h"

namespace {

struct Library {
  decltype(&tabicl_paged_attn_q8) attn_q8;
  decltype(&tabicl_paged_attn_q8_workspace_bytes) attn_q8_ws;
  decltype(&tabicl_paged_sparse_attn) sparse;
  decltype(&tabicl_paged_sparse_attn_workspace_bytes) sparse_ws;
  decltype(&tabicl_paged_append_q8) append_q8;
  decltype(&tabicl_paged_gather_q8) gather_q8;
  decltype(&tabicl_paged_bounds) bounds;
  decltype(&tabicl_paged_select) select;
  decltype(&tabicl_paged_select_workspace_bytes) select_ws;
  decltype(&tabicl_paged_reserve) reserve;
  decltype(&tabicl_paged_release) release;
  decltype(&tabicl_paged_books_workspace_bytes) books_ws;
  decltype(&tabicl_paged_slots) slots;
  decltype(&tabicl_paged_append_slots) append_slots;
} lib;
const char* const NAMES[] = {"tabicl_paged_attn_q8", "tabicl_paged_attn_q8_workspace_bytes", "tabicl_paged_sparse_attn",
                             "tabicl_paged_sparse_attn_workspace_bytes", "tabicl_paged_append_q8", "tabicl_paged_gather_q8",
                             "tabicl_paged_bounds", "tabicl_paged_select", "tabicl_paged_select_workspace_bytes",
                             "tabicl_paged_reserve", "tabicl_paged_release", "tabicl_paged_books_workspace_bytes",
                             "tabicl_paged_slots", "tabicl_paged_append_slots"};
static_assert(sizeof(lib) == sizeof(NAMES), "a name for each function");
bool bound = false;

// bind({name: address}): the functions of the loaded library.
PyObject* bind(PyObject*, PyObject* dict) {
  void* f[sizeof(NAMES) / sizeof(*NAMES)];
  for (size_t i = 0; i < sizeof(NAMES) / sizeof(*NAMES); ++i) {
    PyObject* v = PyDict_Check(dict) ? PyDict_GetItemString(dict, NAMES[i]) : nullptr;
    f[i] = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!f[i]) return PyErr_Format(PyExc_ValueError, "%s: no address", NAMES[i]);
  }
  memcpy((void*)&lib, f, sizeof(lib));
  bound = true;
  Py_RETURN_NONE;
}

const at::Tensor& T(PyObject* o) { return THPVariable_Unpack(o); }
bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
bool tensors(PyObject* const* a, std::initializer_list<int> which) {
  for (int i : which)
    if (!is_tensor(a[i])) return false;
  return true;
}

int current_device() { return c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index(); }

int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kFloat ? 1 : -1; }
int pool_format(const at::Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 ? 0 : s == at::kFloat ? 1 : s == at::kFloat8_e4m3fn ? 2 : s == at::kChar ? 3 : -1;
}

struct Table {
  int64_t N, M, sn;
  const int32_t* p;
  int dev;
  bool read(const at::Tensor& t) {
    if (t.dim() != 2 || t.scalar_type() != at::kInt) return false;
    N = t.size(0), M = t.size(1);
    if (M > 1 && t.stride(1) != 1) return false;
    sn = N > 1 ? t.stride(0) : M;
    p = (const int32_t*)t.data_ptr();
    dev = t.get_device();
    return dev >= 0 && dev == current_device();
  }
  bool list(const at::Tensor& t, int64_t n) const {  // a contiguous int32 list on the table's device
    return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && (n < 2 || t.stride(0) == 1) && t.get_device() == dev;
  }
};

struct Pool {
  int64_t P, H, R, D, sp;
  int format;
  bool read(const at::Tensor& k, const at::Tensor& v, int dev) {
    if (k.dim() != 4) return false;
    P = k.size(0), H = k.size(1), R = k.size(2), D = k.size(3);
    const auto st = k.strides();
    if (st[3] != 1 || st[2] != D || (st[1] != R * D && H > 1)) return false;
    if (k.unsafeGetTensorImpl() != v.unsafeGetTensorImpl() &&
        (v.sizes() != k.sizes() || v.strides() != st || v.scalar_type() != k.scalar_type() || v.get_device() != dev))
      return false;
    sp = P > 1 ? st[0] : H * R * D;
    format = pool_format(k);
    return format >= 0 && k.get_device() == dev;
  }
  // scales of an 8-bit pool, none of another
  bool scaled(PyObject* o, int dev, const float** s) const {
    *s = nullptr;
    if (format < 2) return o == Py_None;
    if (!is_tensor(o)) return false;
    const at::Tensor& t = T(o);
    *s = (const float*)t.data_ptr();
    return t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(0) == P && t.size(1) == H && t.size(2) == 2 && t.is_contiguous() &&
           ((uintptr_t)*s & 7) == 0 && t.get_device() == dev;
  }
};

// Strides of [N, H, T, D] whose rows can be read and written as they are; a dim of one entry counts as stride 0.
struct Rows {
  int64_t n, h, r;
  bool read(const at::Tensor& t, int dev) {
    const auto sz = t.sizes(), st = t.strides();
    n = sz[0] > 1 ? st[0] : 0, h = sz[1] > 1 ? st[1] : 0, r = sz[2] > 1 ? st[2] : 0;
    return (st[3] == 1 || sz[3] == 1) && (((n | h | r) * (int64_t)t.element_size() | (int64_t)(uintptr_t)t.data_ptr()) & 15) == 0 &&
           t.get_device() == dev;
  }
};

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// The interpreter's lock, let go over an allocation and a launch: either may wait for the GPU, and other threads go on meanwhile.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
void* stream_arg(PyObject* o) { return PyLong_AsVoidPtr(o); }

// attn(q, k_pages, v_pages, scales, table, lengths, out, index, scale, stream) -> out; index None: every page (8-bit pools)
PyObject* attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !bound || !tensors(a, {0, 1, 2, 4, 5})) Py_RETURN_NONE;
  const at::Tensor &q = T(a[0]), &k = T(a[1]), &v = T(a[2]), &lengths = T(a[5]);
  Table t;
  Pool p;
  Rows rq, ro;
  const float* scales;
  if (!t.read(T(a[4])) || !p.read(k, v, t.dev) || !p.scaled(a[3], t.dev, &scales) || !t.list(lengths, t.N)) Py_RETURN_NONE;
  const int dt = dtype_code(q);
  if (q.dim() != 4 || dt < 0 || q.size(0) != t.N || q.size(3) != p.D || p.H < 1 || q.size(1) % p.H || !rq.read(q, t.dev)) Py_RETURN_NONE;
  const int64_t Hq = q.size(1), Tq = q.size(2);
  const int32_t* index = nullptr;
  int64_t K = 0;
  if (a[7] == Py_None) {
    if (p.format < 2) Py_RETURN_NONE;
  } else {
    if (!is_tensor(a[7]) || (p.format < 2 && p.format != dt)) Py_RETURN_NONE;
    const at::Tensor& x = T(a[7]);
    if (x.dim() != 4 || x.scalar_type() != at::kInt || x.size(0) != t.N || x.size(1) != p.H || x.size(2) != Tq || !x.is_contiguous() ||
        x.get_device() != t.dev)
      Py_RETURN_NONE;
    index = (const int32_t*)x.data_ptr();
    K = x.size(3);
  }
  const bool make = a[6] == Py_None;
  if (!make) {
    if (!is_tensor(a[6])) Py_RETURN_NONE;
    const at::Tensor& o = T(a[6]);
    if (o.dim() != 4 || o.sizes() != q.sizes() || o.scalar_type() != q.scalar_type() || o.storage().data() == q.storage().data() ||
        !ro.read(o, t.dev) || (t.N > 1 && !ro.n) || (Hq > 1 && !ro.h) || (Tq > 1 && !ro.r))
      Py_RETURN_NONE;
  }
  const float scale = (float)PyFloat_AsDouble(a[8]);
  void* stream = stream_arg(a[9]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t bytes = a[7] != Py_None ? lib.sparse_ws(t.N, Hq, p.H, Tq, p.D, K * p.R)
                                        : lib.attn_q8_ws(t.N, Hq, p.H, Tq, p.D, t.M * p.R, dt);
  if (bytes < 0) Py_RETURN_NONE;
  const bool listed = a[7] != Py_None;
  at::Tensor o, ws;
  if (!make) o = T(a[6]);
  int st;
  {
    Unlocked u;
    if (make) {
      o = at::empty(q.sizes(), q.options());
      ro.read(o, t.dev);
    }
    ws = workspace(bytes, q);
    st = listed
             ? lib.sparse(q.data_ptr(), k.data_ptr(), v.data_ptr(), scales, p.P, p.sp, p.R, t.p, t.sn, t.M,
                          (const int32_t*)lengths.data_ptr(), index, K, o.data_ptr(), t.N, Hq, p.H, Tq, p.D, rq.n, rq.h, rq.r, ro.n, ro.h,
                          ro.r, scale, dt, p.format, pointer(ws), bytes, stream)
             : lib.attn_q8(q.data_ptr(), k.data_ptr(), v.data_ptr(), scales, p.P, p.sp, p.R, t.p, t.sn, t.M,
                          (const int32_t*)lengths.data_ptr(), o.data_ptr(), t.N, Hq, p.H, Tq, p.D, rq.n, rq.h, rq.r, ro.n, ro.h, ro.r,
                          scale, dt, p.format - 2, pointer(ws), bytes, stream);
  }
  if (st) Py_RETURN_NONE;
  if (make) return THPVariable_Wrap(o);
  Py_INCREF(a[6]);
  return a[6];
  END_HANDLE_TH_ERRORS
}

// append(k_pages, v_pages, scales, table, lengths, k, v, count, stream) -> True
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !bound || !tensors(a, {0, 1, 3, 4, 5, 6})) Py_RETURN_NONE;
  const at::Tensor &kp = T(a[0]), &vp = T(a[1]), &lengths = T(a[4]), &k = T(a[5]), &v = T(a[6]);
  Table t;
  Pool p;
  Rows rk, rv;
  const float* scales;
  if (!t.read(T(a[3])) || !p.read(kp, vp, t.dev) || p.format < 2 || !p.scaled(a[2], t.dev, &scales) || !t.list(lengths, t.N))
    Py_RETURN_NONE;
  const int dt = dtype_code(k);
  if (k.dim() != 4 || dt < 0 || v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() || k.size(0) != t.N || k.size(1) != p.H ||
      k.size(3) != p.D || !rk.read(k, t.dev) || !rv.read(v, t.dev))
    Py_RETURN_NONE;
  const int32_t* count = nullptr;
  if (a[7] != Py_None) {
    if (!is_tensor(a[7]) || !t.list(T(a[7]), t.N)) Py_RETURN_NONE;
    count = (const int32_t*)T(a[7]).data_ptr();
  }
  void* stream = stream_arg(a[8]);
  if (PyErr_Occurred()) return nullptr;
  int st;
  {
    Unlocked u;
    st = lib.append_q8(kp.data_ptr(), vp.data_ptr(), (float*)scales, p.P, p.sp, p.R, t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(),
                       k.data_ptr(), v.data_ptr(), count, nullptr, t.N, p.H, k.size(2), p.D, rk.n, rk.h, rk.r, rv.n, rv.h, rv.r, dt,
                       p.format - 2, stream);
  }
  if (st) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// gather(k_pages, v_pages, scales, table, lengths, rows, fp32, stream) -> (k, v)
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !bound || !tensors(a, {0, 1, 3, 4})) Py_RETURN_NONE;
  const at::Tensor &kp = T(a[0]), &vp = T(a[1]), &lengths = T(a[4]);
  Table t;
  Pool p;
  const float* scales;
  if (!t.read(T(a[3])) || !p.read(kp, vp, t.dev) || p.format < 2 || !p.scaled(a[2], t.dev, &scales) || !t.list(lengths, t.N))
    Py_RETURN_NONE;
  const int64_t rows = PyLong_AsLongLong(a[5]);
  const int dt = PyObject_IsTrue(a[6]);
  void* stream = stream_arg(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (rows < 0) Py_RETURN_NONE;
  const auto options = kp.options().dtype(dt ? at::kFloat : at::kBFloat16);
  at::Tensor k, v;
  int st;
  {
    Unlocked u;
    k = at::empty({t.N, p.H, rows, p.D}, options), v = at::empty({t.N, p.H, rows, p.D}, options);
    st = lib.gather_q8(kp.data_ptr(), vp.data_ptr(), scales, p.P, p.sp, p.R, t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(),
                       k.data_ptr(), v.data_ptr(), t.N, p.H, rows, p.D, dt, p.format - 2, stream);
  }
  if (st) Py_RETURN_NONE;
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  END_HANDLE_TH_ERRORS
}

bool bounds_args(const at::Tensor& b, const at::Tensor& s, int64_t P, int64_t H, int64_t D, int dev) {
  return b.scalar_type() == at::kChar && b.dim() == 4 && b.size(0) == P && b.size(1) == H && b.size(2) == 2 && b.size(3) == D &&
         b.is_contiguous() && ((uintptr_t)b.data_ptr() & 15) == 0 && b.get_device() == dev && s.scalar_type() == at::kFloat &&
         s.dim() == 2 && s.size(0) == P && s.size(1) == H && s.is_contiguous() && s.get_device() == dev;
}

// bounds(k_pages, table, lengths, bounds, bound_scales, start, rows, scales, stream) -> True
PyObject* bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !bound || !tensors(a, {0, 1, 2, 3, 4})) Py_RETURN_NONE;
  const at::Tensor &kp = T(a[0]), &lengths = T(a[2]), &b = T(a[3]), &s = T(a[4]);
  Table t;
  Pool p;
  const float* scales;
  if (!t.read(T(a[1])) || !p.read(kp, kp, t.dev) || !p.scaled(a[7], t.dev, &scales) || !t.list(lengths, t.N) ||
      !bounds_args(b, s, p.P, p.H, p.D, t.dev))
    Py_RETURN_NONE;
  const int32_t* start = nullptr;
  if (a[5] != Py_None) {
    if (!is_tensor(a[5]) || !t.list(T(a[5]), t.N)) Py_RETURN_NONE;
    start = (const int32_t*)T(a[5]).data_ptr();
  }
  const int64_t rows = PyLong_AsLongLong(a[6]), most = t.M * p.R;
  void* stream = stream_arg(a[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();  // a number beyond 64 bits
    Py_RETURN_NONE;
  }
  int st;
  {
    Unlocked u;
    st = lib.bounds(kp.data_ptr(), scales, p.P, p.sp, p.R, t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(), start,
                    rows < most ? rows : most, (int8_t*)b.data_ptr(), (float*)s.data_ptr(), t.N, p.H, p.D, p.format, stream);
  }
  if (st) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// select(q, bounds, bound_scales, table, lengths, page_rows, pages, stream) -> index
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !bound || !tensors(a, {0, 1, 2, 3, 4})) Py_RETURN_NONE;
  const at::Tensor &q = T(a[0]), &b = T(a[1]), &s = T(a[2]), &lengths = T(a[4]);
  Table t;
  Rows rq;
  if (!t.read(T(a[3])) || b.dim() != 4 || !t.list(lengths, t.N)) Py_RETURN_NONE;
  const int64_t P = b.size(0), H = b.size(1), D = b.size(3), R = PyLong_AsLongLong(a[5]), K = PyLong_AsLongLong(a[6]);
  void* stream = stream_arg(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const int dt = dtype_code(q);
  if (!bounds_args(b, s, P, H, D, t.dev) || q.dim() != 4 || dt < 0 || q.size(0) != t.N || q.size(3) != D || H < 1 || q.size(1) % H ||
      !rq.read(q, t.dev) || K < 0)
    Py_RETURN_NONE;
  const int64_t Hq = q.size(1), Tq = q.size(2), bytes = lib.select_ws(t.N, H, Tq, t.M);
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor index, ws;
  int st;
  {
    Unlocked u;
    index = at::empty({t.N, H, Tq, K}, q.options().dtype(at::kInt)), ws = workspace(bytes, q);
    st = lib.select(q.data_ptr(), (const int8_t*)b.data_ptr(), (const float*)s.data_ptr(), P, R, t.p, t.sn, t.M,
                    (const int32_t*)lengths.data_ptr(), (int32_t*)index.data_ptr(), K, t.N, Hq, H, Tq, D, rq.n, rq.h, rq.r, dt, pointer(ws),
                    bytes, stream);
  }
  if (st) Py_RETURN_NONE;
  return THPVariable_Wrap(index);
  END_HANDLE_TH_ERRORS
}

bool free_args(const at::Tensor& f, const at::Tensor& c, int dev) {
  return f.scalar_type() == at::kInt && f.dim() == 1 && f.is_contiguous() && f.get_device() == dev && c.scalar_type() == at::kInt &&
         c.numel() == 1 && c.get_device() == dev;
}

// reserve(table, lengths, count, free, free_count, page_rows, stream) -> granted
PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !bound || !tensors(a, {0, 1, 2, 3, 4})) Py_RETURN_NONE;
  const at::Tensor &lengths = T(a[1]), &count = T(a[2]), &f = T(a[3]), &c = T(a[4]);
  Table t;
  if (!t.read(T(a[0])) || !t.list(lengths, t.N) || !t.list(count, t.N) || !free_args(f, c, t.dev)) Py_RETURN_NONE;
  const int64_t R = PyLong_AsLongLong(a[5]), bytes = lib.books_ws(t.N);
  void* stream = stream_arg(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor granted, ws;
  int st;
  {
    Unlocked u;
    granted = at::empty({t.N}, lengths.options()), ws = workspace(bytes, lengths);
    st = lib.reserve((int32_t*)t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(), (const int32_t*)count.data_ptr(),
                     (const int32_t*)f.data_ptr(), (int32_t*)c.data_ptr(), (int32_t*)granted.data_ptr(), f.size(0), R, t.N, pointer(ws),
                     bytes, stream);
  }
  if (st) Py_RETURN_NONE;
  return THPVariable_Wrap(granted);
  END_HANDLE_TH_ERRORS
}

// release(table, lengths, free, free_count, page_rows, stream) -> True
PyObject* release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !bound || !tensors(a, {0, 1, 2, 3})) Py_RETURN_NONE;
  const at::Tensor &lengths = T(a[1]), &f = T(a[2]), &c = T(a[3]);
  Table t;
  if (!t.read(T(a[0])) || !t.list(lengths, t.N) || !free_args(f, c, t.dev)) Py_RETURN_NONE;
  const int64_t R = PyLong_AsLongLong(a[4]), bytes = lib.books_ws(t.N);
  void* stream = stream_arg(a[5]);
  if (PyErr_Occurred()) return nullptr;
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor ws;
  int st;
  {
    Unlocked u;
    ws = workspace(bytes, lengths);
    st = lib.release((int32_t*)t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(), (int32_t*)f.data_ptr(), (int32_t*)c.data_ptr(),
                     f.size(0), R, t.N, pointer(ws), bytes, stream);
  }
  if (st) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// slots(table, lengths, count, total, pages, page_rows, stream) -> (slots, starts)
PyObject* slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !bound || !tensors(a, {0, 1, 2})) Py_RETURN_NONE;
  const at::Tensor &lengths = T(a[1]), &count = T(a[2]);
  Table t;
  if (!t.read(T(a[0])) || !t.list(lengths, t.N) || !t.list(count, t.N)) Py_RETURN_NONE;
  const int64_t total = PyLong_AsLongLong(a[3]), pages = PyLong_AsLongLong(a[4]), R = PyLong_AsLongLong(a[5]);
  void* stream = stream_arg(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (total < 0) Py_RETURN_NONE;
  at::Tensor out, starts;
  int st;
  {
    Unlocked u;
    out = at::empty({total}, lengths.options().dtype(at::kLong)), starts = at::empty({t.N + 1}, lengths.options());
    st = lib.slots(t.p, t.sn, t.M, (const int32_t*)lengths.data_ptr(), (const int32_t*)count.data_ptr(), (int64_t*)out.data_ptr(),
                   (int32_t*)starts.data_ptr(), total, pages, R, t.N, stream);
  }
  if (st) Py_RETURN_NONE;
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(starts));
  END_HANDLE_TH_ERRORS
}

// append_slots(k_pages, v_pages, slots, k, v, stream) -> True
PyObject* append_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !bound || !tensors(a, {0, 1, 2, 3, 4})) Py_RETURN_NONE;
  const at::Tensor &kp = T(a[0]), &vp = T(a[1]), &s = T(a[2]), &k = T(a[3]), &v = T(a[4]);
  const int dev = kp.get_device();
  Pool p;
  if (dev < 0 || dev != current_device() || !p.read(kp, vp, dev) || p.format > 1) Py_RETURN_NONE;
  if (k.dim() != 3 || k.size(1) != p.H || k.size(2) != p.D || v.sizes() != k.sizes() || dtype_code(k) != p.format ||
      dtype_code(v) != p.format || k.get_device() != dev || v.get_device() != dev || s.get_device() != dev || s.dim() != 1 ||
      s.scalar_type() != at::kLong || s.size(0) != k.size(0) || !s.is_contiguous())
    Py_RETURN_NONE;
  int64_t st[2][2];
  const at::Tensor* x[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    const auto& y = *x[i];
    st[i][0] = y.size(0) > 1 ? y.stride(0) : 0, st[i][1] = y.size(1) > 1 ? y.stride(1) : 0;
    if ((y.stride(2) != 1 && y.size(2) > 1) ||
        (((st[i][0] | st[i][1]) * (int64_t)y.element_size() | (int64_t)(uintptr_t)y.data_ptr()) & 15))
      Py_RETURN_NONE;
  }
  void* stream = stream_arg(a[5]);
  if (PyErr_Occurred()) return nullptr;
  int done;
  {
    Unlocked u;
    done = lib.append_slots(kp.data_ptr(), vp.data_ptr(), p.P, p.sp, p.R, (const int64_t*)s.data_ptr(), k.data_ptr(), v.data_ptr(),
                            k.size(0), p.H, p.D, st[0][0], st[0][1], st[1][0], st[1][1], p.format, stream);
  }
  if (done) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

#define FAST(name) \
  { #name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr }
PyMethodDef METHODS[] = {{"bind", bind, METH_O, nullptr}, FAST(attn),    FAST(append),  FAST(gather), FAST(bounds),
                         FAST(select),                    FAST(reserve), FAST(release), FAST(slots),  FAST(append_slots),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "tabicl_mi355_direct", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tabicl_mi355_direct() { return PyModule_Create(&MODULE); }
