// Python binding of the residual recurrent block's entry points (include/daydreamer_hip.h): the module
// daydreamer_amd._block.  The rest of the library is bound with ctypes (hipops.py), 0.1 us an argument and 0.8 us
// a checked tensor; a single step of serving is four launches of 4 us kernels, so here the tensors are checked
// and the entry point is called in native code, 0.2 us together.  hipops.HipOps holds the documented methods.
//
// Every function takes (device index, stream, ...) and raises AssertionError for arguments it refuses,
// RuntimeError with dd_last_error()'s text where the library refuses or a launch fails.
#include <Python.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>
#include "../../include/daydreamer_hip.h"

namespace {

#define DD_BLOCK_ENTRIES(X) \
  X(dd_rms_norm_fwd) X(dd_rms_norm_bwd) X(dd_quant_rows) X(dd_linear_fwd) X(dd_linear_act_bwd) \
  X(dd_linear_bwd_data) X(dd_linear_bwd_weight) X(dd_gated_scan_fwd) X(dd_gated_scan_bwd) X(dd_last_error)
#define X(name) decltype(&::name) name##_ = nullptr;
DD_BLOCK_ENTRIES(X)
#undef X

constexpr unsigned F32 = 1u << DD_F32, BF16 = 1u << DD_BF16, E4M3 = 1u << DD_E4M3, REAL = F32 | BF16;

struct Refused {};   // a Python error is set

[[noreturn]] void refuse(const char* format, ...) {
  va_list a;
  va_start(a, format);
  PyErr_FormatV(PyExc_AssertionError, format, a);
  va_end(a);
  throw Refused();
}

const char* names(unsigned types) {
  switch (types) {
    case F32: return "float32";
    case BF16: return "bfloat16";
    case E4M3: return "float8_e4m3fn";
    case REAL: return "float32 or bfloat16";
    case BF16 | E4M3: return "bfloat16 or float8_e4m3fn";
    default: return "float32, bfloat16 or float8_e4m3fn";
  }
}

// Memory of a view: rows of `width` bytes, `step` bytes from one to the next.
struct Span {
  long at = 0, step = 0, width = 0, rows = 0;
  long end() const { return at + (rows - 1) * step + width; }
};
inline long floor_div(long a, long b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); }
// Is there a k in [lo, hi] with low < at + k step < high (all exclusive)?
inline bool any_between(long at, long step, long lo, long hi, long low, long high) {
  if (step == 0) return low < at && at < high;
  return std::max(lo, floor_div(low - at, step) + 1) <= std::min(hi, floor_div(high - at - 1, step));
}
inline bool overlap(const Span& a, const Span& b) {
  if (a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0 || a.end() <= b.at || b.end() <= a.at) return false;
  // rows k of a and j of b share bytes if b.at + j step - a.width < a.at + k step < b.at + j step + b.width
  if (a.step == b.step) return any_between(a.at, a.step, 1 - b.rows, a.rows - 1, b.at - a.width, b.at + b.width);
  const Span &few = a.rows < b.rows ? a : b, &many = a.rows < b.rows ? b : a;
  for (long j = 0; j < few.rows; ++j) {
    const long at = few.at + j * few.step;
    if (any_between(many.at, many.step, 0, many.rows - 1, at - many.width, at + few.width)) return true;
  }
  return false;
}

struct View {
  void* p = nullptr;
  long ld = 0;
  int type = DD_F32;
  Span m;
  unsigned mask() const { return 1u << type; }
  operator Span() const { return m; }
};

const at::Tensor& tensor(PyObject* o, const char* what, int device, unsigned types, int& type) {
  if (!THPVariable_Check(o)) refuse("%s is no tensor", what);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device) refuse("%s is not on device %d", what, device);
  switch (t.scalar_type()) {
    case at::kFloat: type = DD_F32; break;
    case at::kBFloat16: type = DD_BF16; break;
    case at::kFloat8_e4m3fn: type = DD_E4M3; break;
    default: type = 31;
  }
  if (!(types >> type & 1)) refuse("%s has another type than %s", what, names(types));
  if (t.layout() != at::kStrided) refuse("%s is not strided", what);
  return t;
}

struct Args {
  PyObject* const* a;
  int device;
  void* stream;

  bool given(int i) const { return a[i] != Py_None; }
  long number(int i) const {
    const long v = PyLong_AsLong(a[i]);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
  }
  float real(int i) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return (float)v;
  }
  // rows x cols of a 2-D tensor (what the other operands are checked against)
  void shape(int i, const char* what, long& rows, long& cols) const {
    if (!THPVariable_Check(a[i])) refuse("%s is no tensor", what);
    const at::Tensor& t = THPVariable_Unpack(a[i]);
    if (t.dim() != 2) refuse("%s has %d axes, not 2", what, (int)t.dim());
    rows = t.size(0);
    cols = t.size(1);
    if (rows > INT32_MAX || cols > INT32_MAX) refuse("%s is too large", what);
  }
  // a row-major [rows, cols] view: columns next to each other, any row stride of at least cols
  View view(int i, const char* what, long rows, long cols, unsigned types, bool optional = false) const {
    View v;
    if (a[i] == Py_None && optional) return v;
    const at::Tensor& t = tensor(a[i], what, device, types, v.type);
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols) refuse("%s is not [%ld, %ld]", what, rows, cols);
    if (cols > 1 && t.stride(1) != 1) refuse("%s: the columns are strided", what);
    v.p = t.data_ptr();
    v.ld = rows > 1 ? t.stride(0) : std::max<long>(cols, t.stride(0));
    if (v.ld < cols) refuse("%s: rows overlap", what);
    const long es = t.element_size();
    v.m = {(long)(uintptr_t)v.p, rows > 1 ? v.ld * es : 0, cols * es, v.p ? rows : 0};
    return v;
  }
  // n contiguous values
  void* flat(int i, const char* what, long n, unsigned types = F32, bool optional = true, int* type = nullptr) const {
    if (a[i] == Py_None && optional) return nullptr;
    int ty;
    const at::Tensor& t = tensor(a[i], what, device, types, ty);
    if (t.numel() != n || !t.is_contiguous()) refuse("%s: %ld contiguous values are needed", what, n);
    if (type) *type = ty;
    return t.data_ptr();
  }
  int activation(int i) const {
    if (a[i] == Py_None) return DD_ACT_NONE;
    const char* s = PyUnicode_Check(a[i]) ? PyUnicode_AsUTF8(a[i]) : "?";
    const char* known[] = {"none", "elu", "silu", "gelu"};
    for (int k = 0; s && k < 4; ++k)
      if (!strcmp(s, known[k])) return k;
    refuse("act is %R: None, 'none', 'elu', 'silu' or 'gelu'", a[i]);
  }
};

// Contiguous values as a span; NULL: nothing.
Span line(const void* p, long n, int es = 4) { return {(long)(uintptr_t)p, 0, n * es, p ? 1 : 0}; }

// What is written shares no memory with these operands, whose elements other workgroups read or write.
void apart(const Span& out, const char* what, std::initializer_list<Span> operands) {
  for (const Span& o : operands)
    if (overlap(out, o)) refuse("%s shares memory with another operand", what);
}
// ... except with this one if it is the same view: every element is read by the lane, or behind the wait, that writes it.
void apart_or_same(const View& out, const char* what, const View& in) {
  const bool same = out.p == in.p && out.type == in.type && out.m.step == in.m.step && out.m.rows == in.m.rows;
  if (!same && overlap(out, in)) refuse("%s shares memory with an operand that it may be, but is another view of it", what);
}

template <typename F>
void call(const char* name, F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  if (rc == 0) return;
  PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, dd_last_error_());
  throw Refused();
}

template <int N, void (*BODY)(const Args&)>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (!dd_last_error_) refuse("the library is not bound: daydreamer_amd._block.bind(handle)");
    if (n != N + 2) refuse("%d arguments are needed, got %zd", N + 2, n);
    Args args{a + 2, 0, nullptr};
    args.device = (int)PyLong_AsLong(a[0]);
    args.stream = PyLong_AsVoidPtr(a[1]);
    if (PyErr_Occurred()) return nullptr;
    BODY(args);
    Py_RETURN_NONE;
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// x, gamma, y, rstd, res, s, scale, eps
void rms_norm_fwd(const Args& a) {
  long rows, C;
  a.shape(0, "x", rows, C);
  const View x = a.view(0, "x", rows, C, REAL), y = a.view(2, "y", rows, C, REAL | E4M3), r = a.view(4, "res", rows, C, REAL, true);
  const View s = a.view(5, "s", rows, C, r.p || a.given(4) ? r.mask() : REAL, true);
  const int rt = a.given(4) ? r.type : a.given(5) ? s.type : x.type;
  const float* gamma = (const float*)a.flat(1, "gamma", C, F32, false);
  float *rstd = (float*)a.flat(3, "rstd", rows), *scale = (float*)a.flat(6, "scale", rows);
  if ((y.type == DD_E4M3) != a.given(6)) refuse("scale goes with an e4m3 y, and only with it");
  const float eps = a.real(7);
  if (rows == 0) return;
  const Span g = line(gamma, C), inv = line(rstd, rows), sc = line(scale, rows);
  apart(y, "y", {x, r, s, g, inv, sc});
  apart(s, "s", {g, inv, sc});
  apart_or_same(s, "s", x);
  apart_or_same(s, "s", r);
  apart(inv, "rstd", {x, r, g, sc});
  apart(sc, "scale", {x, r, g});
  call("dd_rms_norm_fwd", [&] {
    return dd_rms_norm_fwd_(x.p, x.ld, x.type, r.p, r.ld, rt, s.p, s.ld, gamma, y.p, y.ld, y.type, rstd, scale, (int)rows, (int)C,
                            eps, a.stream);
  });
}

// dy, s, rstd, gamma, ds, dgamma, dres, accumulate, ws, ws_bytes
void rms_norm_bwd(const Args& a) {
  long rows, C;
  a.shape(1, "s", rows, C);
  const View dy = a.view(0, "dy", rows, C, REAL), s = a.view(1, "s", rows, C, REAL), ds = a.view(4, "ds", rows, C, s.mask()),
             dr = a.view(6, "dres", rows, C, s.mask(), true);
  const float *rstd = (const float*)a.flat(2, "rstd", rows, F32, false), *gamma = (const float*)a.flat(3, "gamma", C, F32, false);
  float* dgamma = (float*)a.flat(5, "dgamma", C);
  const Span g = line(gamma, C), dg = line(dgamma, C), inv = line(rstd, rows);
  apart(ds, "ds", {dy, s, g, inv, dg});
  apart_or_same(ds, "ds", dr);
  apart(dg, "dgamma", {dy, s, g, inv, dr});
  const int accumulate = (int)a.number(7);
  float* ws = (float*)a.number(8);
  const size_t bytes = (size_t)a.number(9);
  call("dd_rms_norm_bwd", [&] {
    return dd_rms_norm_bwd_(dy.p, dy.ld, dy.type, s.p, s.ld, s.type, rstd, gamma, dr.p, dr.ld, ds.p, ds.ld, dgamma, accumulate,
                            (int)rows, (int)C, ws, bytes, a.stream);
  });
}

// x, q, scale
void quant_rows(const Args& a) {
  long rows, C;
  a.shape(0, "x", rows, C);
  const View x = a.view(0, "x", rows, C, REAL), q = a.view(1, "q", rows, C, E4M3);
  float* scale = (float*)a.flat(2, "scale", rows, F32, false);
  apart(q, "q", {x, line(scale, rows)});
  apart(line(scale, rows), "scale", {x});
  call("dd_quant_rows", [&] { return dd_quant_rows_(x.p, x.ld, x.type, q.p, q.ld, scale, (int)rows, (int)C, a.stream); });
}

// x, w, y, bias, act, res, z, x_scale, w_scale, ws, ws_bytes
void linear_fwd(const Args& a) {
  long M, K, N, K2;
  a.shape(0, "x", M, K);
  a.shape(1, "w", N, K2);
  const View x = a.view(0, "x", M, K, BF16 | E4M3), w = a.view(1, "w", N, K, x.mask()), y = a.view(2, "y", M, N, REAL),
             r = a.view(5, "res", M, N, y.mask(), true), z = a.view(6, "z", M, N, BF16, true);
  const float* bias = (const float*)a.flat(3, "bias", N);
  const int act = a.activation(4);
  const float *xs = (const float*)a.flat(7, "x_scale", M), *wsc = (const float*)a.flat(8, "w_scale", N);
  if ((x.type == DD_E4M3) != a.given(7) || (x.type == DD_E4M3) != a.given(8))
    refuse("x_scale and w_scale go with e4m3 operands, and only with them");
  float* ws = (float*)a.number(9);
  const size_t bytes = (size_t)a.number(10);
  if (M == 0) return;
  const Span b = line(bias, N), sx = line(xs, M), sw = line(wsc, N);
  apart(y, "y", {x, w, z, b, sx, sw});
  apart_or_same(y, "y", r);
  apart(z, "z", {x, w, r, b, sx, sw});
  call("dd_linear_fwd", [&] {
    return dd_linear_fwd_(x.p, x.ld, w.p, w.ld, x.type, xs, wsc, bias, act, r.p, r.ld, y.p, y.ld, y.type, z.p, z.ld, (int)M,
                          (int)N, (int)K, ws, bytes, a.stream);
  });
}

// dy, x, w, dx, dw, dbias, act, z, dz, accumulate, ws, ws_bytes
void linear_bwd(const Args& a) {
  long M, K, N, K2;
  a.shape(1, "x", M, K);
  a.shape(2, "w", N, K2);
  const View dy = a.view(0, "dy", M, N, BF16), x = a.view(1, "x", M, K, BF16), w = a.view(2, "w", N, K, BF16),
             dx = a.view(3, "dx", M, K, REAL, true), dw = a.view(4, "dw", N, K, REAL, true);
  int bias_type = DD_F32;
  void* db = a.flat(5, "dbias", N, REAL, true, &bias_type);
  const int act = a.activation(6);
  if (act != DD_ACT_NONE && (!a.given(7) || !a.given(8))) refuse("an activation needs z and dz");
  const View z = act == DD_ACT_NONE ? View() : a.view(7, "z", M, N, BF16), dz = act == DD_ACT_NONE ? dy : a.view(8, "dz", M, N, BF16);
  const int accumulate = (int)a.number(9);
  float* ws = (float*)a.number(10);
  const size_t bytes = (size_t)a.number(11);
  const Span b = line(db, N, bias_type == DD_F32 ? 4 : 2);
  if (act != DD_ACT_NONE) {
    apart(dz, "dz", {x, w});
    apart_or_same(dz, "dz", dy);
    apart_or_same(dz, "dz", z);
  }
  apart(dx, "dx", {dy, dz, x, w, dw, b});   // (x: dw reads it behind dx)
  apart(dw, "dw", {dy, dz, x, w, b});
  apart(b, "dbias", {dy, dz, x, w, z});
  if (act != DD_ACT_NONE || db)
    call("dd_linear_act_bwd", [&] {
      return dd_linear_act_bwd_(dy.p, dy.ld, z.p, z.ld, act, dz.p, dz.ld, db, bias_type, accumulate, (int)M, (int)N, ws, bytes, a.stream);
    });
  if (a.given(3))
    call("dd_linear_bwd_data", [&] {
      return dd_linear_bwd_data_(dz.p, dz.ld, w.p, w.ld, dx.p, dx.ld, dx.type, (int)M, (int)N, (int)K, ws, bytes, a.stream);
    });
  if (a.given(4))
    call("dd_linear_bwd_weight", [&] {
      return dd_linear_bwd_weight_(dz.p, dz.ld, x.p, x.ld, dw.p, dw.ld, dw.type, accumulate, (int)M, (int)N, (int)K, ws, bytes, a.stream);
    });
}

// What the scan's directions share: u, c, i, T, first, shift, cand at the given places.
struct Scan {
  long rows, D, T, B, fstride = 0;
  View u, c, i;
  const float* first = nullptr;
  Span restarts;
  float shift;
  int tanh;
  Scan(const Args& a, int at_u, int at_c, int at_i, int at_T, int at_first, int at_shift, int at_cand) {
    a.shape(at_u, "u", rows, D);
    T = a.number(at_T);
    if (T < 1 || rows % T) refuse("%ld rows are no sequences of %ld steps", rows, T);
    B = rows / T;
    u = a.view(at_u, "u", rows, D, REAL);
    c = a.view(at_c, "c", rows, D, u.mask());
    i = a.view(at_i, "i", rows, D, u.mask(), true);
    if (a.given(at_first)) {
      int ty;
      const at::Tensor& t = tensor(a.a[at_first], "first", a.device, F32, ty);
      if (t.dim() != 1 || t.size(0) != rows) refuse("first is not [%ld]", rows);
      first = (const float*)t.data_ptr();
      fstride = rows > 1 ? t.stride(0) : 1;
      restarts = {(long)(uintptr_t)first, fstride * 4, 4, fstride ? rows : 1};
    }
    shift = a.real(at_shift);
    PyObject* cand = a.a[at_cand];
    if (cand != Py_None && !(PyUnicode_Check(cand) && PyUnicode_CompareWithASCIIString(cand, "tanh") == 0))
      refuse("cand is %R: 'tanh' or None", cand);
    tanh = cand != Py_None;
  }
};

// u, c, h, T, i, first, h0, hT, shift, cand, ws, ws_bytes
void gated_scan_fwd(const Args& a) {
  const Scan s(a, 0, 1, 4, 3, 5, 8, 9);
  const View h = a.view(2, "h", s.rows, s.D, s.u.mask());
  const float* h0 = (const float*)a.flat(6, "h0", s.B * s.D);
  float* hT = (float*)a.flat(7, "hT", s.B * s.D);
  const Span from = line(h0, s.B * s.D), to = line(hT, s.B * s.D);
  apart(h, "h", {s.u, s.c, s.i, s.restarts, from, to});
  apart(to, "hT", {s.u, s.c, s.i, s.restarts});
  if (hT != h0) apart(to, "hT", {from});
  float* ws = (float*)a.number(10);
  const size_t bytes = (size_t)a.number(11);
  call("dd_gated_scan_fwd", [&] {
    return dd_gated_scan_fwd_(s.u.p, s.u.ld, s.c.p, s.c.ld, s.i.p, s.i.ld, s.u.type, s.first, s.fstride, h0, h.p, h.ld, hT, (int)s.B,
                              (int)s.T, (int)s.D, s.shift, s.tanh, ws, bytes, a.stream);
  });
}

// dh, u, c, h, du, dc, T, i, di, first, h0, dhT, dh0, shift, cand, ws, ws_bytes
void gated_scan_bwd(const Args& a) {
  const Scan s(a, 1, 2, 7, 6, 9, 13, 14);
  const unsigned m = s.u.mask();
  const View dh = a.view(0, "dh", s.rows, s.D, m), h = a.view(3, "h", s.rows, s.D, m), du = a.view(4, "du", s.rows, s.D, m),
             dc = a.view(5, "dc", s.rows, s.D, m), di = a.view(8, "di", s.rows, s.D, m, true);
  if (a.given(7) != a.given(8)) refuse("di goes with i, and only with it");
  const float *h0 = (const float*)a.flat(10, "h0", s.B * s.D), *dhT = (const float*)a.flat(11, "dhT", s.B * s.D);
  float* dh0 = (float*)a.flat(12, "dh0", s.B * s.D);
  const Span from = line(h0, s.B * s.D), end = line(dhT, s.B * s.D), start = line(dh0, s.B * s.D);
  apart(du, "du", {dh, s.u, s.c, s.i, h, s.restarts, from, end, start, dc, di});
  apart(dc, "dc", {dh, s.u, s.c, s.i, h, s.restarts, from, end, start, di});
  apart(di, "di", {dh, s.u, s.c, s.i, h, s.restarts, from, end, start});
  apart(start, "dh0", {dh, s.u, s.c, s.i, h, s.restarts, from});
  if (dh0 != dhT) apart(start, "dh0", {end});
  float* ws = (float*)a.number(15);
  const size_t bytes = (size_t)a.number(16);
  call("dd_gated_scan_bwd", [&] {
    return dd_gated_scan_bwd_(dh.p, dh.ld, s.u.p, s.u.ld, s.c.p, s.c.ld, s.i.p, s.i.ld, h.p, h.ld, s.u.type, s.first, s.fstride, h0,
                              dhT, du.p, du.ld, dc.p, dc.ld, di.p, di.ld, dh0, (int)s.B, (int)s.T, (int)s.D, s.shift, s.tanh, ws,
                              bytes, a.stream);
  });
}

// bind(handle): the entry points of the library that hipops.load_library() opened and checked
PyObject* bind(PyObject*, PyObject* handle) {
  void* h = PyLong_AsVoidPtr(handle);
  if (PyErr_Occurred()) return nullptr;
#define X(name)                                                                   \
  name##_ = (decltype(&::name))dlsym(h, #name);                                   \
  if (!name##_) { PyErr_SetString(PyExc_RuntimeError, "no " #name " in the library"); return nullptr; }
  DD_BLOCK_ENTRIES(X)
#undef X
  Py_RETURN_NONE;
}

// overlap(at, step, width, rows, at, step, width, rows), in bytes: do two views share memory?
PyObject* share(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long v[8];
  if (n != 8) { PyErr_SetString(PyExc_TypeError, "overlap: 8 numbers are needed"); return nullptr; }
  for (int k = 0; k < 8; ++k) {
    v[k] = PyLong_AsLong(a[k]);
    if (v[k] == -1 && PyErr_Occurred()) return nullptr;
  }
  return PyBool_FromLong(overlap({v[0], v[1], v[2], v[3]}, {v[4], v[5], v[6], v[7]}));
}

#define DD_METHOD(name, n) {#name, (PyCFunction)(void*)entry<n, name>, METH_FASTCALL, nullptr}
PyMethodDef METHODS[] = {
    DD_METHOD(rms_norm_fwd, 8), DD_METHOD(rms_norm_bwd, 10), DD_METHOD(quant_rows, 3), DD_METHOD(linear_fwd, 11),
    DD_METHOD(linear_bwd, 12), DD_METHOD(gated_scan_fwd, 12), DD_METHOD(gated_scan_bwd, 17),
    {"overlap", (PyCFunction)(void*)share, METH_FASTCALL, nullptr}, {"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_block", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block() { return PyModule_Create(&MODULE); }
