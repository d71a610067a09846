// orca_amd._host: the host side of the embedding and gradient-clipping calls (ops.py) for torch tensors.  A call of one of these
// operators on a small batch costs less on the GPU than a Python wrapper spends on taking a few hundred tensors apart (data_ptr,
// numel, dtype, device, contiguity: 230 ns per tensor; 17 ctypes arguments: 3 us); here the tensors are taken apart in C++.  Checks,
// allocation and the current stream only: the work is the C ABI's (include/orca_hip.h), whose entry points setup() receives as
// addresses from the library that _lib.py loaded.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <algorithm>
#include <vector>
#include "../../include/orca_hip.h"

namespace {
decltype(&orca_last_error) last_error;
decltype(&orca_embedding_forward) embedding_forward;
decltype(&orca_embedding_backward_workspace_bytes) backward_workspace_bytes;
decltype(&orca_embedding_backward) embedding_backward_c;
decltype(&orca_embedding_backward_rows) embedding_backward_rows_c;
decltype(&orca_grad_norm_workspace_bytes) grad_norm_workspace_bytes;
decltype(&orca_grad_norm) grad_norm_c;
decltype(&orca_clip_grads) clip_grads_c;
PyObject *orca_error, *row_grad;

struct refusal { PyObject* type; std::string text; };       // becomes that Python exception
template <class... A> [[noreturn]] void refuse(PyObject* type, const A&... a) { throw refusal{type, c10::str(a...)}; }

void check(int rc, const char* who) {
  if (rc == ORCA_OK) return;
  refuse(rc == ORCA_EINVAL ? PyExc_ValueError : rc == ORCA_ERANGE ? PyExc_IndexError : orca_error, who, ": ", last_error());
}
int elem_of(at::ScalarType t) { return t == at::kFloat ? ORCA_F32 : t == at::kBFloat16 ? ORCA_BF16 : t == at::kHalf ? ORCA_F16 : -1; }
const at::ScalarType TYPES[3] = {at::kFloat, at::kBFloat16, at::kHalf};

// a float tensor of the three types on the HIP device
const at::Tensor& elements(PyObject* o, const char* what, int* code) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, what, ": expected a tensor, got ", Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  *code = t.layout() == at::kStrided ? elem_of(t.scalar_type()) : -1;
  if (*code < 0) refuse(PyExc_TypeError, what, ": expected a dense float32, bfloat16 or float16 tensor, got ", t.scalar_type());
  if (!t.is_cuda()) refuse(orca_error, what, ": expected a tensor on the HIP device (no CPU fallback)");
  return t;
}
// one whose memory holds its values (the imaginary part of a conjugated tensor is a view that torch negates when it is read)
const at::Tensor& plain_elements(PyObject* o, const char* what, int* code) {
  const at::Tensor& t = elements(o, what, code);
  if (t.is_neg()) refuse(PyExc_ValueError, what, ": a lazily negated view (resolve_neg() makes a tensor of it)");
  return t;
}
struct id_list {
  at::Tensor t;
  const int64_t* i64 = nullptr;
  const int32_t* i32 = nullptr;
};
id_list ids_of(PyObject* o, c10::Device dev, const char* who) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, who, ": ids must be an int64 or int32 tensor, got ", Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided || (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt))
    refuse(PyExc_TypeError, who, ": ids must be an int64 or int32 tensor, got ", t.scalar_type());
  if (t.device() != dev) refuse(orca_error, who, ": ids are on ", t.device(), ", the rows on ", dev);
  id_list r{t.contiguous()};
  if (t.scalar_type() == at::kLong) r.i64 = r.t.const_data_ptr<int64_t>();
  else r.i32 = r.t.const_data_ptr<int32_t>();
  if (r.t.numel() && !r.i64 && !r.i32) refuse(PyExc_ValueError, who, ": ids have no storage");
  return r;
}
void* stream_of(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse(PyExc_TypeError, "expected ", want, " arguments, got ", n);
}

// A caller's tensor that the kernels write: autograd has to see it (it refuses a backward pass through a value that was saved and then
// changed).  Inference tensors have no version.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The bytes of a strided tensor: runs of `run` bytes, repeated along `outer` (stride in bytes ascending, size at least 2).
struct region {
  const char* p;
  int64_t run;
  c10::SmallVector<std::pair<int64_t, int64_t>, 4> outer;
  const char* end() const {
    int64_t n = run;
    for (const auto& d : outer) n += d.first * (d.second - 1);
    return p + n;
  }
};
region region_of(const at::Tensor& t) {
  region r{(const char*)t.const_data_ptr(), t.numel() ? (int64_t)t.element_size() : 0, {}};
  if (!r.run) return r;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d)) r.outer.emplace_back(t.stride(d) * r.run, t.size(d));
  std::sort(r.outer.begin(), r.outer.end());
  while (!r.outer.empty() && r.outer.front().first <= r.run) {        // (no gap between the repetitions)
    r.run += r.outer.front().first * (r.outer.front().second - 1);
    r.outer.erase(r.outer.begin());
  }
  for (size_t d = 1; d < r.outer.size();) {       // (a dimension that goes on where the one before ends)
    auto& before = r.outer[d - 1];
    if (r.outer[d].first != before.first * before.second) ++d;
    else {
      before.second *= r.outer[d].second;
      r.outer.erase(r.outer.begin() + d);
    }
  }
  return r;
}
// Whether they share a byte.  Views that interleave (column blocks of one matrix) do not.
bool meet(const region& a, const region& b) {
  if (!a.run || !b.run || a.end() <= b.p || b.end() <= a.p) return false;
  if (a.outer.empty() && b.outer.empty()) return true;
  if (a.outer.size() == 1 && b.outer.size() == 1 && a.outer[0].first == b.outer[0].first) {
    // a's run i lies at `at` of the pitch behind the beginning of b's run i + k: it may reach that one and the next
    const int64_t pitch = a.outer[0].first, d = a.p - b.p, k = d >= 0 ? d / pitch : -((-d + pitch - 1) / pitch), at = d - k * pitch;
    auto both = [&](int64_t k) { return std::max<int64_t>(0, -k) <= std::min(a.outer[0].second - 1, b.outer[0].second - 1 - k); };
    return (at < b.run && both(k)) || (at + a.run > pitch && both(k + 1));
  }
  const bool left = !a.outer.empty() && (b.outer.empty() || a.end() - a.p >= b.end() - b.p);        // halve the longer one
  region x = left ? a : b, y = x;
  auto& [stride, size] = x.outer.back();
  y.p += stride * (size / 2);
  y.outer.back().second -= size / 2;
  size /= 2;
  if (size == 1) x.outer.pop_back();
  if (y.outer.back().second == 1) y.outer.pop_back();
  return left ? meet(x, b) || meet(y, b) : meet(a, x) || meet(a, y);
}

// an output that shares memory with an input
void apart(const at::Tensor& out, const at::Tensor& in, const char* who, const char* what) {
  if (meet(region_of(out), region_of(in))) refuse(PyExc_ValueError, who, ": out overlaps ", what);
}

// embedding(table, ids, scale, out)
PyObject* embedding(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 4);
  int code;
  const at::Tensor& table = plain_elements(a[0], "embedding table", &code);
  if (table.dim() != 2) refuse(PyExc_ValueError, "embedding: table has shape ", table.sizes(), ", expected [n_rows, width]");
  const c10::Device dev = table.device();
  const id_list ids = ids_of(a[1], dev, "embedding");
  const int64_t width = table.size(1);
  if (width != 1 && table.stride(1) != 1)
    refuse(PyExc_ValueError, "embedding: the table's columns lie ", table.stride(1), " elements apart (a copy of a table is the caller's to make)");
  const double scale = number(a[2]);
  at::DimVector shape(ids.t.sizes());
  shape.push_back(width);
  const c10::DeviceGuard guard(dev);
  at::Tensor out;
  if (a[3] == Py_None) {
    out = at::empty(shape, table.options().requires_grad(c10::nullopt));
  } else {
    int c;
    out = plain_elements(a[3], "embedding out", &c);
    if (c != code || out.device() != dev || !out.is_contiguous() || out.sizes() != at::IntArrayRef(shape))
      refuse(PyExc_ValueError, "embedding: out must be a contiguous ", table.scalar_type(), " tensor of shape ", at::IntArrayRef(shape), " on ", dev);
    apart(out, table, "embedding", "the table");
    apart(out, ids.t, "embedding", "the ids");
  }
  check(embedding_forward(table.const_data_ptr(), code, table.size(0), width, table.stride(0), ids.i64, ids.i32, ids.t.numel(), (float)scale,
                          out.data_ptr(), stream_of(dev)),
        "orca_embedding_forward");
  if (a[3] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

// what both forms of the gradient take: grad_out, ids, num_rows, scale, padding_idx
struct backward_args {
  at::Tensor g;
  id_list ids;
  int64_t n, width, num_rows, padding;
  int code;
  float scale;
  c10::Device dev{at::kCPU};
};
backward_args backward_of(PyObject* const* a, const char* who) {
  backward_args b;
  const at::Tensor& g = elements(a[0], who, &b.code);
  b.dev = g.device();
  b.ids = ids_of(a[1], b.dev, who);
  if (g.dim() < 1 || g.sizes().slice(0, g.dim() - 1) != b.ids.t.sizes())
    refuse(PyExc_ValueError, who, ": grad_out has shape ", g.sizes(), ", expected ", b.ids.t.sizes(), " and the width");
  b.n = b.ids.t.numel();
  b.width = g.size(-1);
  b.num_rows = integer(a[2]);
  b.scale = (float)number(a[3]);
  b.padding = a[4] == Py_None ? -1 : integer(a[4]);
  // rows one element apart, any row stride (0 included), or a copy
  b.g = (g.dim() == 2 || b.n == 0 || b.width == 0 ? g : g.reshape({b.n, b.width})).resolve_neg();
  if (b.n && b.width > 1 && b.g.stride(-1) != 1) b.g = b.g.contiguous();
  return b;
}
int type_of(PyObject* o, const backward_args& b, const char* who) {        // the output's type: None = the gradient's
  if (o == Py_None) return b.code;
  if (!THPDtype_Check(o)) refuse(PyExc_TypeError, who, ": dtype must be a torch.dtype");
  const int t = elem_of(((THPDtype*)o)->scalar_type);
  if (t != b.code && t != ORCA_F32)
    refuse(PyExc_TypeError, who, ": a ", b.g.scalar_type(), " gradient cannot be returned as ", ((THPDtype*)o)->scalar_type,
           " (its own type, or float32)");
  return t;
}
at::Tensor workspace_of(const backward_args& b, int64_t* bytes, const char* who) {
  *bytes = backward_workspace_bytes(b.n, b.width, b.num_rows);
  if (*bytes < 0) refuse(PyExc_ValueError, who, ": unsupported sizes: ", b.n, " ids, width ", b.width, ", ", b.num_rows, " rows");
  return at::empty({*bytes}, at::TensorOptions(b.dev).dtype(at::kByte));
}

// embedding_backward(grad_out, ids, num_rows, scale, padding_idx, out, accumulate, dtype)
PyObject* embedding_backward(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 8);
  const char* who = "embedding_backward";
  const backward_args b = backward_of(a, who);
  const int accumulate = PyObject_IsTrue(a[6]);
  if (accumulate < 0) throw python_error();
  const c10::DeviceGuard guard(b.dev);
  int64_t bytes;
  const at::Tensor ws = workspace_of(b, &bytes, who);
  at::Tensor out;
  int type;
  if (a[5] == Py_None) {
    if (accumulate) refuse(PyExc_ValueError, "embedding_backward: accumulate needs out");
    type = type_of(a[7], b, who);
    out = at::empty({b.num_rows, b.width}, at::TensorOptions(b.dev).dtype(TYPES[type]));
  } else {
    out = plain_elements(a[5], "embedding_backward out", &type);
    if (out.dim() != 2 || out.size(0) != b.num_rows || out.size(1) != b.width || out.device() != b.dev || (b.width > 1 && out.stride(1) != 1) ||
        (b.num_rows > 1 && out.stride(0) < b.width) || (type != b.code && type != ORCA_F32) || (a[7] != Py_None && type_of(a[7], b, who) != type))
      refuse(PyExc_ValueError, "embedding_backward: out must be a tensor of shape [", b.num_rows, ", ", b.width, "] on ", b.dev,
             " of the gradient's type or float32, whose rows are contiguous and do not overlap");
    apart(out, b.g, who, "grad_out");
    apart(out, b.ids.t, who, "the ids");
  }
  check(embedding_backward_c(b.g.const_data_ptr(), b.code, b.n ? b.g.stride(0) : 0, b.ids.i64, b.ids.i32, b.n, b.width, b.num_rows, b.padding, b.scale,
                             accumulate, out.data_ptr(), type, out.stride(0), ws.data_ptr(), bytes, stream_of(b.dev)),
        "orca_embedding_backward");
  if (a[5] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

// embedding_backward_rows(grad_out, ids, num_rows, scale, padding_idx, out, dtype) -> (ids, rows, count)
PyObject* embedding_backward_rows(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 7);
  const char* who = "embedding_backward_rows";
  const backward_args b = backward_of(a, who);
  const c10::DeviceGuard guard(b.dev);
  int64_t bytes;
  const at::Tensor ws = workspace_of(b, &bytes, who);
  at::Tensor ids, rows, count;
  int type;
  if (a[5] == Py_None) {
    type = type_of(a[6], b, who);
    ids = at::empty({b.n}, at::TensorOptions(b.dev).dtype(at::kLong));
    rows = at::empty({b.n, b.width}, at::TensorOptions(b.dev).dtype(TYPES[type]));
    count = at::empty({1}, at::TensorOptions(b.dev).dtype(at::kInt));
  } else {
    if (!PyTuple_Check(a[5]) || PyTuple_GET_SIZE(a[5]) < 3) refuse(PyExc_TypeError, who, ": out must be (ids, rows, count) or a RowGrad");
    for (int i = 0; i < 3; ++i)
      if (!THPVariable_Check(PyTuple_GET_ITEM(a[5], i))) refuse(PyExc_TypeError, who, ": out must hold tensors");
    ids = THPVariable_Unpack(PyTuple_GET_ITEM(a[5], 0));
    rows = plain_elements(PyTuple_GET_ITEM(a[5], 1), "embedding_backward_rows out", &type);
    count = THPVariable_Unpack(PyTuple_GET_ITEM(a[5], 2));
    if (ids.dim() != 1 || ids.size(0) != b.n || ids.scalar_type() != at::kLong || rows.dim() != 2 || rows.size(0) != b.n || rows.size(1) != b.width ||
        count.dim() != 1 || count.size(0) != 1 || count.scalar_type() != at::kInt || ids.device() != b.dev || rows.device() != b.dev ||
        count.device() != b.dev || !ids.is_contiguous() || !rows.is_contiguous() || (type != b.code && type != ORCA_F32) ||
        (a[6] != Py_None && type_of(a[6], b, who) != type))
      refuse(PyExc_ValueError, who, ": out must be contiguous int64 [", b.n, "], gradient-typed or float32 [", b.n, ", ", b.width,
             "] and int32 [1] tensors on ", b.dev);
    for (const at::Tensor* o : {&ids, &rows, &count}) {
      apart(*o, b.g, who, "grad_out");
      apart(*o, b.ids.t, who, "the ids");
    }
    apart(ids, rows, who, "itself (ids and rows)");
    apart(ids, count, who, "itself (ids and count)");
    apart(rows, count, who, "itself (rows and count)");
  }
  check(embedding_backward_rows_c(b.g.const_data_ptr(), b.code, b.n ? b.g.stride(0) : 0, b.ids.i64, b.ids.i32, b.n, b.width, b.num_rows, b.padding,
                                  b.scale, (int64_t*)ids.data_ptr(), rows.data_ptr(), type, (int32_t*)count.data_ptr(), ws.data_ptr(), bytes,
                                  stream_of(b.dev)),
        "orca_embedding_backward_rows");
  if (a[5] != Py_None)
    for (const at::Tensor* o : {&ids, &rows, &count}) written(*o);
  PyObject* r = PyTuple_New(3);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(ids));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(rows));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(count));
  return r;
}

// a list of tensors, RowGrads and Nones as the host arrays of orca_grad_norm / orca_clip_grads
struct grad_arrays {
  std::vector<void*> data;
  std::vector<const at::Tensor*> tensors;     // the list's own
  std::vector<int64_t> sizes;
  std::vector<uint8_t> types;
  std::vector<const int32_t*> rows;           // empty: none is row-sparse
  std::vector<int32_t> widths;
  std::vector<std::pair<at::Tensor, size_t>> copies;        // contiguous copies, their places in the list
  c10::Device dev{at::kCUDA, (c10::DeviceIndex)-1};
};
grad_arrays grads_of(PyObject* list, const char* who) {
  if (!PyList_Check(list)) refuse(PyExc_TypeError, who, ": expected a list of gradients");
  grad_arrays r;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  r.data.reserve(n);
  r.tensors.reserve(n);
  r.sizes.reserve(n);
  r.types.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (o == Py_None) continue;
    const bool sparse = (PyObject*)Py_TYPE(o) == row_grad;
    const at::Tensor* count = nullptr;
    if (sparse) {
      PyObject* c = PyTuple_GET_ITEM(o, 2);
      if (!THPVariable_Check(c)) refuse(PyExc_TypeError, who, ": a RowGrad's count must be a tensor");
      count = &THPVariable_Unpack(c);
      o = PyTuple_GET_ITEM(o, 1);
    }
    int code;
    const at::Tensor& t = elements(o, who, &code);
    if (r.dev.index() < 0) r.dev = t.device();
    if (t.device() != r.dev) refuse(orca_error, who, ": the gradients must be on one HIP device");
    if (sparse) {
      if (t.dim() != 2 || t.size(1) < 1 || t.size(1) > INT32_MAX || !t.is_contiguous() || t.is_neg() || count->scalar_type() != at::kInt || count->numel() != 1 ||
          count->device() != r.dev)
        refuse(PyExc_ValueError, who, ": a RowGrad needs contiguous [n, width] rows and an int32 count on their device");
      r.rows.resize(r.data.size() + 1, nullptr);
      r.widths.resize(r.data.size() + 1, 0);
      r.rows.back() = count->const_data_ptr<int32_t>();
      r.widths.back() = (int32_t)t.size(1);
    }
    if (t.is_contiguous() && !t.is_neg()) {
      r.data.push_back(t.data_ptr());
    } else {
      r.copies.emplace_back(t.contiguous().resolve_neg(), r.data.size());
      r.data.push_back(r.copies.back().first.data_ptr());
    }
    r.tensors.push_back(&t);
    r.sizes.push_back(t.numel());
    r.types.push_back((uint8_t)code);
  }
  if (!r.rows.empty()) {
    r.rows.resize(r.data.size(), nullptr);
    r.widths.resize(r.data.size(), 0);
  }
  if (r.data.size() > 65536) refuse(PyExc_ValueError, who, ": ", r.data.size(), " gradients (65536 at most)");
  if (r.dev.index() < 0) r.dev = c10::Device(at::kCUDA, c10::hip::current_device());
  return r;
}

// grad_norm(list, max_norm or None) -> norm, or (norm, coefficient)
PyObject* grad_norm(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 2);
  const grad_arrays g = grads_of(a[0], "grad_norm");
  const double max_norm = a[1] == Py_None ? 0.0 : number(a[1]);
  const c10::DeviceGuard guard(g.dev);
  const auto opt = at::TensorOptions(g.dev).dtype(at::kFloat);
  const at::Tensor norm = at::empty({}, opt), coef = a[1] == Py_None ? at::Tensor() : at::empty({}, opt),
                   ws = at::empty({grad_norm_workspace_bytes()}, opt.dtype(at::kByte));
  check(grad_norm_c((int)g.data.size(), g.data.data(), g.sizes.data(), g.types.data(), g.rows.empty() ? nullptr : g.rows.data(), g.widths.data(),
                    max_norm, norm.data_ptr<float>(), coef.defined() ? coef.data_ptr<float>() : nullptr, ws.data_ptr(), stream_of(g.dev)),
        "orca_grad_norm");
  if (!coef.defined()) return THPVariable_Wrap(norm);
  PyObject* r = PyTuple_New(2);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(norm));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(coef));
  return r;
}

// where a tensor's bytes begin and end in its caller's storage
typedef std::pair<const char*, const char*> span;
span span_of(const void* p, int64_t n, int code) { return {(const char*)p, (const char*)p + n * (code == ORCA_F32 ? 4 : 2)}; }
// a list's tensors, the empty ones left out.  `strided`: those that are copied, by their strides (else null, and the span says it all)
struct place { span s; const at::Tensor* strided; };
std::vector<place> places_of(const grad_arrays& g) {
  std::vector<place> r;
  r.reserve(g.data.size());
  size_t next = 0;
  for (size_t i = 0; i < g.data.size(); ++i) {
    const bool copied = next < g.copies.size() && g.copies[next].second == i;
    next += copied;
    if (!g.sizes[i]) continue;
    if (copied) {
      const region q = region_of(*g.tensors[i]);
      r.push_back({{q.p, q.end()}, g.tensors[i]});
    } else {
      r.push_back({span_of(g.data[i], g.sizes[i], g.types[i]), nullptr});
    }
  }
  return r;
}
bool meet(const place& a, const place& b) {
  auto bytes = [](const place& p) { return p.strided ? region_of(*p.strided) : region{p.s.first, p.s.second - p.s.first, {}}; };
  return a.s.first < b.s.second && b.s.first < a.s.second && ((!a.strided && !b.strided) || meet(bytes(a), bytes(b)));
}
constexpr const char* TWICE = ": a tensor is in the list twice, or two of them overlap";
void apart_in_list(std::vector<span> s, const char* who) {
  if (!std::is_sorted(s.begin(), s.end())) std::sort(s.begin(), s.end());
  for (size_t i = 1; i < s.size(); ++i)
    if (s[i].first < s[i - 1].second) refuse(PyExc_ValueError, who, TWICE);
}
void apart_in_list(const grad_arrays& g, const char* who) {
  if (g.copies.empty()) {
    std::vector<span> s;
    s.reserve(g.data.size());
    for (size_t i = 0; i < g.data.size(); ++i)
      if (g.sizes[i]) s.push_back(span_of(g.data[i], g.sizes[i], g.types[i]));
    return apart_in_list(std::move(s), who);
  }
  std::vector<place> all = places_of(g);
  std::sort(all.begin(), all.end(), [](const place& a, const place& b) { return a.s < b.s; });
  std::vector<const place*> open;               // those that reach past the beginning of the next one
  for (const place& x : all) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const place* o) { return o->s.second <= x.s.first; }), open.end());
    for (const place* o : open)
      if (meet(*o, x)) refuse(PyExc_ValueError, who, TWICE);
    open.push_back(&x);
  }
}
void apart_from_list(const std::vector<span>& flat, const grad_arrays& g, const char* who) {
  constexpr const char* text = ": a flat buffer overlaps a gradient";
  if (g.copies.empty()) {
    for (size_t i = 0; i < g.data.size(); ++i) {
      const span r = span_of(g.data[i], g.sizes[i], g.types[i]);
      for (const span& f : flat)
        if (f.first < r.second && r.first < f.second && g.sizes[i]) refuse(PyExc_ValueError, who, text);
    }
    return;
  }
  for (const place& r : places_of(g))
    for (const span& f : flat)
      if (meet(place{f, nullptr}, r)) refuse(PyExc_ValueError, who, text);
}

// clip_grad_norm(list, max_norm, flat buffers or None) -> norm
PyObject* clip_grad_norm(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 3);
  const char* who = "clip_grad_norm";
  const grad_arrays g = grads_of(a[0], who);
  const double max_norm = number(a[1]);
  const c10::DeviceGuard guard(g.dev);
  void* flat[3] = {nullptr, nullptr, nullptr};
  if (a[2] == Py_None) {
    apart_in_list(g, who);
    for (const auto& c : g.copies)
      for (int64_t d = 0; d < g.tensors[c.second]->dim(); ++d)
        if (g.tensors[c.second]->stride(d) == 0 && g.tensors[c.second]->size(d) > 1) refuse(PyExc_ValueError, who, ": an expanded tensor cannot be clipped in place");
  } else {
    if (!PyList_Check(a[2])) refuse(PyExc_TypeError, who, ": flat must be a list of tensors");
    std::vector<int> order;                       // the types as they first appear
    int64_t need[3] = {0, 0, 0};
    std::vector<span> outputs;
    for (size_t i = 0; i < g.data.size(); ++i) {
      const int t = g.types[i];
      if (std::find(order.begin(), order.end(), t) == order.end()) order.push_back(t);
      need[t] += g.sizes[i];
    }
    if (PyList_GET_SIZE(a[2]) != (Py_ssize_t)order.size())
      refuse(PyExc_ValueError, who, ": ", PyList_GET_SIZE(a[2]), " flat buffers for gradients of ", order.size(), " types");
    for (size_t k = 0; k < order.size(); ++k) {
      int code;
      const at::Tensor& f = plain_elements(PyList_GET_ITEM(a[2], k), "clip_grad_norm flat", &code);
      if (code != order[k] || f.numel() != need[code] || f.device() != g.dev || !f.is_contiguous())
        refuse(PyExc_ValueError, who, ": flat buffer ", k, " is not a contiguous ", TYPES[order[k]], " tensor of ", need[order[k]], " elements on ", g.dev);
      flat[code] = f.data_ptr();
      if (f.numel()) outputs.push_back(span_of(f.data_ptr(), f.numel(), code));
    }
    apart_from_list(outputs, g, who);
    apart_in_list(std::move(outputs), who);
  }
  const auto opt = at::TensorOptions(g.dev).dtype(at::kFloat);
  const at::Tensor norm = at::empty({}, opt), ws = at::empty({grad_norm_workspace_bytes()}, opt.dtype(at::kByte));
  check(clip_grads_c((int)g.data.size(), g.data.data(), g.sizes.data(), g.types.data(), g.rows.empty() ? nullptr : g.rows.data(), g.widths.data(), max_norm,
                     a[2] == Py_None ? nullptr : flat, norm.data_ptr<float>(), ws.data_ptr(), stream_of(g.dev)),
        "orca_clip_grads");
  if (a[2] == Py_None) {
    for (const auto& c : g.copies) g.tensors[c.second]->detach().copy_(c.first);
    for (const at::Tensor* t : g.tensors) written(*t);
  } else {
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(a[2]); ++k) written(THPVariable_Unpack(PyList_GET_ITEM(a[2], k)));
  }
  return THPVariable_Wrap(norm);
}

// setup(OrcaError, RowGrad, the addresses of the entry points above in their order)
PyObject* setup(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 10);
  void* f[8];
  for (int i = 0; i < 8; ++i) f[i] = (void*)(uintptr_t)integer(a[2 + i]);
  last_error = (decltype(last_error))f[0];
  embedding_forward = (decltype(embedding_forward))f[1];
  backward_workspace_bytes = (decltype(backward_workspace_bytes))f[2];
  embedding_backward_c = (decltype(embedding_backward_c))f[3];
  embedding_backward_rows_c = (decltype(embedding_backward_rows_c))f[4];
  grad_norm_workspace_bytes = (decltype(grad_norm_workspace_bytes))f[5];
  grad_norm_c = (decltype(grad_norm_c))f[6];
  clip_grads_c = (decltype(clip_grads_c))f[7];
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  orca_error = a[0];
  row_grad = a[1];
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (!orca_error && F != setup) refuse(PyExc_RuntimeError, "orca_amd._host: setup() comes first");
    return F(a, n);
  } catch (const refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))entry<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(setup), ENTRY(embedding), ENTRY(embedding_backward), ENTRY(embedding_backward_rows), ENTRY(grad_norm),
                         ENTRY(clip_grad_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "host side of orca_amd.ops' embedding and clipping calls", -1, methods};
}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
