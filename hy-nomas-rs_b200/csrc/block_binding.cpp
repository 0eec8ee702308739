// block_binding.cpp — the short way from nomas_kv/block.py into the C ABI: a
// Python extension that takes the plain calls (exact torch tensors on the
// current device, torch's current stream), checks them, allocates the outputs
// that are not given and calls the library.  Whatever is not plain or not
// valid returns None, and block.py's own checks run: they serve the call or
// say what is wrong with it.  A call of a few microseconds of GPU work is bound
// by this path: one token's rotary takes 7 us of host time here, 14 in Python
// (torch's own addition of two rows: 4.6).
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <utility>

#include "nomas_kv.h"

namespace {

// The library's entry points, as block.py's ctypes handle has them.
struct Entries {
  decltype(&nkv_rope_tables) rope_tables = nullptr;
  decltype(&nkv_rotary) rotary = nullptr;
  decltype(&nkv_residual_norm) residual_norm = nullptr;
  decltype(&nkv_attend_packed) attend_packed = nullptr;
} entries;

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NKV_F32;
    case at::kBFloat16: return NKV_BF16;
    case at::kHalf: return NKV_F16;
    default: return -1;
  }
}

int position_code(at::ScalarType t) {
  switch (t) {
    case at::kInt: return NKV_POS_I32;
    case at::kLong: return NKV_POS_I64;
    case at::kFloat: return NKV_POS_F32;
    default: return -1;
  }
}

// The tensors of one call: all on one device, the current one.
struct Tensors {
  int device = c10::cuda::current_device();
  bool grad = c10::GradMode::is_enabled();
  bool ok = true;
  const at::Tensor* optional(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_CheckExact(o)) return refuse();
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.get_device() != device || (grad && t.requires_grad()))
      return refuse();
    return &t;
  }
  const at::Tensor* required(PyObject* o) {
    const at::Tensor* t = optional(o);
    ok &= t != nullptr;
    return t;
  }
  const at::Tensor* refuse() {
    ok = false;
    return nullptr;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream(); }
};

int64_t bytes_of(const at::Tensor& t) {  // from the first element to the end of the last
  if (t.numel() == 0) return 0;
  int64_t n = 1;
  for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  return n * int64_t(t.element_size());
}

// No byte in common: ranges that do not meet, or column blocks beside each
// other in rows of one pitch.
bool apart(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  const char *pa = static_cast<const char*>(a.data_ptr()), *pb = static_cast<const char*>(b.data_ptr());
  if (pa + bytes_of(a) <= pb || pb + bytes_of(b) <= pa) return true;
  if (a.dim() < 1 || b.dim() < 1 || a.size(0) < 2 || b.size(0) < 2) return false;
  const int64_t pitch = a.stride(0) * int64_t(a.element_size());
  if (pitch <= 0 || pitch != b.stride(0) * int64_t(b.element_size())) return false;
  const int64_t ra = bytes_of(a) - (a.size(0) - 1) * pitch, rb = bytes_of(b) - (b.size(0) - 1) * pitch;
  const int64_t d = ((pb - pa) % pitch + pitch) % pitch;
  return ra <= pitch && rb <= pitch && d >= ra && d + rb <= pitch;
}

// A caller's output (object o) for `inputs`: shape and type as given, rows
// dense, no element twice in memory, no byte of an input's but where it is one
// of the `same` inputs itself.
bool output_fits(const at::Tensor& t, PyObject* o, at::IntArrayRef shape, at::ScalarType type,
                 std::initializer_list<std::pair<const at::Tensor*, PyObject*>> inputs, bool may_alias) {
  if (t.sizes() != shape || t.scalar_type() != type) return false;
  if (t.dim() && t.size(-1) > 1 && t.stride(-1) != 1) return false;
  if (!t.is_contiguous()) {
    int64_t need = 1;  // strides that nest, from the last dimension out
    for (int64_t d = t.dim() - 1; d >= 0; --d) {
      if (t.size(d) < 2) continue;
      if (t.stride(d) < need) return false;
      need += t.stride(d) * (t.size(d) - 1);
    }
  }
  for (const auto& in : inputs)
    if (in.first && !(may_alias && in.second == o) && !apart(t, *in.first)) return false;
  return true;
}

PyObject* handed(PyObject* given, at::Tensor& made) {  // a new reference
  if (given == Py_None) return THPVariable_Wrap(std::move(made));
  Py_INCREF(given);
  return given;
}

// A write to a caller's output, counted as torch's in-place operations do: a
// backward pass that saved it raises.
void written(const at::Tensor* given) {
  if (given && !given->is_inference()) given->unsafeGetTensorImpl()->bump_version();
}

void* address(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// A Python number; false (and no error set) if it is none.
bool number(PyObject* o, double* out) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *out = PyFloat_AsDouble(o);
  if (*out == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool eps_of(PyObject* o, float* out) {
  double v;
  if (!number(o, &v) || !(v >= 0.0 && v <= 3.4e38)) return false;
  *out = float(v);
  return true;
}

bool axes_of(PyObject* o, nkv_rope_axes* out) {
  if (!PyBytes_CheckExact(o) || PyBytes_GET_SIZE(o) != Py_ssize_t(sizeof(*out))) return false;
  std::memcpy(out, PyBytes_AS_STRING(o), sizeof(*out));
  return true;
}

bool positions_fit(const at::Tensor& p, int32_t n_axes) {
  return p.dim() == 2 && p.size(1) == n_axes && p.is_contiguous() && position_code(p.scalar_type()) >= 0;
}

// The library's call without the interpreter's lock.
template <typename F>
bool run(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f();
  Py_END_ALLOW_THREADS;
  return rc == NKV_OK;
}

// A call's body; None for whatever it does not take and for any exception (the
// caller's own checks then meet it again).
template <typename F>
PyObject* guarded(F&& f) {
  try {
    if (PyObject* r = f()) return r;
  } catch (...) {
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyObject* pair_of(PyObject* a, PyObject* b) {  // takes both references
  PyObject* r = a && b ? PyTuple_New(2) : nullptr;
  if (!r) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(r, 0, a);
  PyTuple_SET_ITEM(r, 1, b);
  return r;
}

// bind(rope_tables, rotary, residual_norm, attend_packed): their addresses.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[4];
  if (n != 4) return PyErr_Format(PyExc_TypeError, "four addresses expected");
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "null address");
  }
  entries.rope_tables = reinterpret_cast<decltype(entries.rope_tables)>(p[0]);
  entries.rotary = reinterpret_cast<decltype(entries.rotary)>(p[1]);
  entries.residual_norm = reinterpret_cast<decltype(entries.residual_norm)>(p[2]);
  entries.attend_packed = reinterpret_cast<decltype(entries.attend_packed)>(p[3]);
  Py_RETURN_NONE;
}

// rope_tables(axes, positions, cos, sin) -> (cos, sin)
PyObject* rope_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    nkv_rope_axes axes;
    if (n != 4 || !entries.rope_tables || !axes_of(a[0], &axes)) return nullptr;
    Tensors in;
    const at::Tensor *pos = in.required(a[1]), *given[2] = {in.optional(a[2]), in.optional(a[3])};
    if (!in.ok || !positions_fit(*pos, axes.n_axes)) return nullptr;
    int64_t pairs = 0;
    for (int i = 0; i < axes.n_axes && i < 4; ++i) pairs += axes.dims[i] / 2;
    const auto opt = pos->options().dtype(at::kFloat);
    const int64_t shape[2] = {pos->size(0), pairs};
    at::Tensor made[2];
    float* to[2];
    for (int i = 0; i < 2; ++i) {
      if (given[i] && (!given[i]->is_contiguous() ||
                       !output_fits(*given[i], a[2 + i], shape, at::kFloat, {{pos, a[1]}, {given[1 - i], a[3 - i]}}, false)))
        return nullptr;
      if (!given[i]) made[i] = at::empty(shape, opt);
      to[i] = static_cast<float*>((given[i] ? *given[i] : made[i]).data_ptr());
    }
    void* st = in.stream();
    const void* p = pos->data_ptr();
    if (!run([&] {
          return entries.rope_tables(&axes, p, position_code(pos->scalar_type()), uint64_t(pos->size(0)), to[0], to[1],
                                     st);
        }))
      return nullptr;
    written(given[0]), written(given[1]);
    return pair_of(handed(a[2], made[0]), handed(a[3], made[1]));
  });
}

// rotary(axes, positions, q, k, norm, q_weight, k_weight, eps, q_out, k_out) ->
// q_out or (q_out, k_out)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    nkv_rotary_args r{};
    if (n != 10 || !entries.rotary || !axes_of(a[0], &r.axes) || !PyBool_Check(a[4]) || !eps_of(a[7], &r.eps))
      return nullptr;
    Tensors in;
    const at::Tensor *pos = in.required(a[1]), *q = in.required(a[2]), *k = in.optional(a[3]),
                     *qw = in.optional(a[5]), *kw = in.optional(a[6]), *qo = in.optional(a[8]),
                     *ko = in.optional(a[9]);
    if (!in.ok || q->dim() != 3 || !positions_fit(*pos, r.axes.n_axes)) return nullptr;
    const int64_t tokens = q->size(0), D = q->size(2);
    const int code = type_code(q->scalar_type());
    if (code < 0 || D < 2 || D > 256 || pos->size(0) != tokens || q->stride(2) != 1) return nullptr;
    if (k && (k->dim() != 3 || k->size(0) != tokens || k->size(2) != D || k->scalar_type() != q->scalar_type() ||
              k->stride(2) != 1))
      return nullptr;
    r.norm = a[4] == Py_True;
    if ((!r.norm && (qw || kw)) || (!k && (kw || ko))) return nullptr;
    // (q and k one tensor: read as both, so neither may be rotated in place)
    const bool in_place = a[2] != a[3];
    if (qo && (!output_fits(*qo, a[8], q->sizes(), q->scalar_type(), {{pos, a[1]}, {q, a[2]}, {qw, a[5]}, {kw, a[6]}},
                            in_place) ||
               (k && !apart(*qo, *k)) || (ko && !apart(*qo, *ko))))
      return nullptr;
    if (ko && (!output_fits(*ko, a[9], k->sizes(), k->scalar_type(), {{pos, a[1]}, {k, a[3]}, {qw, a[5]}, {kw, a[6]}},
                            in_place) ||
               !apart(*ko, *q)))
      return nullptr;
    for (const at::Tensor* w : {qw, kw})
      if (w && (w->dim() != 1 || w->size(0) != D || w->scalar_type() != q->scalar_type() || !w->is_contiguous()))
        return nullptr;
    at::Tensor out[2];
    auto side = [&](const at::Tensor& t, const at::Tensor* w, const at::Tensor* given, at::Tensor& made) {
      if (!given) made = at::empty(t.sizes(), t.options());
      const at::Tensor& o = given ? *given : made;
      return nkv_rotary_side{t.data_ptr(), o.data_ptr(), t.stride(0), t.stride(1), o.stride(0), o.stride(1), address(w),
                             int32_t(t.size(1))};
    };
    if (q->size(1) > 65535 || (k && k->size(1) > 65535)) return nullptr;
    r.positions = pos->data_ptr();
    r.position_type = position_code(pos->scalar_type());
    r.dtype = code;
    r.tokens = uint64_t(tokens);
    r.head_dim = int32_t(D);
    r.q = side(*q, qw, qo, out[0]);
    if (k) r.k = side(*k, kw, ko, out[1]);
    void* st = in.stream();
    if (!run([&] { return entries.rotary(&r, st); })) return nullptr;
    written(qo), written(ko);
    PyObject* first = handed(a[8], out[0]);
    return k ? pair_of(first, handed(a[9], out[1])) : first;
  });
}

// residual_norm(x, branch, gate, post, post_weight, norm, weight, scale, shift,
// mod_index, eps, h_out, y_out) -> (h, y); post and norm as nkv_norm_kind
PyObject* residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    nkv_residual_norm_args r{};
    if (n != 13 || !entries.residual_norm || !PyLong_CheckExact(a[3]) || !PyLong_CheckExact(a[5]) ||
        !eps_of(a[10], &r.eps))
      return nullptr;
    r.post = int32_t(PyLong_AsLong(a[3]));
    r.norm = int32_t(PyLong_AsLong(a[5]));
    Tensors in;
    const at::Tensor *x = in.required(a[0]), *branch = in.optional(a[1]), *index = in.optional(a[9]),
                     *ho = in.optional(a[11]), *yo = in.optional(a[12]);
    const at::Tensor* mods[3] = {in.optional(a[2]), in.optional(a[7]), in.optional(a[8])};  // gate, scale, shift
    const at::Tensor* weights[2] = {in.optional(a[4]), in.optional(a[6])};                  // post's, norm's
    if (!in.ok || x->dim() != 2) return nullptr;
    const int64_t tokens = x->size(0), dim = x->size(1);
    const at::ScalarType type = x->scalar_type();
    const int code = type_code(type);
    auto dense_rows = [&](const at::Tensor& t) { return dim <= 1 || t.stride(1) == 1; };
    if (code < 0 || dim < 1 || dim > 32768 || !dense_rows(*x)) return nullptr;
    if (branch && (branch->sizes() != x->sizes() || branch->scalar_type() != type || !dense_rows(*branch)))
      return nullptr;
    if (!branch && (r.post || mods[0] || weights[0] || !r.norm || ho)) return nullptr;
    if (!r.norm && (weights[1] || mods[1] || mods[2] || yo)) return nullptr;
    auto fits = [&](const at::Tensor& t, PyObject* o) {
      if (!output_fits(t, o, x->sizes(), type, {{x, a[0]}, {branch, a[1]}}, true)) return false;
      for (const at::Tensor* v : {mods[0], mods[1], mods[2], weights[0], weights[1], index})
        if (v && !apart(t, *v)) return false;
      return true;
    };
    if ((ho && !fits(*ho, a[11])) || (yo && !fits(*yo, a[12])) || (ho && yo && !apart(*ho, *yo))) return nullptr;
    r.weight_dtype = r.mod_dtype = code;
    bool seen = false;
    for (const at::Tensor* w : weights) {
      if (!w) continue;
      const int c = type_code(w->scalar_type());
      if (w->dim() != 1 || w->size(0) != dim || !w->is_contiguous() || (c != NKV_F32 && c != code) ||
          (seen && c != r.weight_dtype))
        return nullptr;
      r.weight_dtype = c;
      seen = true;
    }
    int64_t groups = 0;
    for (const at::Tensor* m : mods) {
      if (!m) continue;
      const int c = type_code(m->scalar_type());
      if (m->dim() < 1 || m->dim() > 2) return nullptr;
      const int64_t g = m->dim() == 1 ? 1 : m->size(0);
      if (m->size(-1) != dim || !m->is_contiguous() || g < 1 || g > INT32_MAX || (c != NKV_F32 && c != code) ||
          (groups && (c != r.mod_dtype || g != groups)))
        return nullptr;
      r.mod_dtype = c;
      groups = g;
    }
    if (index ? (index->dim() != 1 || index->size(0) != tokens || index->scalar_type() != at::kInt ||
                 !index->is_contiguous() || !groups)
              : groups > 1)
      return nullptr;
    at::Tensor h, y;
    if (branch && !ho) h = at::empty(x->sizes(), x->options());
    if (r.norm && !yo) y = at::empty(x->sizes(), x->options());
    const at::Tensor &hr = ho ? *ho : h, &yr = yo ? *yo : y;
    r.tokens = uint64_t(tokens);
    r.dim = dim;
    r.dtype = code;
    r.x = x->data_ptr(), r.x_stride = x->stride(0);
    if (branch) r.branch = branch->data_ptr(), r.branch_stride = branch->stride(0);
    if (branch) r.h_out = hr.data_ptr(), r.h_stride = hr.stride(0);
    if (r.norm) r.y_out = yr.data_ptr(), r.y_stride = yr.stride(0);
    r.post_weight = address(weights[0]), r.weight = address(weights[1]);
    r.gate = address(mods[0]), r.scale = address(mods[1]), r.shift = address(mods[2]);
    r.mod_index = static_cast<const int32_t*>(address(index));
    r.mod_rows = int32_t(groups);
    void* st = in.stream();
    if (!run([&] { return entries.residual_norm(&r, st); })) return nullptr;
    written(ho), written(yo);
    PyObject* first = a[0];
    if (branch) first = handed(a[11], h);
    else Py_INCREF(first);
    PyObject* second = Py_None;
    if (r.norm) second = handed(a[12], y);
    else Py_INCREF(second);
    return pair_of(first, second);
  });
}

// What an AttendPlan packs for attend_packed.
struct PlanKey {
  uint64_t plan;
  int32_t heads, kv_heads, head_dim, device;
  uint64_t q_tokens, k_tokens, workspace;
};

// attend_packed(key, q, k, v, scale or None, history's o, its lse, out, lse) -> (out, lse)
PyObject* attend_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    PlanKey plan;
    if (n != 9 || !entries.attend_packed || !PyBytes_CheckExact(a[0]) ||
        PyBytes_GET_SIZE(a[0]) != Py_ssize_t(sizeof(plan)))
      return nullptr;
    std::memcpy(&plan, PyBytes_AS_STRING(a[0]), sizeof(plan));
    double scale = 1.0 / std::sqrt(double(plan.head_dim));
    if (a[4] != Py_None && (!number(a[4], &scale) || !(scale > 0.0 && scale <= 3.4e38))) return nullptr;
    Tensors in;
    const at::Tensor *q = in.required(a[1]), *k = in.required(a[2]), *v = in.required(a[3]), *ho = in.optional(a[5]),
                     *hl = in.optional(a[6]), *out = in.optional(a[7]), *lse = in.optional(a[8]);
    const int64_t H = plan.heads, KV = plan.kv_heads, D = plan.head_dim, rows = int64_t(plan.q_tokens);
    if (!in.ok || in.device != plan.device || (ho == nullptr) != (hl == nullptr)) return nullptr;
    const at::ScalarType type = q->scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return nullptr;
    nkv_attend_args r{};
    // strides of a (tokens, heads, D) tensor; one that has a single element to step over does not count
    auto strides = [&](const at::Tensor& t, int64_t tokens, int64_t heads, bool exact, int64_t* token, int64_t* head) {
      if (t.dim() != 3 || t.size(1) != heads || t.size(2) != D || (exact ? t.size(0) != tokens : t.size(0) < tokens) ||
          t.scalar_type() != type || t.stride(2) != 1)
        return false;
      *token = t.size(0) < 2 ? 0 : t.stride(0);
      *head = heads < 2 ? 0 : t.stride(1);
      return ((reinterpret_cast<uintptr_t>(t.data_ptr()) | uintptr_t(2 * *token) | uintptr_t(2 * *head)) & 15u) == 0;
    };
    // (a batch padded behind the last sequence wants its outputs cleared: not here)
    if (!strides(*q, rows, H, true, &r.q_token_stride, &r.q_head_stride) ||
        !strides(*k, int64_t(plan.k_tokens), KV, false, &r.k_token_stride, &r.k_head_stride) ||
        !strides(*v, int64_t(plan.k_tokens), KV, false, &r.v_token_stride, &r.v_head_stride))
      return nullptr;
    if (ho && (ho->dim() != 3 || ho->size(0) != rows || ho->size(1) != H || ho->size(2) != D || hl->dim() != 2 ||
               hl->size(0) != H || hl->size(1) != rows || ho->scalar_type() != at::kFloat ||
               hl->scalar_type() != at::kFloat || !ho->is_contiguous() || !hl->is_contiguous()))
      return nullptr;
    const int64_t shape[3] = {rows, H, D}, lse_shape[2] = {H, rows};
    const at::ScalarType out_type = out && out->scalar_type() == at::kFloat ? at::kFloat : type;
    if (out && (!out->is_contiguous() || (lse && !apart(*out, *lse)) ||
                !output_fits(*out, a[7], shape, out_type, {{q, a[1]}, {k, a[2]}, {v, a[3]}, {ho, a[5]}, {hl, a[6]}}, false)))
      return nullptr;
    if (lse && (!lse->is_contiguous() || !output_fits(*lse, a[8], lse_shape, at::kFloat,
                                                      {{q, a[1]}, {k, a[2]}, {v, a[3]}, {ho, a[5]}, {hl, a[6]}}, false)))
      return nullptr;
    at::Tensor made, made_lse, ws;
    if (!out) made = at::empty(shape, q->options());
    if (!lse) made_lse = at::empty(lse_shape, q->options().dtype(at::kFloat));
    if (plan.workspace) ws = at::empty({int64_t(plan.workspace)}, q->options().dtype(at::kByte));
    r.dtype = type_code(type);
    r.out_dtype = type_code(out_type);
    r.q_rows = uint64_t(rows);
    r.k_rows = uint64_t(std::min(k->size(0), v->size(0)));
    r.q = q->data_ptr(), r.k = k->data_ptr(), r.v = v->data_ptr();
    r.scale = float(scale);
    r.out = (out ? *out : made).data_ptr();
    r.lse = static_cast<float*>((lse ? *lse : made_lse).data_ptr());
    r.hist_out = static_cast<const float*>(address(ho));
    r.hist_lse = static_cast<const float*>(address(hl));
    if (plan.workspace) r.workspace = ws.data_ptr();
    r.workspace_bytes = plan.workspace;
    void* st = in.stream();
    if (!run([&] { return entries.attend_packed(reinterpret_cast<const nkv_attend_plan*>(plan.plan), &r, st); }))
      return nullptr;
    written(out), written(lse);
    return pair_of(handed(a[7], made), handed(a[8], made_lse));
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {{"bind", fast<bind>(), METH_FASTCALL, nullptr},
                         {"rope_tables", fast<rope_tables>(), METH_FASTCALL, nullptr},
                         {"rotary", fast<rotary>(), METH_FASTCALL, nullptr},
                         {"residual_norm", fast<residual_norm>(), METH_FASTCALL, nullptr},
                         {"attend_packed", fast<attend_packed>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block_binding", nullptr, -1, methods, nullptr, nullptr, nullptr,
                      nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block_binding() { return PyModule_Create(&module); }
