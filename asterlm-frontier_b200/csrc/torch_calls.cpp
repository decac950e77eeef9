// The shortest way from torch tensors to the entry points of the C library that a step calls for every
// layer, or once for its drafts: and at a few microseconds of GPU work the checks of a call in Python (some 15 us)
// are what the step waits for.
//
// A function here takes well-formed calls only.  Whatever else it is given (a wrong type, shape or device,
// strides to be copied, a missing workspace, a status of the library) it answers NotImplemented, having
// done nothing, and the caller's own checks in Python decide what to say or do about it.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <map>
#include <utility>

#include "asterq.h"

namespace {

using Entry = int (*)(const void*, void*);
Entry g_append = nullptr, g_attend = nullptr, g_linear = nullptr, g_normed = nullptr, g_rows = nullptr, g_keep = nullptr,
      g_verify = nullptr;

struct Workspace {
  void* ptr;
  int64_t bytes;
};
std::map<std::pair<int, intptr_t>, Workspace> g_workspaces[3];  // of paged attention, of linear attention, of the attention of prompts and trees

PyObject* pass() { Py_RETURN_NOTIMPLEMENTED; }

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor* t, int device) { return t && t->is_cuda() && t->get_device() == device && t->layout() == at::kStrided; }

bool ints(const at::Tensor* t, int device, std::initializer_list<int64_t> shape) {
  return on(t, device) && t->scalar_type() == at::kInt && t->sizes() == at::IntArrayRef(shape) && t->is_contiguous();
}

// what Python refuses: there is no backward pass
bool wants_gradient(const at::Tensor* t) { return t->requires_grad() && at::GradMode::is_enabled(); }

// [rows, heads, dim] that the kernels read in 16-byte loads
bool rows(const at::Tensor* t, int device, at::ScalarType type, int64_t dim) {
  return on(t, device) && t->dim() == 3 && t->scalar_type() == type && t->size(2) == dim && t->stride(2) == 1 &&
         ((t->stride(0) | t->stride(1)) & 7) == 0 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0 && !wants_gradient(t);
}

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? ASTERQ_DTYPE_BF16 : t == at::kHalf ? ASTERQ_DTYPE_F16 : t == at::kFloat ? ASTERQ_DTYPE_F32 : -1;
}

bool pools_ok(const at::Tensor* k, const at::Tensor* v) {
  return k && v && k->is_cuda() && v->is_cuda() && k->get_device() == v->get_device() && k->dim() == 4 &&
         k->sizes() == v->sizes() && k->scalar_type() == v->scalar_type() &&
         (k->scalar_type() == at::kBFloat16 || k->scalar_type() == at::kHalf) && k->is_contiguous() && v->is_contiguous();
}

void* status_of(PyObject* o, int device, bool& ok) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  ok = ok && ints(t, device, {1});
  return ok ? t->data_ptr() : nullptr;
}

intptr_t stream_of(int device) { return reinterpret_cast<intptr_t>(c10::cuda::getCurrentCUDAStream(device).stream()); }

// pools_ok(k, v)
PyObject* check_pools(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return pass();
  if (pools_ok(tensor(args[0]), tensor(args[1]))) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

// What a vector of weights [dim] is to a call: absent, of a type code, or not for here
bool weights(PyObject* o, int device, int64_t dim, int rows_type, const void*& ptr, int& type) {
  if (o == Py_None) return true;
  const at::Tensor* w = tensor(o);
  if (!on(w, device) || w->sizes() != at::IntArrayRef({dim}) || !w->is_contiguous() || wants_gradient(w)) return false;
  const int code = type_code(w->scalar_type());
  if ((code != ASTERQ_DTYPE_F32 && code != rows_type) || (type >= 0 && type != code)) return false;
  ptr = w->data_ptr();
  type = code;
  return true;
}

// append(k_pool, v_pool, page_table, lengths, row_offsets, k, v, q, cos, sin, interleaved, q_out, status,
//        q_norm, k_norm, norm_eps, positions)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 17 || !g_append || !g_normed) return pass();
  const at::Tensor *kp = tensor(args[0]), *vp = tensor(args[1]), *table = tensor(args[2]), *lengths = tensor(args[3]),
                   *offsets = tensor(args[4]), *k = tensor(args[5]), *v = tensor(args[6]);
  if (!pools_ok(kp, vp) || !table || table->dim() != 2) return pass();
  const int device = kp->get_device();
  const at::ScalarType type = kp->scalar_type();
  const int64_t n_seqs = table->size(0), max_pages = table->size(1), n_kv = kp->size(1), page = kp->size(2), dim = kp->size(3);
  if (device != c10::cuda::current_device() || !rows(k, device, type, dim) || !rows(v, device, type, dim) ||
      k->size(1) != n_kv || v->size(1) != n_kv || v->size(0) != k->size(0) || !ints(table, device, {n_seqs, max_pages}) ||
      !ints(lengths, device, {n_seqs}) || !ints(offsets, device, {n_seqs + 1}))
    return pass();
  asterq_kv_append_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[12], device, ok));
  at::Tensor out;
  const bool has_q = args[7] != Py_None, given = args[11] != Py_None;
  if (has_q) {
    const at::Tensor* q = tensor(args[7]);
    if (!rows(q, device, type, dim) || q->size(0) != k->size(0)) return pass();
    p.q = q->data_ptr();
    p.n_heads = (int32_t)q->size(1);
    p.q_row_stride = q->stride(0);
    p.q_head_stride = q->stride(1);
    if (given) {
      const at::Tensor* o = tensor(args[11]);
      if (!on(o, device) || o->sizes() != q->sizes() || o->scalar_type() != type || !o->is_contiguous()) return pass();
      out = *o;
    }
  } else if (given) {
    return pass();
  }
  if ((args[8] == Py_None) != (args[9] == Py_None)) return pass();
  if (args[8] != Py_None) {
    const at::Tensor *cos = tensor(args[8]), *sin = tensor(args[9]);
    if (!on(cos, device) || !on(sin, device) || cos->dim() != 2 || cos->sizes() != sin->sizes() ||
        cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || !cos->is_contiguous() || !sin->is_contiguous())
      return pass();
    p.cos = static_cast<const float*>(cos->data_ptr());
    p.sin = static_cast<const float*>(sin->data_ptr());
    p.n_positions = cos->size(0);
    p.rotary_dim = (int32_t)(2 * cos->size(1));
  }
  const int interleaved = PyObject_IsTrue(args[10]);
  if (!ok || interleaved < 0 || n_seqs > INT32_MAX || max_pages > INT32_MAX) {
    PyErr_Clear();
    return pass();
  }
  if (has_q && !given) out = at::empty({k->size(0), p.n_heads, dim}, k->options());
  const bool normed = args[13] != Py_None || args[14] != Py_None || args[16] != Py_None;
  asterq_kv_append_normed_params w = {};
  if (normed) {
    int norm_type = -1;
    if ((args[13] != Py_None && !has_q) || !PyFloat_CheckExact(args[15]) || !(PyFloat_AS_DOUBLE(args[15]) >= 0) ||
        !weights(args[13], device, dim, type_code(type), w.q_norm, norm_type) ||
        !weights(args[14], device, dim, type_code(type), w.k_norm, norm_type))
      return pass();
    w.norm_dtype = norm_type < 0 ? type_code(type) : norm_type;
    w.norm_eps = (float)PyFloat_AS_DOUBLE(args[15]);
    if (args[16] != Py_None) {
      const at::Tensor* at = tensor(args[16]);
      if (!p.cos || !ints(at, device, {k->size(0)})) return pass();
      w.positions = static_cast<const int32_t*>(at->data_ptr());
    }
  }
  const auto fill = [&](auto& p) {
    p.dtype = type_code(type);
    p.n_seqs = (int32_t)n_seqs;
    p.n_kv_heads = (int32_t)n_kv;
    p.head_dim = (int32_t)dim;
    p.interleaved = interleaved;
    p.page_tokens = (int32_t)page;
    p.max_pages = (int32_t)max_pages;
    p.n_rows = k->size(0);
    p.n_pages = kp->size(0);
    p.k_row_stride = k->stride(0);
    p.k_head_stride = k->stride(1);
    p.v_row_stride = v->stride(0);
    p.v_head_stride = v->stride(1);
    p.k = k->data_ptr();
    p.v = v->data_ptr();
    p.page_table = static_cast<const int32_t*>(table->data_ptr());
    p.lengths = static_cast<const int32_t*>(lengths->data_ptr());
    p.row_offsets = static_cast<const int32_t*>(offsets->data_ptr());
    p.q_out = has_q ? out.data_ptr() : nullptr;
    p.k_pool = kp->data_ptr();
    p.v_pool = vp->data_ptr();
  };
  int status;
  if (normed) {
    w.n_heads = p.n_heads;
    w.rotary_dim = p.rotary_dim;
    w.n_positions = p.n_positions;
    w.q_row_stride = p.q_row_stride;
    w.q_head_stride = p.q_head_stride;
    w.q = p.q;
    w.cos = p.cos;
    w.sin = p.sin;
    w.status = p.status;
    fill(w);
    status = g_normed(&w, reinterpret_cast<void*>(stream_of(device)));
  } else {
    fill(p);
    status = g_append(&p, reinterpret_cast<void*>(stream_of(device)));
  }
  if (status != ASTERQ_OK) return pass();
  if (!has_q) Py_RETURN_NONE;
  if (given) {
    Py_INCREF(args[11]);
    return args[11];
  }
  return THPVariable_Wrap(out);
}

// attend(k_pool, v_pool, page_table, lengths, q, n_new, window, sink, scale, softcap, out, want_lse, status)
//   -> out, or (out, lse)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 13 || !g_attend) return pass();
  const at::Tensor *kp = tensor(args[0]), *vp = tensor(args[1]), *table = tensor(args[2]), *lengths = tensor(args[3]),
                   *q = tensor(args[4]);
  if (!pools_ok(kp, vp) || !table || table->dim() != 2) return pass();
  const int device = kp->get_device();
  const at::ScalarType type = kp->scalar_type();
  const int64_t n_rows = table->size(0), max_pages = table->size(1), n_kv = kp->size(1), dim = kp->size(3);
  if (device != c10::cuda::current_device() || !rows(q, device, type, dim) || q->size(0) != n_rows || n_kv == 0 ||
      q->size(1) % n_kv || !ints(table, device, {n_rows, max_pages}) || !ints(lengths, device, {n_rows}) ||
      n_rows > INT32_MAX || max_pages > INT32_MAX)
    return pass();
  for (int i : {5, 6, 7})
    if (!PyLong_CheckExact(args[i])) return pass();
  if (!PyFloat_CheckExact(args[8]) || !PyFloat_CheckExact(args[9])) return pass();
  const long n_new = PyLong_AsLong(args[5]), window = PyLong_AsLong(args[6]), sink = PyLong_AsLong(args[7]);
  const int want_lse = PyObject_IsTrue(args[11]);
  if (PyErr_Occurred() || n_new < 0 || window < 0 || sink < 0 || n_new > INT32_MAX || window > INT32_MAX || sink > INT32_MAX) {
    PyErr_Clear();
    return pass();
  }
  const intptr_t stream = stream_of(device);
  const auto ws = g_workspaces[0].find({device, stream});
  if (ws == g_workspaces[0].end()) return pass();
  asterq_paged_attention_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[12], device, ok));
  if (!ok) return pass();
  at::Tensor out, lse;
  const bool given = args[10] != Py_None;
  if (given) {
    const at::Tensor* o = tensor(args[10]);
    if (!on(o, device) || o->sizes() != q->sizes() || !o->is_contiguous()) return pass();
    out = *o;
  } else {
    out = at::empty({n_rows, q->size(1), dim}, q->options());
  }
  if (want_lse) lse = at::empty({n_rows, q->size(1)}, q->options().dtype(at::kFloat));
  p.dtype = type_code(type);
  p.out_dtype = type_code(out.scalar_type());
  p.n_rows = (int32_t)n_rows;
  p.n_heads = (int32_t)q->size(1);
  p.n_kv_heads = (int32_t)n_kv;
  p.head_dim = (int32_t)dim;
  p.page_tokens = (int32_t)kp->size(2);
  p.max_pages = (int32_t)max_pages;
  p.n_new = (int32_t)n_new;
  p.window = (int32_t)window;
  p.sink = (int32_t)sink;
  p.softmax_scale = (float)PyFloat_AS_DOUBLE(args[8]);
  p.logit_softcap = (float)PyFloat_AS_DOUBLE(args[9]);
  p.n_pages = kp->size(0);
  p.q_row_stride = q->stride(0);
  p.q_head_stride = q->stride(1);
  p.q = q->data_ptr();
  p.k_pool = kp->data_ptr();
  p.v_pool = vp->data_ptr();
  p.page_table = static_cast<const int32_t*>(table->data_ptr());
  p.lengths = static_cast<const int32_t*>(lengths->data_ptr());
  p.out = out.data_ptr();
  p.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  p.workspace = ws->second.ptr;
  p.workspace_bytes = ws->second.bytes;
  if (g_attend(&p, reinterpret_cast<void*>(stream)) != ASTERQ_OK) return pass();
  PyObject* o = args[10];
  if (given) Py_INCREF(o);
  else o = THPVariable_Wrap(out);
  if (!want_lse) return o;
  PyObject* l = THPVariable_Wrap(lse);
  PyObject* both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_XDECREF(o);
  Py_XDECREF(l);
  return both;
}

// linear(state, slots, lengths, row_offsets, q, k, v, log_decay, scale, out, status) -> out
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11 || !g_linear) return pass();
  const at::Tensor *state = tensor(args[0]), *slots = tensor(args[1]), *q = tensor(args[4]), *k = tensor(args[5]),
                   *v = tensor(args[6]), *g = tensor(args[7]);
  if (!state || !state->is_cuda() || state->dim() != 4 || state->scalar_type() != at::kFloat || !state->is_contiguous() ||
      !q || q->dim() != 3 || !slots || slots->dim() != 1)
    return pass();
  const int device = state->get_device();
  const at::ScalarType type = q->scalar_type();
  const int64_t n_rows = q->size(0), heads = q->size(1), dk = state->size(2), dv = state->size(3), n_seqs = slots->size(0);
  if (device != c10::cuda::current_device() || type_code(type) < 0 || state->size(1) != heads || !rows(q, device, type, dk) ||
      !rows(k, device, type, dk) || !rows(v, device, type, dv) || k->size(0) != n_rows || v->size(0) != n_rows ||
      k->size(1) != heads || v->size(1) != heads || !ints(slots, device, {n_seqs}) || n_seqs > INT32_MAX ||
      heads > INT32_MAX || state->size(0) > INT32_MAX)
    return pass();
  if (!on(g, device) || wants_gradient(g) || wants_gradient(state) || g->scalar_type() != at::kFloat || g->dim() < 1 || g->dim() > 2 || g->stride(-1) != 1 ||
      g->size(-1) != heads || (g->dim() == 2 && g->size(0) != n_rows) || !PyFloat_CheckExact(args[8]))
    return pass();
  asterq_linear_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[10], device, ok));
  if (!ok) return pass();
  if (args[2] != Py_None) {
    const at::Tensor* lengths = tensor(args[2]);
    if (!ints(lengths, device, {n_seqs})) return pass();
    p.lengths = static_cast<const int32_t*>(lengths->data_ptr());
  }
  const intptr_t stream = stream_of(device);
  if (args[3] != Py_None) {
    const at::Tensor* offsets = tensor(args[3]);
    if (!ints(offsets, device, {n_seqs + 1})) return pass();
    p.row_offsets = static_cast<const int32_t*>(offsets->data_ptr());
    const auto ws = g_workspaces[1].find({device, stream});
    if (ws == g_workspaces[1].end()) return pass();
    p.workspace = ws->second.ptr;
    p.workspace_bytes = ws->second.bytes;
  } else if (n_seqs != n_rows) {
    return pass();
  }
  at::Tensor out;
  const bool given = args[9] != Py_None;
  if (given) {
    const at::Tensor* o = tensor(args[9]);
    if (!on(o, device) || o->sizes() != at::IntArrayRef({n_rows, heads, dv}) || o->scalar_type() != type || !o->is_contiguous())
      return pass();
    out = *o;
  } else {
    out = at::empty({n_rows, heads, dv}, q->options());
  }
  p.dtype = type_code(type);
  p.n_seqs = (int32_t)n_seqs;
  p.n_heads = (int32_t)heads;
  p.dk = (int32_t)dk;
  p.dv = (int32_t)dv;
  p.n_slots = (int32_t)state->size(0);
  p.scale = (float)PyFloat_AS_DOUBLE(args[8]);
  p.n_rows = n_rows;
  p.q_row_stride = q->stride(0);
  p.q_head_stride = q->stride(1);
  p.k_row_stride = k->stride(0);
  p.k_head_stride = k->stride(1);
  p.v_row_stride = v->stride(0);
  p.v_head_stride = v->stride(1);
  p.decay_row_stride = g->dim() == 2 ? g->stride(0) : 0;
  p.q = q->data_ptr();
  p.k = k->data_ptr();
  p.v = v->data_ptr();
  p.log_decay = static_cast<const float*>(g->data_ptr());
  p.state = static_cast<float*>(state->data_ptr());
  p.slots = static_cast<const int32_t*>(slots->data_ptr());
  p.out = out.data_ptr();
  if (g_linear(&p, reinterpret_cast<void*>(stream)) != ASTERQ_OK) return pass();
  if (given) {
    Py_INCREF(args[9]);
    return args[9];
  }
  return THPVariable_Wrap(out);
}

// rows(k_pool, v_pool, page_table, lengths, row_offsets, parents, q, scale, softcap, window, sink, out, want_lse, status,
//      active sequences)
//   -> out, or (out, lse)
PyObject* rows_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 15 || !g_rows) return pass();
  const at::Tensor *kp = tensor(args[0]), *vp = tensor(args[1]), *table = tensor(args[2]), *lengths = tensor(args[3]),
                   *offsets = tensor(args[4]), *q = tensor(args[6]);
  if (!pools_ok(kp, vp) || !table || table->dim() != 2) return pass();
  const int device = kp->get_device();
  const at::ScalarType type = kp->scalar_type();
  const int64_t n_seqs = table->size(0), max_pages = table->size(1), n_kv = kp->size(1), dim = kp->size(3);
  if (device != c10::cuda::current_device() || !rows(q, device, type, dim) || n_kv == 0 || q->size(1) == 0 ||
      q->size(1) % n_kv || q->size(0) == 0 || n_seqs == 0 || q->stride(0) <= 0 || q->stride(1) <= 0 ||
      !ints(table, device, {n_seqs, max_pages}) || !ints(lengths, device, {n_seqs}) || !ints(offsets, device, {n_seqs + 1}) ||
      n_seqs > INT32_MAX || max_pages > INT32_MAX)
    return pass();
  if (!PyFloat_CheckExact(args[7]) || !PyFloat_CheckExact(args[8]) || !PyLong_CheckExact(args[9]) || !PyLong_CheckExact(args[10]) ||
      !PyLong_CheckExact(args[14]))
    return pass();
  const long window = PyLong_AsLong(args[9]), sink = PyLong_AsLong(args[10]), active = PyLong_AsLong(args[14]);
  const int want_lse = PyObject_IsTrue(args[12]);
  if (PyErr_Occurred() || window < 0 || sink < 0 || window > INT32_MAX || sink > INT32_MAX || active < 0 || active > INT32_MAX) {
    PyErr_Clear();
    return pass();
  }
  // a graph's calls take a workspace of the graph's own memory
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return pass();
  const intptr_t stream = stream_of(device);
  const auto ws = g_workspaces[2].find({device, stream});
  if (ws == g_workspaces[2].end()) return pass();
  asterq_rows_attention_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[13], device, ok));
  if (!ok) return pass();
  if (args[5] != Py_None) {
    const at::Tensor* parents = tensor(args[5]);
    if (!ints(parents, device, {q->size(0)})) return pass();
    p.parents = static_cast<const int32_t*>(parents->data_ptr());
  }
  at::Tensor out, lse;
  const bool given = args[11] != Py_None;
  if (given) {
    const at::Tensor* o = tensor(args[11]);
    if (!on(o, device) || o->sizes() != q->sizes() || !o->is_contiguous() || wants_gradient(o)) return pass();
    out = *o;
  } else {
    out = at::empty(q->sizes(), q->options());
  }
  if (want_lse) lse = at::empty({q->size(0), q->size(1)}, q->options().dtype(at::kFloat));
  p.dtype = type_code(type);
  p.out_dtype = type_code(out.scalar_type());
  p.n_seqs = (int32_t)n_seqs;
  p.n_heads = (int32_t)q->size(1);
  p.n_kv_heads = (int32_t)n_kv;
  p.head_dim = (int32_t)dim;
  p.page_tokens = (int32_t)kp->size(2);
  p.max_pages = (int32_t)max_pages;
  p.window = (int32_t)window;
  p.sink = (int32_t)sink;
  p.softmax_scale = (float)PyFloat_AS_DOUBLE(args[7]);
  p.logit_softcap = (float)PyFloat_AS_DOUBLE(args[8]);
  p.n_rows = q->size(0);
  p.n_pages = kp->size(0);
  p.q_row_stride = q->stride(0);
  p.q_head_stride = q->stride(1);
  p.q = q->data_ptr();
  p.k_pool = kp->data_ptr();
  p.v_pool = vp->data_ptr();
  p.page_table = static_cast<const int32_t*>(table->data_ptr());
  p.lengths = static_cast<const int32_t*>(lengths->data_ptr());
  p.row_offsets = static_cast<const int32_t*>(offsets->data_ptr());
  p.out = out.data_ptr();
  p.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  p.n_active = (int32_t)active;
  p.workspace = ws->second.ptr;
  p.workspace_bytes = ws->second.bytes;
  if (g_rows(&p, reinterpret_cast<void*>(stream)) != ASTERQ_OK) return pass();
  PyObject* o = args[11];
  if (given) Py_INCREF(o);
  else o = THPVariable_Wrap(out);
  if (!want_lse) return o;
  PyObject* l = THPVariable_Wrap(lse);
  PyObject* both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_XDECREF(o);
  Py_XDECREF(l);
  return both;
}

// keep(k_pool of layer 0, n_layers, address of the k pools' addresses, of the v pools', page_table, lengths, row_offsets,
//      kept, n_kept, status)
PyObject* keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 10 || !g_keep) return pass();
  const at::Tensor *kp = tensor(args[0]), *table = tensor(args[4]), *lengths = tensor(args[5]), *offsets = tensor(args[6]),
                   *kept = tensor(args[7]), *n_kept = tensor(args[8]);
  if (!pools_ok(kp, kp) || !table || table->dim() != 2 || !kept || kept->dim() != 1) return pass();
  const int device = kp->get_device();
  const int64_t n_seqs = table->size(0), max_pages = table->size(1);
  if (device != c10::cuda::current_device() || !ints(table, device, {n_seqs, max_pages}) || !ints(lengths, device, {n_seqs}) ||
      !ints(offsets, device, {n_seqs + 1}) || !ints(kept, device, {kept->size(0)}) || !ints(n_kept, device, {n_seqs}) ||
      n_seqs > INT32_MAX || max_pages > INT32_MAX)
    return pass();
  asterq_kv_keep_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[9], device, ok));
  const long layers = PyLong_AsLong(args[1]);
  p.k_pools = reinterpret_cast<void* const*>(PyLong_AsSize_t(args[2]));
  p.v_pools = reinterpret_cast<void* const*>(PyLong_AsSize_t(args[3]));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return pass();
  }
  if (!ok || layers > INT32_MAX) return pass();
  p.dtype = type_code(kp->scalar_type());
  p.n_layers = (int32_t)layers;
  p.n_seqs = (int32_t)n_seqs;
  p.n_kv_heads = (int32_t)kp->size(1);
  p.head_dim = (int32_t)kp->size(3);
  p.page_tokens = (int32_t)kp->size(2);
  p.max_pages = (int32_t)max_pages;
  p.n_rows = kept->size(0);
  p.n_pages = kp->size(0);
  p.page_table = static_cast<const int32_t*>(table->data_ptr());
  p.lengths = static_cast<const int32_t*>(lengths->data_ptr());
  p.row_offsets = static_cast<const int32_t*>(offsets->data_ptr());
  p.kept = static_cast<const int32_t*>(kept->data_ptr());
  p.n_kept = static_cast<const int32_t*>(n_kept->data_ptr());
  if (g_keep(&p, reinterpret_cast<void*>(stream_of(device))) != ASTERQ_OK) return pass();
  Py_RETURN_NONE;
}

// verify(target_probs, tokens, row_offsets, parents, accept_uniforms, sample_uniforms, draft_probs, status)
//   -> (kept, n_kept, next_token)
PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8 || !g_verify) return pass();
  const at::Tensor *target = tensor(args[0]), *tokens = tensor(args[1]), *offsets = tensor(args[2]), *accept = tensor(args[4]),
                   *sample = tensor(args[5]);
  if (!target || !target->is_cuda() || target->dim() != 2 || !offsets || offsets->dim() != 1 || offsets->size(0) < 2) return pass();
  const int device = target->get_device();
  const int64_t n_rows = target->size(0), vocab = target->size(1), n_seqs = offsets->size(0) - 1;
  const auto probs = [&](const at::Tensor* t) {
    return on(t, device) && t->sizes() == target->sizes() && t->scalar_type() == target->scalar_type() && t->stride(1) == 1 &&
           !wants_gradient(t);
  };
  const auto uniforms = [&](const at::Tensor* t, int64_t count) {
    return on(t, device) && t->scalar_type() == at::kFloat && t->sizes() == at::IntArrayRef({count}) && t->is_contiguous();
  };
  if (device != c10::cuda::current_device() || type_code(target->scalar_type()) < 0 || vocab == 0 || vocab > INT32_MAX ||
      n_seqs > INT32_MAX || !probs(target) || !ints(tokens, device, {n_rows}) || !ints(offsets, device, {n_seqs + 1}) ||
      !uniforms(accept, n_rows) || !uniforms(sample, n_seqs))
    return pass();
  asterq_verify_params p = {};
  bool ok = true;
  p.status = static_cast<int32_t*>(status_of(args[7], device, ok));
  if (!ok) return pass();
  if (args[3] != Py_None) {
    const at::Tensor* parents = tensor(args[3]);
    if (!ints(parents, device, {n_rows})) return pass();
    p.parents = static_cast<const int32_t*>(parents->data_ptr());
  }
  if (args[6] != Py_None) {
    const at::Tensor* draft = tensor(args[6]);
    if (!probs(draft)) return pass();
    p.draft = draft->data_ptr();
    p.draft_stride = draft->stride(0);
  }
  const auto kind = tokens->options();
  at::Tensor kept = at::empty({n_rows}, kind), n_kept = at::empty({n_seqs}, kind), next = at::empty({n_seqs}, kind);
  p.dtype = type_code(target->scalar_type());
  p.n_seqs = (int32_t)n_seqs;
  p.vocab = (int32_t)vocab;
  p.n_rows = n_rows;
  p.target_stride = target->stride(0);
  p.target = target->data_ptr();
  p.tokens = static_cast<const int32_t*>(tokens->data_ptr());
  p.row_offsets = static_cast<const int32_t*>(offsets->data_ptr());
  p.accept = static_cast<const float*>(accept->data_ptr());
  p.sample = static_cast<const float*>(sample->data_ptr());
  p.kept = static_cast<int32_t*>(kept.data_ptr());
  p.n_kept = static_cast<int32_t*>(n_kept.data_ptr());
  p.next_token = static_cast<int32_t*>(next.data_ptr());
  if (g_verify(&p, reinterpret_cast<void*>(stream_of(device))) != ASTERQ_OK) return pass();
  PyObject *a = THPVariable_Wrap(kept), *b = THPVariable_Wrap(n_kept), *c = THPVariable_Wrap(next);
  PyObject* all = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(c);
  return all;
}

// bind(append, attend, linear, normed append, rows, keep, verify): addresses of the library's entry points
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Entry* to[] = {&g_append, &g_attend, &g_linear, &g_normed, &g_rows, &g_keep, &g_verify};
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes seven addresses");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i) *to[i] = reinterpret_cast<Entry>(PyLong_AsSize_t(args[i]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// workspace(kind, device, stream, pointer, bytes): what calls on this stream use; the caller keeps it alive
PyObject* workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "workspace takes kind, device, stream, pointer and bytes");
    return nullptr;
  }
  const long kind = PyLong_AsLong(args[0]), device = PyLong_AsLong(args[1]);
  const size_t stream = PyLong_AsSize_t(args[2]), ptr = PyLong_AsSize_t(args[3]);
  const long long bytes = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  if (kind < 0 || kind > 2) {
    PyErr_SetString(PyExc_ValueError, "kind is 0, 1 or 2");
    return nullptr;
  }
  g_workspaces[kind][{(int)device, (intptr_t)stream}] = {reinterpret_cast<void*>(ptr), bytes};
  Py_RETURN_NONE;
}

// C++ exceptions (an allocation that failed, say) end here: the Python side then meets the same
// condition by itself and raises torch's own error.
template <PyObject* (*kFn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return kFn(self, args, n);
  } catch (...) {
    return pass();
  }
}

template <PyObject* (*kFn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<kFn>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<check_pools>("check_pools"), method<append>("append"), method<attend>("attend"),
                           method<linear>("linear"),           method<bind>("bind"),     method<workspace>("workspace"),
                           method<rows_attention>("rows"),     method<keep>("keep"),     method<verify>("verify"),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `version` names the torch that this was compiled against: with another one the module is not to be used
PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "version", ASTERQ_CALLS_VERSION) != 0) Py_CLEAR(m);
  return m;
}
