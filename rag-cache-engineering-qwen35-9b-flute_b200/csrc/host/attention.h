// Native route of the attention side (rotary.py, kvcache.py): the calls that need no conversion and break no
// rule. Anything else returns None, nothing launched, and the Python route converts it or refuses it.
#pragma once

#include <c10/core/AutogradState.h>

#include "route.h"

namespace b200host {

// A KVCache4's buffers (its C view and the tensors that keep them).
struct Cache {
  PyObject_HEAD
  b200lut_kv_cache view;
  at::Tensor* buffers[4];
  at::ScalarType scalar;
  int device;
};

extern PyTypeObject CacheType;

inline void cache_dealloc(PyObject* o) {
  for (at::Tensor* t : reinterpret_cast<Cache*>(o)->buffers) delete t;
  PyObject_Free(o);
}

inline const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// no gradient to lose, backward or forward
inline bool plain(const at::Tensor& t) {
  return !(t.requires_grad() && c10::GradMode::is_enabled()) &&
         !(t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}

// [tokens, heads, D] in `scalar` with rows of 16 bytes.
inline bool head_rows(const at::Tensor& t, at::ScalarType scalar, int device, int64_t heads, int64_t D) {
  return t.is_cuda() && t.get_device() == device && t.scalar_type() == scalar && t.dim() == 3 && t.size(1) == heads &&
         t.size(2) == D && t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && plain(t) &&
         (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 && t.size(0) > 0 && t.size(0) <= 0x7fffffff;
}
// contiguous int32 [n]
inline bool ints(const at::Tensor& t, int device, int64_t n) {
  return t.is_cuda() && t.get_device() == device && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n &&
         (n <= 1 || t.stride(0) == 1);
}

inline const int32_t* i32(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

// n elements of `st` of base's memory, from byte `at` on (a dispatched view costs several times as much).
inline at::Tensor piece(const at::Tensor& base, at::ScalarType st, int64_t at, int64_t n) {
  const auto type = c10::scalarTypeToTypeMeta(st);
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), type);
  c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  impl->set_storage_offset(at / int64_t(type.itemsize()));
  impl->set_sizes_contiguous({n});
  return t;
}

template <size_t N>
PyObject* tuple_of(at::Tensor (&ts)[N]) {
  PyObject* r = PyTuple_New(N);
  if (!r) return nullptr;
  for (size_t i = 0; i < N; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(ts[i]));
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, Py_ssize_t(i), o);
  }
  return r;
}

// bind_cache(k_codes, v_codes, k_pairs, v_pairs, n_pages, page_size, n_kv_heads, head_dim)
inline PyObject* bind_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bind_cache(k_codes, v_codes, k_pairs, v_pairs, n_pages, page_size, n_kv_heads, head_dim)");
    return nullptr;
  }
  for (int i = 0; i < 4; ++i)
    if (!THPVariable_Check(a[i])) {
      PyErr_SetString(PyExc_TypeError, "bind_cache: tensors wanted");
      return nullptr;
    }
  long v[4];
  for (int i = 0; i < 4; ++i) {
    v[i] = PyLong_AsLong(a[4 + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  Cache* c = PyObject_New(Cache, &CacheType);
  if (!c) return nullptr;
  for (int i = 0; i < 4; ++i) c->buffers[i] = nullptr;
  for (int i = 0; i < 4; ++i) c->buffers[i] = new at::Tensor(THPVariable_Unpack(a[i]));
  c->scalar = c->buffers[2]->scalar_type();
  c->device = int(c->buffers[0]->get_device());
  c->view = {c->buffers[0]->mutable_data_ptr(), c->buffers[1]->mutable_data_ptr(), c->buffers[2]->mutable_data_ptr(),
             c->buffers[3]->mutable_data_ptr(), int(v[0]), int(v[1]), int(v[2]), int(v[3]),
             c->scalar == at::kHalf ? B200LUT_F16 : B200LUT_BF16};
  return reinterpret_cast<PyObject*>(c);
}

inline Cache* cache_of(PyObject* o) { return Py_TYPE(o) == &CacheType ? reinterpret_cast<Cache*>(o) : nullptr; }

// kv_write(cache, k, v, slots): True when the rows were written.
template <typename Guard, typename Context>
PyObject* kv_write(Guard&& guarded, Context&& context, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "kv_write(cache, k, v, slots)");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor *k = tensor_of(a[1]), *v = tensor_of(a[2]), *s = tensor_of(a[3]);
    Ctx x;
    if (!c || !k || !v || !s || !head_rows(*k, c->scalar, c->device, c->view.n_kv_heads, c->view.head_dim) ||
        !head_rows(*v, c->scalar, c->device, c->view.n_kv_heads, c->view.head_dim) || v->size(0) != k->size(0) ||
        !ints(*s, c->device, k->size(0)) || !context(c->device, false, &x))
      Py_RETURN_NONE;
    const Held held(c);
    {
      const WithoutGil free;
      check(b200lut_kv_write(&c->view, k->const_data_ptr(), v->const_data_ptr(), k->stride(0), k->stride(1), v->stride(0),
                             v->stride(1), i32(*s), int(k->size(0)), x.stream));
    }
    return Py_NewRef(Py_True);
  });
}

// kv_read(cache, slots): (k, v)
template <typename Guard, typename Context>
PyObject* kv_read(Guard&& guarded, Context&& context, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "kv_read(cache, slots)");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor* s = tensor_of(a[1]);
    Ctx x;
    if (!c || !s || s->dim() != 1 || s->size(0) == 0 || s->size(0) > 0x7fffffff || !ints(*s, c->device, s->size(0)) ||
        !context(c->device, false, &x))
      Py_RETURN_NONE;
    const Held held(c);
    at::Tensor out[2];
    {
      const WithoutGil free;
      for (at::Tensor& t : out) t = empty({s->size(0), c->view.n_kv_heads, c->view.head_dim}, c->scalar, c->device);
      check(b200lut_kv_read(&c->view, out[0].mutable_data_ptr(), out[1].mutable_data_ptr(), i32(*s), int(s->size(0)), x.stream));
    }
    return tuple_of(out);
  });
}

// attend(cache, q, block_table, kv_len, row_start or None, scale, window, sinks, gate or None, out or None): the result
template <typename Guard, typename Context>
PyObject* attend(Guard&& guarded, Context&& context, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "attend(cache, q, block_table, kv_len, row_start, scale, window, sinks, gate, out)");
    return nullptr;
  }
  if (!PyFloat_Check(a[5]) || !PyLong_CheckExact(a[6]) || !PyLong_CheckExact(a[7])) Py_RETURN_NONE;
  const double scale = PyFloat_AS_DOUBLE(a[5]);
  int over = 0, over2 = 0;
  const long window = PyLong_AsLongAndOverflow(a[6], &over), sinks = PyLong_AsLongAndOverflow(a[7], &over2);
  if (over || over2 || window < 0 || sinks < 0 || window > 0x7fffffff || sinks > 0x7fffffff || !(std::fabs(scale) < 0x1p127)) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor *q = tensor_of(a[1]), *table = tensor_of(a[2]), *len = tensor_of(a[3]), *start = tensor_of(a[4]),
                     *gate = tensor_of(a[8]), *given = tensor_of(a[9]);
    Ctx x;
    if (!c || !q || !table || !len || (!start && a[4] != Py_None) || (!gate && a[8] != Py_None) || (!given && a[9] != Py_None))
      Py_RETURN_NONE;
    const int64_t H = c->view.n_kv_heads, D = c->view.head_dim;
    if (q->dim() != 3 || q->size(1) < 1 || q->size(1) % H || q->size(1) / H > 64) Py_RETURN_NONE;
    const int64_t T = q->size(0), Hq = q->size(1);
    if (!head_rows(*q, c->scalar, c->device, Hq, D)) Py_RETURN_NONE;
    if (!table->is_cuda() || table->get_device() != c->device || table->scalar_type() != at::kInt || table->dim() != 2) Py_RETURN_NONE;
    const int64_t B = table->size(0), width = table->size(1);
    if (B < 1 || B > 65536 || width < 1 || width > 0x7fffffff || (width > 1 && table->stride(1) != 1)) Py_RETURN_NONE;
    if (!ints(*len, c->device, B) || (start ? !ints(*start, c->device, B + 1) : T != B)) Py_RETURN_NONE;
    if (gate && (!head_rows(*gate, c->scalar, c->device, Hq, D) || gate->size(0) != T)) Py_RETURN_NONE;
    if (given && (!head_rows(*given, c->scalar, c->device, Hq, D) || given->size(0) != T)) Py_RETURN_NONE;
    if (!context(c->device, false, &x)) Py_RETURN_NONE;
    const Held held(c);
    at::Tensor out, ws;
    {
      const WithoutGil free;
      out = given ? *given : empty({T, Hq, D}, c->scalar, c->device);
      // a buffer of the current stream (of the capture's pool under capture): calls never share one
      const size_t need = b200lut_attend_workspace_bytes(int(Hq), int(H), int(D), !start);
      ws = empty({int64_t(need)}, at::kByte, c->device);
      b200lut_attend_args g = {};
      g.cache = &c->view;
      g.q = q->const_data_ptr(), g.gate = gate ? gate->const_data_ptr() : nullptr, g.out = out.mutable_data_ptr();
      g.block_table = i32(*table), g.kv_len = i32(*len), g.row_start = start ? i32(*start) : nullptr;
      g.q_token_stride = q->stride(0), g.q_head_stride = q->stride(1);
      if (gate) g.gate_token_stride = gate->stride(0), g.gate_head_stride = gate->stride(1);
      g.out_token_stride = out.stride(0), g.out_head_stride = out.stride(1), g.table_stride = table->stride(0);
      g.T = int(T), g.B = int(B), g.width = int(width), g.n_heads = int(Hq);
      g.window = int(window), g.sinks = int(sinks), g.scale = float(scale);
      check(b200lut_attend(&g, ws.mutable_data_ptr(), need, x.stream));
    }
    if (given) return Py_NewRef(a[9]);
    return THPVariable_Wrap(std::move(out));
  });
}

// kv_plan(cached, fresh, block_table, free_pages, taken, page_size, max_tokens): the six results
template <typename Guard, typename Context>
PyObject* kv_plan(Guard&& guarded, Context&& context, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "kv_plan(cached, fresh, block_table, free_pages, taken, page_size, max_tokens)");
    return nullptr;
  }
  if (!PyLong_CheckExact(a[5]) || !PyLong_CheckExact(a[6])) Py_RETURN_NONE;
  int over = 0, over2 = 0;
  const long page = PyLong_AsLongAndOverflow(a[5], &over), room = PyLong_AsLongAndOverflow(a[6], &over2);
  if (over || over2 || page < 1 || page > 65536 || room < 1 || room > 0x7fffffff) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i) {
      t[i] = tensor_of(a[i]);
      if (!t[i]) Py_RETURN_NONE;
    }
    if (!t[0]->is_cuda() || t[0]->dim() != 1) Py_RETURN_NONE;
    const int device = int(t[0]->get_device());
    const int64_t B = t[0]->size(0);
    Ctx x;
    if (B < 1 || B > 8192 || !ints(*t[0], device, B) || !ints(*t[1], device, B) || !t[2]->is_cuda() ||
        t[2]->get_device() != device || t[2]->scalar_type() != at::kInt || t[2]->dim() != 2 || t[2]->size(0) != B ||
        t[2]->size(1) < 1 || t[2]->size(1) > 0x7fffffff || !t[2]->is_contiguous() || t[3]->dim() != 1 || t[3]->size(0) < 1 ||
        t[3]->size(0) > 0x7fffffff || !ints(*t[3], device, t[3]->size(0)) || !ints(*t[4], device, 1) || !context(device, false, &x))
      Py_RETURN_NONE;
    at::Tensor out[6];
    {
      const WithoutGil free;
      // row_start, kv_len, positions, slots, taken, served: pieces of one allocation, 16-byte aligned
      const int64_t sizes[6] = {4 * (B + 1), 4 * B, 4 * room, 4 * room, 4, B};
      int64_t at[7] = {0};
      for (int i = 0; i < 6; ++i) at[i + 1] = (at[i] + sizes[i] + 15) / 16 * 16;
      const at::Tensor base = empty({at[6]}, at::kByte, device);
      for (int i = 0; i < 6; ++i) out[i] = piece(base, i == 5 ? at::kBool : at::kInt, at[i], i == 5 ? B : sizes[i] / 4);
      auto p = [&](int i) { return static_cast<int32_t*>(out[i].mutable_data_ptr()); };
      b200lut_kv_plan_args g = {i32(*t[0]), i32(*t[1]), static_cast<int32_t*>(t[2]->mutable_data_ptr()), i32(*t[3]), i32(*t[4]),
                                p(0), p(1), p(2), p(3), p(4), static_cast<uint8_t*>(out[5].mutable_data_ptr()), int(B),
                                int(t[2]->size(1)), int(t[3]->size(0)), int(page), int(room)};
      check(b200lut_kv_plan(&g, x.stream));
    }
    return tuple_of(out);
  });
}

// rotary(q, k, positions, q_gain or None, k_gain or None, eps, turns, axis, axes): (q, k)
template <typename Guard, typename Context>
PyObject* rotary(Guard&& guarded, Context&& context, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "rotary(q, k, positions, q_gain, k_gain, eps, turns, axis, axes)");
    return nullptr;
  }
  if (!PyFloat_Check(a[5])) Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(a[5]);
  const long axes = PyLong_AsLong(a[8]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *pos = tensor_of(a[2]), *turns = tensor_of(a[6]), *axis = tensor_of(a[7]);
    const at::Tensor* gain[2] = {tensor_of(a[3]), tensor_of(a[4])};
    Ctx x;
    if (!q || !k || !pos || !turns || !axis || (a[3] == Py_None) != (a[4] == Py_None) || q->dim() != 3 || k->dim() != 3 || !q->is_cuda())
      Py_RETURN_NONE;
    const at::ScalarType st = q->scalar_type();
    const int device = int(q->get_device());
    const int64_t T = q->size(0), D = q->size(2);
    if ((st != at::kBFloat16 && st != at::kHalf) || !head_rows(*q, st, device, q->size(1), D) ||
        !head_rows(*k, st, device, k->size(1), D) || k->size(0) != T || turns->get_device() != device)
      Py_RETURN_NONE;
    if (!pos->is_cuda() || pos->get_device() != device || (pos->scalar_type() != at::kLong && pos->scalar_type() != at::kInt) ||
        pos->dim() < 1 || pos->dim() > 2 || pos->size(-1) != T || (T > 1 && pos->stride(-1) != 1) ||
        (pos->dim() == 2 && (pos->size(0) != axes || pos->stride(0) < 0)))
      Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i) {
      if (a[3 + i] == Py_None) continue;
      const at::Tensor* t = gain[i];
      if (!t || !t->is_cuda() || t->get_device() != device || t->scalar_type() != st || t->dim() != 1 || t->size(0) != D ||
          t->stride(0) != 1 || !plain(*t) || (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15))
        Py_RETURN_NONE;
    }
    if (!context(device, false, &x)) Py_RETURN_NONE;
    at::Tensor out[2];
    {
      const WithoutGil free;
      out[0] = empty(q->sizes(), st, device);
      out[1] = empty(k->sizes(), st, device);
      b200lut_rotary_args g = {};
      g.q = q->const_data_ptr(), g.k = k->const_data_ptr(), g.q_out = out[0].mutable_data_ptr(), g.k_out = out[1].mutable_data_ptr();
      if (gain[0]) g.q_gain = gain[0]->const_data_ptr(), g.k_gain = gain[1]->const_data_ptr();
      g.positions = pos->const_data_ptr(), g.pos64 = pos->scalar_type() == at::kLong;
      g.turns = static_cast<const double*>(turns->const_data_ptr()), g.axis = i32(*axis);
      g.q_token_stride = q->stride(0), g.q_head_stride = q->stride(1);
      g.k_token_stride = k->stride(0), g.k_head_stride = k->stride(1);
      g.pos_stride = pos->dim() == 2 ? pos->stride(0) : 0;
      g.T = int(T), g.n_heads = int(q->size(1)), g.n_kv_heads = int(k->size(1)), g.D = int(D), g.R = int(2 * turns->size(0));
      g.dtype = st == at::kHalf ? B200LUT_F16 : B200LUT_BF16, g.eps = float(eps);
      check(b200lut_rotary(&g, x.stream));
    }
    return tuple_of(out);
  });
}

}  // namespace b200host
