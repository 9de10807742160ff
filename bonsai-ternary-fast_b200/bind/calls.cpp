// The ordinary calls of btf_b200.rope, tree_attention, prefix_attention, adapters and sample,
// from torch tensors straight to the C ABI: a call of the ctypes mirror spends 6 to 15 us on
// reading the tensors and packing arguments, more than most of these kernels run. Only what needs no
// thought is done here: tensors of the expected types and shapes on the current
// device, its current stream. Everything else, errors among it, returns None, and the
// mirror does the call (nothing has been launched then).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "btf_b200.h"

namespace {

// The library that the mirror loaded.
struct Library {
  decltype(&btf_rope) rope = nullptr;
  decltype(&btf_tree_attention_work) tree_work = nullptr;
  decltype(&btf_tree_attention) tree = nullptr;
  decltype(&btf_sample) sample = nullptr;
  decltype(&btf_rope_axes) rope_axes = nullptr;
  decltype(&btf_prefix_attention_work) prefix_work = nullptr;
  decltype(&btf_prefix_attention) prefix = nullptr;
  decltype(&btf_adapters_work) adapters_work = nullptr;
  decltype(&btf_adapters) adapters = nullptr;
} lib;

// A refused fast call: caught below, becomes None.
struct Other {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw Other{};
  return THPVariable_Unpack(o);
}
const at::Tensor& on(PyObject* o, int dev) {
  const at::Tensor& t = tensor(o);
  if (!t.is_cuda() || t.get_device() != dev) throw Other{};
  return t;
}
// A tensor of a call that records no graph; the mirror refuses one that wants a gradient.
const at::Tensor& plain(const at::Tensor& t) {
  if (t.requires_grad() && at::GradMode::is_enabled()) throw Other{};
  return t;
}
// Autograd learns that a kernel has written it.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int elem(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BTF_F32;
    case at::kHalf: return BTF_F16;
    case at::kBFloat16: return BTF_BF16;
    default: throw Other{};
  }
}
// Address of a contiguous vector of n (or a matrix of n x m) of this type; null for None.
const void* vec(PyObject* o, int dev, at::ScalarType type, int64_t n, int64_t m = -1) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = on(o, dev);
  if (t.scalar_type() != type || t.dim() != (m < 0 ? 1 : 2) || t.size(0) != n || (m >= 0 && t.size(1) != m) ||
      !t.is_contiguous())
    throw Other{};
  return t.data_ptr();
}
template <typename T>
const T* vec(PyObject* o, int dev, at::ScalarType type, int64_t n, int64_t m = -1) {
  return static_cast<const T*>(vec(o, dev, type, n, m));
}
// References of a call, kept to its end (an attribute may be made anew each time it is read).
struct Kept {
  PyObject* of[3 * 6 + 6];
  int n = 0;
  Kept() = default;
  Kept(const Kept&) = delete;
  PyObject* keep(PyObject* o) {
    Py_INCREF(o);
    return of[n++] = o;
  }
  PyObject* attr(PyObject* from, PyObject* name) {
    PyObject* o = PyObject_GetAttr(from, name);
    if (!o) {
      PyErr_Clear();
      throw Other{};
    }
    return of[n++] = o;
  }
  ~Kept() {
    while (n) Py_DECREF(of[--n]);
  }
};
int flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    throw Other{};
  }
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Other{};
  }
  return v;
}
int64_t stride(const at::Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }  // of one entry none matters
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }
int device() { return c10::cuda::current_device(); }

// Runs fn; None when it is not for here (an exception of torch among it: the mirror's own call raises it).
template <typename Fn>
PyObject* attempt(Fn fn) {
  try {
    if (PyObject* r = fn()) return r;
  } catch (const Other&) {
  } catch (const std::exception&) {
  }
  Py_RETURN_NONE;
}

PyObject *s_x, *s_y, *s_normw, *s_rotate, *s_rows, *s_turns, *s_n_rot, *s_mscale, *s_interleaved, *s_axis, *s_n_axes;
PyObject *s_a, *s_b, *s_base, *s_plan, *s_T, *s_n_adapters;

// rope(segs, table, pos, inverse, eps) -> True, or None
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return attempt([&]() -> PyObject* {
    if (nargs != 5 || !PyList_Check(args[0])) throw Other{};
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    if (n < 1 || n > 3) throw Other{};
    const int dev = device();
    btf_rope_seg segs[3];
    const at::Tensor* to[3];
    Kept kept;
    int64_t T = 0, D = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (i >= PyList_GET_SIZE(args[0])) throw Other{};
      PyObject* s = kept.keep(PyList_GET_ITEM(args[0], i));
      PyObject *ox = kept.attr(s, s_x), *oy = kept.attr(s, s_y), *ow = kept.attr(s, s_normw);
      PyObject *orot = kept.attr(s, s_rotate), *orows = kept.attr(s, s_rows);
      const at::Tensor& x = plain(on(ox, dev));
      const at::Tensor& y = oy == Py_None ? x : plain(on(oy, dev));
      if (ow != Py_None) plain(on(ow, dev));
      if (x.dim() != 3 || y.dim() != 3) throw Other{};
      if (i == 0) T = x.size(0), D = x.size(2);
      if (x.size(0) != T || x.size(2) != D || y.size(2) != D || y.size(1) != x.size(1) || T > INT32_MAX || D > INT32_MAX ||
          x.size(1) > INT32_MAX || (D > 1 && (x.stride(2) != 1 || y.stride(2) != 1)) ||
          (orows == Py_None && y.size(0) != T))
        throw Other{};
      segs[i] = {x.data_ptr(), y.data_ptr(), elem(x), elem(y), (int)x.size(1), flag(orot),
                 stride(x, 0), stride(x, 1), stride(y, 0), stride(y, 1), vec<float>(ow, dev, at::kFloat, D),
                 vec<int32_t>(orows, dev, at::kInt, T), y.size(0)};
      to[i] = &y;
    }
    PyObject *turns = kept.attr(args[1], s_turns), *n_rot = kept.attr(args[1], s_n_rot);
    PyObject *mscale = kept.attr(args[1], s_mscale), *inter = kept.attr(args[1], s_interleaved);
    if (args[2] == Py_None || turns == Py_None || !PyLong_Check(n_rot)) throw Other{};
    const at::Tensor& f = on(turns, dev);
    if (f.scalar_type() != at::kDouble || !f.is_contiguous()) throw Other{};
    const long rot = PyLong_AsLong(n_rot);
    if (rot < 0 || rot > 2 * f.numel()) {
      PyErr_Clear();
      throw Other{};
    }
    const double* freq = static_cast<const double*>(f.data_ptr());
    PyObject* oaxis = kept.attr(args[1], s_axis);
    if (oaxis == Py_None) {
      if (lib.rope(segs, (int)n, (int)T, (int)D, (int)rot, freq, (float)number(mscale), flag(inter), flag(args[3]),
                   (float)number(args[4]), vec<int32_t>(args[2], dev, at::kInt, T), stream_of(dev)))
        throw Other{};
    } else {
      const at::Tensor& axis = on(oaxis, dev);
      const long axes = PyLong_AsLong(kept.attr(args[1], s_n_axes));
      if (axes < 1 || axes > BTF_ROPE_MAX_AXES || axis.scalar_type() != at::kByte || !axis.is_contiguous() ||
          rot > 2 * axis.numel()) {
        PyErr_Clear();
        throw Other{};
      }
      if (lib.rope_axes(segs, (int)n, (int)T, (int)D, (int)rot, freq, static_cast<const uint8_t*>(axis.data_ptr()),
                        (int)axes, (float)number(mscale), flag(inter), flag(args[3]), (float)number(args[4]),
                        vec<int32_t>(args[2], dev, at::kInt, axes, T), T, stream_of(dev)))
        throw Other{};
    }
    for (Py_ssize_t i = 0; i < n; ++i) written(*to[i]);
    Py_RETURN_TRUE;
  });
}

// Both attentions. args: q, k, v, lens, parents, counts, scale, out, work; shared: pk, pv, prefix_len or null.
PyObject* attention(PyObject* const* args, PyObject* const* shared) {
  return attempt([&]() -> PyObject* {
    const int dev = device();
    const at::Tensor &q = plain(on(args[0], dev)), &k = plain(on(args[1], dev)), &v = plain(on(args[2], dev));
    if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3) ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
      throw Other{};
    const int64_t B = q.size(0), n = q.size(1), H = q.size(2), D = q.size(3), ctx = k.size(1), HK = k.size(2);
    for (int64_t s : {B, n, H, D, ctx, HK})
      if (s < 1 || s > INT32_MAX) throw Other{};
    if (args[3] == Py_None || args[4] == Py_None) throw Other{};
    btf_prefix s{};
    if (shared) {
      const at::Tensor &pk = plain(on(shared[0], dev)), &pv = plain(on(shared[1], dev));
      if (pk.dim() != 3 || pv.sizes() != pk.sizes() || pk.size(1) != HK || pk.size(2) != D || pk.size(0) > INT32_MAX ||
          pk.scalar_type() != q.scalar_type() || pv.scalar_type() != q.scalar_type() ||
          stride(pk, 0) != stride(pv, 0) || stride(pk, 1) != stride(pv, 1) || (D > 1 && (pk.stride(2) != 1 || pv.stride(2) != 1)))
        throw Other{};
      s = {pk.data_ptr(), pv.data_ptr(), stride(pk, 0), stride(pk, 1), (int)pk.size(0), vec<int32_t>(shared[2], dev, at::kInt, 1)};
    }
    btf_tree_attn a{};
    a.lens = vec<int32_t>(args[3], dev, at::kInt, B);
    a.parents = vec<int32_t>(args[4], dev, at::kInt, B, n);
    a.counts = vec<int32_t>(args[5], dev, at::kInt, B);
    at::Tensor out, work;
    if (args[7] != Py_None) {
      out = plain(on(args[7], dev));
      if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type()) throw Other{};
    } else {
      out = a.counts ? at::zeros(q.sizes(), q.options()) : at::empty(q.sizes(), q.options());
    }
    if (args[8] != Py_None) {
      work = on(args[8], dev);
      if (!work.is_contiguous()) throw Other{};
    } else {
      const int64_t bytes = shared ? lib.prefix_work((int)B, (int)n, (int)H, (int)HK, (int)D, (int)ctx, s.rows)
                                   : lib.tree_work((int)B, (int)n, (int)H, (int)HK, (int)D, (int)ctx);
      if (bytes < 0) throw Other{};
      work = at::empty({bytes}, q.options().dtype(at::kByte));
    }
    for (int d = 0; d < 3; ++d)
      if (stride(k, d) != stride(v, d)) throw Other{};
    if (D > 1 && (q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1 || out.stride(3) != 1)) throw Other{};
    a.q = q.data_ptr(), a.q_batch = stride(q, 0), a.q_node = stride(q, 1), a.q_head = stride(q, 2);
    a.k = k.data_ptr(), a.v = v.data_ptr();
    a.kv_batch = stride(k, 0), a.kv_row = stride(k, 1), a.kv_head = stride(k, 2);
    a.o = out.data_ptr(), a.o_batch = stride(out, 0), a.o_node = stride(out, 1), a.o_head = stride(out, 2);
    a.type = elem(q);
    a.B = (int)B, a.n = (int)n, a.H = (int)H, a.HK = (int)HK, a.D = (int)D, a.n_ctx = (int)ctx;
    a.scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)number(args[6]);
    a.work = work.data_ptr(), a.work_bytes = (int64_t)work.nbytes();
    if (shared ? lib.prefix(&a, &s, stream_of(dev)) : lib.tree(&a, stream_of(dev))) throw Other{};
    written(out);
    if (args[7] != Py_None) {
      Py_INCREF(args[7]);
      return args[7];
    }
    return THPVariable_Wrap(out);
  });
}
// tree_attention(q, k, v, lens, parents, counts, scale, out, work) -> the output, or None
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9) Py_RETURN_NONE;
  return attention(args, nullptr);
}
// prefix_attention(q, k, v, lens, parents, counts, scale, out, work, pk, pv, prefix_len) -> the output, or None
PyObject* prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 12) Py_RETURN_NONE;
  return attention(args, args + 9);
}

// adapters(x, segs, plan, ranks, scales, work) -> the list of y, or None
PyObject* adapters(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return attempt([&]() -> PyObject* {
    if (nargs != 6 || !PyList_Check(args[1])) throw Other{};
    const Py_ssize_t nseg = PyList_GET_SIZE(args[1]);
    if (nseg < 1 || nseg > 3) throw Other{};
    const int dev = device();
    const at::Tensor& x = plain(on(args[0], dev));
    if (x.dim() != 2 || x.size(0) < 1 || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX || (x.size(1) > 1 && x.stride(1) != 1))
      throw Other{};
    Kept kept;
    PyObject* oT = kept.attr(args[2], s_T);
    PyObject* on_ = kept.attr(args[2], s_n_adapters);
    const long T = PyLong_AsLong(oT), n = PyLong_AsLong(on_);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      throw Other{};
    }
    const at::Tensor& plan = on(kept.attr(args[2], s_plan), dev);
    if (T != x.size(0) || n < 1 || n > INT32_MAX || !plan.is_contiguous()) throw Other{};
    btf_adapters_args a{};
    at::Tensor out[3];
    PyObject* given[3];
    int64_t R = 0;
    bool typed = false;
    at::ScalarType y_type = x.scalar_type(), w_type = y_type;
    for (Py_ssize_t i = 0; i < nseg; ++i) {
      if (i >= PyList_GET_SIZE(args[1])) throw Other{};
      PyObject* s = kept.keep(PyList_GET_ITEM(args[1], i));
      PyObject *oa = kept.attr(s, s_a), *ob = kept.attr(s, s_b), *oy = kept.attr(s, s_y), *obase = kept.attr(s, s_base);
      const at::Tensor &wa = plain(on(oa, dev)), &wb = plain(on(ob, dev));
      if (wa.dim() != 3 || wb.dim() != 3) throw Other{};
      if (i == 0) R = wa.size(1), w_type = wa.scalar_type();
      const int64_t N = wb.size(1);
      if (wa.size(0) != n || wa.size(1) != R || wa.size(2) != x.size(1) || wb.size(0) != n || wb.size(2) != R ||
          wa.stride(2) != 1 || wb.stride(2) != 1 || wa.scalar_type() != w_type || wb.scalar_type() != w_type || R > INT32_MAX ||
          N < 1 || N > INT32_MAX)
        throw Other{};
      const at::Tensor* two[2] = {oy == Py_None ? nullptr : &plain(on(oy, dev)), obase == Py_None ? nullptr : &plain(on(obase, dev))};
      for (const at::Tensor* t : two) {
        if (!t) continue;
        if (t->dim() != 2 || t->size(0) != T || t->size(1) != N || (N > 1 && t->stride(1) != 1)) throw Other{};
        if (typed && t->scalar_type() != y_type) throw Other{};
        typed = true, y_type = t->scalar_type();
      }
      given[i] = oy;
      if (two[0]) out[i] = *two[0];
      btf_adapter_seg& c = a.segs[i];
      c = {wa.data_ptr(), wa.stride(0), wa.stride(1), wb.data_ptr(), wb.stride(0), wb.stride(1), (int)N,
           two[1] ? two[1]->data_ptr() : nullptr, two[1] ? two[1]->stride(0) : 0, nullptr, 0};
    }
    for (Py_ssize_t i = 0; i < nseg; ++i) {
      if (!out[i].defined()) out[i] = at::empty({T, a.segs[i].N}, x.options().dtype(y_type));
      a.segs[i].y = out[i].data_ptr(), a.segs[i].y_row = out[i].stride(0);
    }
    a.x = x.data_ptr(), a.x_row = x.stride(0);
    a.x_type = elem(x), a.w_type = w_type == at::kHalf ? BTF_F16 : w_type == at::kBFloat16 ? BTF_BF16 : BTF_F32;
    a.y_type = elem(out[0]);
    a.T = (int)T, a.K = (int)x.size(1), a.R = (int)R, a.n_adapters = (int)n, a.nseg = (int)nseg;
    a.ranks = vec<int32_t>(args[3], dev, at::kInt, n);
    a.scales = vec<float>(args[4], dev, at::kFloat, n);
    if (args[4] != Py_None) plain(tensor(args[4]));
    a.plan = plan.data_ptr(), a.plan_bytes = (int64_t)plan.nbytes();
    at::Tensor work;
    if (args[5] != Py_None) {
      work = on(args[5], dev);
      if (!work.is_contiguous()) throw Other{};
    } else {
      const int64_t bytes = lib.adapters_work(a.T, a.K, a.R, a.nseg, a.n_adapters);
      if (bytes < 0) throw Other{};
      work = at::empty({bytes}, x.options().dtype(at::kByte));
    }
    a.work = work.data_ptr(), a.work_bytes = (int64_t)work.nbytes();
    if (lib.adapters(&a, stream_of(dev))) throw Other{};
    PyObject* r = PyList_New(nseg);
    if (!r) return nullptr;
    for (Py_ssize_t i = 0; i < nseg; ++i) {
      written(out[i]);
      PyObject* y = given[i];
      if (y != Py_None) Py_INCREF(y);
      else y = THPVariable_Wrap(out[i]);
      PyList_SET_ITEM(r, i, y);
    }
    return r;
  });
}

// sample(logits, u, temperature, top_k, top_p, min_p, tokens, logprobs) -> (tokens, logprobs), or None
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return attempt([&]() -> PyObject* {
    if (nargs != 8) throw Other{};
    const int dev = device();
    const at::Tensor& x = on(args[0], dev);
    if (x.dim() != 2) throw Other{};
    const int64_t B = x.size(0), V = x.size(1);
    if (B < 1 || B > INT32_MAX || V < 1 || V > INT32_MAX || (V > 1 && x.stride(1) != 1) || args[1] == Py_None) throw Other{};
    const float* u = vec<float>(args[1], dev, at::kFloat, B);
    const float* temp = vec<float>(args[2], dev, at::kFloat, B);
    const int32_t* top_k = vec<int32_t>(args[3], dev, at::kInt, B);
    const float* top_p = vec<float>(args[4], dev, at::kFloat, B);
    const float* min_p = vec<float>(args[5], dev, at::kFloat, B);
    at::Tensor tokens, logprobs;
    if (args[6] != Py_None) {
      vec(args[6], dev, at::kInt, B);
      tokens = plain(tensor(args[6]));
    } else {
      tokens = at::empty({B}, x.options().dtype(at::kInt));
    }
    if (args[7] != Py_None) {
      vec(args[7], dev, at::kFloat, B);
      logprobs = plain(tensor(args[7]));
    } else {
      logprobs = at::empty({B}, x.options().dtype(at::kFloat));
    }
    if (lib.sample(x.data_ptr(), elem(x), B > 1 ? x.stride(0) : V, (int)B, (int)V, u, temp, top_k, top_p, min_p,
                   static_cast<int32_t*>(tokens.data_ptr()), static_cast<float*>(logprobs.data_ptr()), stream_of(dev)))
      throw Other{};
    written(tokens);
    written(logprobs);
    PyObject* t = args[6];
    PyObject* l = args[7];
    if (t != Py_None) Py_INCREF(t);
    else t = THPVariable_Wrap(tokens);
    if (l != Py_None) Py_INCREF(l);
    else l = THPVariable_Wrap(logprobs);
    PyObject* r = PyTuple_Pack(2, t, l);
    Py_XDECREF(t);
    Py_XDECREF(l);
    return r;
  });
}

// bind(rope, tree_attention_work, tree_attention, sample, rope_axes, prefix_attention_work, prefix_attention,
// adapters_work, adapters): addresses in the loaded library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8])) return nullptr;
  lib = {reinterpret_cast<decltype(lib.rope)>(a[0]),         reinterpret_cast<decltype(lib.tree_work)>(a[1]),
         reinterpret_cast<decltype(lib.tree)>(a[2]),         reinterpret_cast<decltype(lib.sample)>(a[3]),
         reinterpret_cast<decltype(lib.rope_axes)>(a[4]),    reinterpret_cast<decltype(lib.prefix_work)>(a[5]),
         reinterpret_cast<decltype(lib.prefix)>(a[6]),       reinterpret_cast<decltype(lib.adapters_work)>(a[7]),
         reinterpret_cast<decltype(lib.adapters)>(a[8])};
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"rope", (PyCFunction)(void (*)(void))rope, METH_FASTCALL, nullptr},
                         {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
                         {"prefix_attention", (PyCFunction)(void (*)(void))prefix_attention, METH_FASTCALL, nullptr},
                         {"adapters", (PyCFunction)(void (*)(void))adapters, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "btf_b200_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_btf_b200_calls() {
  s_x = PyUnicode_InternFromString("x");
  s_y = PyUnicode_InternFromString("y");
  s_normw = PyUnicode_InternFromString("normw");
  s_rotate = PyUnicode_InternFromString("rotate");
  s_rows = PyUnicode_InternFromString("rows");
  s_turns = PyUnicode_InternFromString("turns");
  s_n_rot = PyUnicode_InternFromString("n_rot");
  s_mscale = PyUnicode_InternFromString("mscale");
  s_interleaved = PyUnicode_InternFromString("interleaved");
  s_axis = PyUnicode_InternFromString("axis");
  s_n_axes = PyUnicode_InternFromString("n_axes");
  s_a = PyUnicode_InternFromString("a");
  s_b = PyUnicode_InternFromString("b");
  s_base = PyUnicode_InternFromString("base");
  s_plan = PyUnicode_InternFromString("plan");
  s_T = PyUnicode_InternFromString("T");
  s_n_adapters = PyUnicode_InternFromString("n_adapters");
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", BTF_TORCH_VERSION)) {  // the mirror binds it to no other
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
