// bind.cpp — the Python side of the calls that a decode step makes for every layer (rotary positions, the 4-bit cache's
// append and reading, the attention over it): the tensors' checks, the outputs' allocation and the C call.
//
// Why not in Python over ctypes as elsewhere: these kernels take 2 to 10 us for one token, and there the same checks took
// 5 us, the arguments' conversion 2 and the outputs 1.4 to 2.4 each. One token's rotation takes 5.6 us a call here and took
// 11.4, an append 5.2 and 15.3, an attention 7.6 and 18.6. The entry points of ops.py are the names and the documentation.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>

#include "up_sm100.h"

namespace {

struct Raised : std::exception {};  // a Python error is set

[[noreturn]] void raise(PyObject* kind, const char* text) {
  PyErr_SetString(kind, text);
  throw Raised();
}
void need(bool ok, const char* text) {
  if (!ok) raise(PyExc_ValueError, text);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw Raised();
  }
  return THPVariable_Unpack(o);
}
// The tensor that the others have to lie beside.
const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) {
    PyErr_Format(PyExc_TypeError, "%s must be a CUDA tensor", name);
    throw Raised();
  }
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }

int current_device_of(const at::Tensor& t) {
  const int dev = t.get_device();
  need(dev == c10::cuda::current_device(), "the tensors must be on the current CUDA device");
  return dev;
}
void beside(int dev, const at::Tensor& t) { need(t.is_cuda() && t.get_device() == dev, "all tensors must be on one CUDA device"); }
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

int index_kind(const at::Tensor& t) {
  return t.scalar_type() == at::kInt ? UP_EK_I32 : t.scalar_type() == at::kLong ? UP_EK_I64 : -1;
}
int half_kind(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? UP_EK_BF16 : t.scalar_type() == at::kHalf ? UP_EK_F16 : -1;
}
int layout_of(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return UP_ROPE_HALF;
    if (PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) return UP_ROPE_INTERLEAVED;
  }
  PyErr_SetObject(PyExc_KeyError, o);
  throw Raised();
}
void check_table(const at::Tensor& t) {
  need(t.scalar_type() == at::kFloat && t.dim() == 2 && t.is_contiguous(), "table is float32 [positions, rot], contiguous (rope_table)");
}
at::Tensor new_like(const at::Tensor& t) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return at::empty_like(t);
}

PyObject* g_check = nullptr;      // _lib.check(status, where)
PyObject* g_workspace = nullptr;  // ops.workspace(kind, nbytes, device)
PyObject* g_cache = nullptr;      // its dict: (kind, device, stream) -> tensor

void check(int status, const char* where) {
  if (status == UP_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", status, where);
  if (r) {
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, where);
  }
  throw Raised();
}

// The library's call without the interpreter's lock: a launch waits where the device's queue is full.
template <typename F>
int unlocked(F f) {
  struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
  } here;
  return f();
}

// Runs `f` and turns C++ exceptions into Python's.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Raised&) {
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) raise(PyExc_TypeError, "wrong number of arguments");
}

// rope(x, positions, table, layout, out, backward)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 6);
    const at::Tensor& x = cuda_tensor(a[0], "x");
    const int backward = a[5] == Py_True;
    const int kind = x.scalar_type() == at::kFloat ? (int)UP_EK_F32 : half_kind(x);
    const bool four = x.dim() == 4;
    need(kind >= 0 && (four || x.dim() == 3) && (x.stride(-1) == 1 || x.size(-1) <= 1),
         "x is float32, float16 or bfloat16 [tokens, heads, dim] or [batch, seq, heads, dim] with the dimension contiguous");
    const int64_t batch = four ? x.size(0) : 1, seq = x.size(-3), heads = x.size(-2), dim = x.size(-1);
    const at::Tensor& table = tensor(a[2], "table");
    check_table(table);
    const int dev = current_device_of(x);
    beside(dev, table);
    const void* pos = nullptr;
    int pos_kind = 0;
    int64_t pos_stride = 0;
    if (given(a[1])) {
      const at::Tensor& p = tensor(a[1], "positions");
      pos_kind = index_kind(p);
      need(pos_kind >= 0 && p.is_contiguous(), "positions are contiguous int32 or int64");
      if (four && p.dim() == 2 && p.size(0) == batch && p.size(1) == seq)
        pos_stride = seq;
      else
        need(p.dim() == 1 && p.size(0) == seq, "positions are one a token: [tokens], [seq] or [batch, seq]");
      beside(dev, p);
      pos = p.data_ptr();
    }
    const int layout = layout_of(a[3]);
    at::Tensor out;
    if (given(a[4])) {
      out = tensor(a[4], "out");
      need(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && (out.stride(-1) == 1 || dim <= 1),
           "out has x's shape and type, with the dimension contiguous");
      beside(dev, out);
    } else {
      out = new_like(x);
    }
    check(unlocked([&] {
            return up_sm100_rope(x.data_ptr(), kind, batch, seq, heads, dim, four ? x.stride(0) : 0, x.stride(-3), x.stride(-2), pos,
                          pos_kind, pos_stride, table.data_ptr<float>(), table.size(0), table.size(1), layout, backward, out.data_ptr(),
                        four ? out.stride(0) : 0, out.stride(-3), out.stride(-2), stream_of(dev));
          }),
          backward ? "rope_backward" : "rope");
    if (given(a[4])) {
      Py_INCREF(a[4]);
      return a[4];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

up_kv4_cache cache_of(PyObject* o, int dev) {
  if (!PyTuple_Check(o) && !PyList_Check(o)) raise(PyExc_TypeError, "a cache is a tuple (k, v, k_scale, v_scale)");
  need(PySequence_Fast_GET_SIZE(o) == 4, "a cache is (k, v, k_scale, v_scale)");
  PyObject** items = PySequence_Fast_ITEMS(o);
  const at::Tensor &k = tensor(items[0], "k"), &v = tensor(items[1], "v"), &ks = tensor(items[2], "k_scale"),
                   &vs = tensor(items[3], "v_scale");
  need(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte && ks.scalar_type() == at::kHalf && vs.scalar_type() == at::kHalf,
       "a cache is (k uint8, v uint8, k_scale float16, v_scale float16)");
  need(k.dim() == 4 && ks.dim() == 4 && v.sizes() == k.sizes() && vs.sizes() == ks.sizes() && ks.size(0) == k.size(0) &&
           ks.size(1) == k.size(1) && ks.size(2) == k.size(2),
       "cache arrays are [pages, kv_heads, page, dim/2] and [pages, kv_heads, page, dim/group]");
  need(k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(), "cache arrays are contiguous");
  const int64_t dim = 2 * k.size(3), groups = ks.size(3);
  need(groups > 0 && dim % groups == 0, "the scales' groups divide the head size");
  beside(dev, k), beside(dev, v), beside(dev, ks), beside(dev, vs);
  up_kv4_cache c{};
  c.k = k.data_ptr(), c.v = v.data_ptr(), c.k_scale = ks.data_ptr(), c.v_scale = vs.data_ptr();
  c.pages = k.size(0), c.kv_heads = k.size(1), c.page = k.size(2), c.dim = dim, c.group = dim / groups;
  return c;
}

// kv4_append(k, v, cache, slots, positions, table, q, layout, q_out)
PyObject* kv4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 9);
    const at::Tensor &k = cuda_tensor(a[0], "k"), &v = tensor(a[1], "v");
    const int dev = current_device_of(k);
    const up_kv4_cache c = cache_of(a[2], dev);
    const int kind = half_kind(k);
    need(kind >= 0 && v.scalar_type() == k.scalar_type(), "kv4_append takes bfloat16 or float16, q, k and v alike");
    need(k.dim() == 3 && k.size(1) == c.kv_heads && k.size(2) == c.dim && v.sizes() == k.sizes() && k.stride(2) == 1 && v.stride(2) == 1,
         "k and v are [tokens, kv_heads, dim] of the cache, with the dimension contiguous");
    beside(dev, v);
    const int64_t tokens = k.size(0);
    const at::Tensor& slots = tensor(a[3], "slots");
    const int slot_kind = index_kind(slots);
    need(slot_kind >= 0 && slots.dim() == 1 && slots.size(0) == tokens && slots.is_contiguous(),
         "slots are contiguous int32 or int64, one a token");
    beside(dev, slots);
    const void* pos = nullptr;
    const float* table = nullptr;
    int pos_kind = 0;
    int64_t n_pos = 0, rot = 0;
    if (given(a[5])) {
      const at::Tensor& t = tensor(a[5], "table");
      check_table(t);
      need(given(a[4]), "positions are contiguous int32 or int64, one a token");
      const at::Tensor& p = tensor(a[4], "positions");
      pos_kind = index_kind(p);
      need(pos_kind >= 0 && p.dim() == 1 && p.size(0) == tokens && p.is_contiguous(),
           "positions are contiguous int32 or int64, one a token");
      beside(dev, t), beside(dev, p);
      pos = p.data_ptr(), table = t.data_ptr<float>(), n_pos = t.size(0), rot = t.size(1);
    }
    const int layout = layout_of(a[7]);
    at::Tensor out;
    const void* q_ptr = nullptr;
    void* out_ptr = nullptr;
    int64_t heads = 0, qs = 0, qh = 0, qos = 0, qoh = 0;
    if (given(a[6])) {
      const at::Tensor& q = tensor(a[6], "q");
      need(q.dim() == 3 && q.scalar_type() == k.scalar_type() && q.size(0) == tokens && q.size(2) == c.dim && q.stride(2) == 1,
           "q is [tokens, heads, dim] of k's type, with the dimension contiguous");
      beside(dev, q);
      if (given(a[8])) {
        out = tensor(a[8], "q_out");
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1,
             "q_out has q's shape and type, with the dimension contiguous");
        beside(dev, out);
      } else {
        out = new_like(q);
      }
      heads = q.size(1), qs = q.stride(0), qh = q.stride(1), qos = out.stride(0), qoh = out.stride(1);
      q_ptr = q.data_ptr(), out_ptr = out.data_ptr();
    } else {
      need(!given(a[8]), "q_out without q");
    }
    check(unlocked([&] {
            return up_sm100_kv4_append(q_ptr, k.data_ptr(), v.data_ptr(), kind, tokens, heads, qs, qh, k.stride(0), k.stride(1), v.stride(0),
                              v.stride(1), pos, pos_kind, table, n_pos, rot, layout, slots.data_ptr(), slot_kind, &c, out_ptr, qos, qoh,
                              stream_of(dev));
          }),
          "kv4_append");
    if (given(a[6]) && !given(a[8])) return THPVariable_Wrap(std::move(out));
    Py_INCREF(a[8]);  // q_out, or None
    return a[8];
  });
}

// kv4_attention(q, cache, block_table, seq_lens, cu_q, causal, window, scale, out, want_lse, ws)
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 11);
    const at::Tensor& q = cuda_tensor(a[0], "q");
    const int dev = current_device_of(q);
    const up_kv4_cache c = cache_of(a[1], dev);
    const int kind = half_kind(q);
    need(kind >= 0 && q.dim() == 3 && q.size(2) == c.dim && q.stride(2) == 1,
         "q is bfloat16 or float16 [tokens, heads, dim] of the cache's dim, with the dimension contiguous");
    const int64_t tokens = q.size(0), heads = q.size(1);
    need(c.kv_heads > 0 && heads % c.kv_heads == 0, "q's heads are a multiple of the cache's");
    const at::Tensor &table = tensor(a[2], "block_table"), &lens = tensor(a[3], "seq_lens");
    need(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.is_contiguous(), "seq_lens is contiguous int32 [batch]");
    const int64_t batch = lens.size(0);
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == batch && (table.stride(1) == 1 || table.size(1) <= 1),
         "block_table is int32 [batch, width] with contiguous rows");
    beside(dev, table), beside(dev, lens);
    const int32_t* cu = nullptr;
    if (given(a[4])) {
      const at::Tensor& t = tensor(a[4], "cu_q");
      need(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == batch + 1 && t.is_contiguous(), "cu_q is contiguous int32 [batch + 1]");
      beside(dev, t);
      cu = t.data_ptr<int32_t>();
    } else {
      need(tokens == batch, "without cu_q there is one query token a sequence");
    }
    const int causal = PyObject_IsTrue(a[5]);
    if (causal < 0) throw Raised();
    const int64_t window = PyLong_AsLongLong(a[6]);
    if (window == -1 && PyErr_Occurred()) throw Raised();
    need(window >= 0, "window is not negative");
    const double scale = PyFloat_AsDouble(a[7]);
    if (scale == -1.0 && PyErr_Occurred()) throw Raised();
    at::Tensor out, lse;
    if (given(a[8])) {
      out = tensor(a[8], "out");
      need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1,
           "out has q's shape and type, with the dimension contiguous");
      beside(dev, out);
    } else {
      out = new_like(q);
    }
    const int want_lse = PyObject_IsTrue(a[9]);
    if (want_lse < 0) throw Raised();
    if (want_lse) {
      at::AutoDispatchBelowADInplaceOrView guard;
      lse = at::empty({tokens, heads}, q.options().dtype(at::kFloat));
    }
    void* stream = stream_of(dev);
    at::Tensor ws;
    if (given(a[10])) {
      ws = tensor(a[10], "ws");
      beside(dev, ws);
      need(ws.is_contiguous(), "ws is contiguous");
    } else if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
      // A graph has a workspace of its own, as ops.workspace's have; of this kind only the counters need be zero (the
      // fill of all of it takes 2 us).
      ws = at::empty({(int64_t)up_sm100_kv4_attention_workspace_bytes(tokens, heads, batch, c.kv_heads, c.dim)},
                     q.options().dtype(at::kByte));
      ws.narrow(0, 0, (int64_t)up_sm100_kv4_attention_workspace_bytes(0, heads, batch, c.kv_heads, c.dim)).zero_();
    } else {
      const size_t bytes = up_sm100_kv4_attention_workspace_bytes(tokens, heads, batch, c.kv_heads, c.dim);
      PyObject* key = Py_BuildValue("siK", "kv4", dev, (unsigned long long)reinterpret_cast<uintptr_t>(stream));
      key = key ? key : throw Raised();
      PyObject* held = PyDict_GetItemWithError(g_cache, key);
      Py_DECREF(key);
      if (held && (size_t)tensor(held, "workspace").nbytes() >= bytes) {
        ws = tensor(held, "workspace");
      } else {
        if (PyErr_Occurred()) throw Raised();
        PyObject* device = PyObject_GetAttrString(a[0], "device");
        PyObject* made = device ? PyObject_CallFunction(g_workspace, "snO", "kv4", (Py_ssize_t)bytes, device) : nullptr;
        Py_XDECREF(device);
        if (!made) throw Raised();
        ws = tensor(made, "workspace");
        Py_DECREF(made);
      }
    }
    check(unlocked([&] {
            return up_sm100_kv4_attention(q.data_ptr(), kind, tokens, heads, q.stride(0), q.stride(1), &c, table.data_ptr<int32_t>(),
                                 table.stride(0), table.size(1), lens.data_ptr<int32_t>(), cu, batch, causal, window, (float)scale,
                                 out.data_ptr(), out.stride(0), out.stride(1), want_lse ? lse.data_ptr<float>() : nullptr, heads,
                                 ws.data_ptr(), ws.nbytes(), stream);
          }),
          "kv4_attention");
    PyObject* o = a[8];
    if (given(o))
      Py_INCREF(o);
    else
      o = THPVariable_Wrap(std::move(out));
    if (!o || !want_lse) return o;
    PyObject* l = THPVariable_Wrap(std::move(lse));
    PyObject* both = l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_DECREF(o);
    Py_XDECREF(l);
    return both;
  });
}

// dequant_i4(w, scale, group, out): the cache's rows as values, among others
PyObject* dequant_i4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 4);
    const at::Tensor &w = cuda_tensor(a[0], "w"), &scale = cuda_tensor(a[1], "scale");
    need(w.dim() == 2, "w is [n, k / 2]");
    const int64_t rows = w.size(0), k = 2 * w.size(1), group = PyLong_AsLongLong(a[2]);
    if (group == -1 && PyErr_Occurred()) throw Raised();
    at::Tensor out;
    if (given(a[3])) {
      out = tensor(a[3], "out");
    } else {
      at::AutoDispatchBelowADInplaceOrView guard;
      out = at::empty({rows, k}, w.options().dtype(at::kBFloat16));
    }
    check(unlocked([&] {
            return up_sm100_dequant_i4_bf16(static_cast<const uint8_t*>(w.data_ptr()), static_cast<const uint16_t*>(scale.data_ptr()),
                                            rows, k, group, static_cast<uint16_t*>(out.data_ptr()), stream_of(w.get_device()));
          }),
          "dequant_i4");
    if (given(a[3])) {
      Py_INCREF(a[3]);
      return a[3];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// init(check, workspace, workspaces)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 3);
    if (!PyDict_Check(a[2])) raise(PyExc_TypeError, "the workspaces are a dict");
    for (int i = 0; i < 3; ++i) Py_INCREF(a[i]);
    Py_XDECREF(g_check), Py_XDECREF(g_workspace), Py_XDECREF(g_cache);
    g_check = a[0], g_workspace = a[1], g_cache = a[2];
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {
    {"init", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(init)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope)), METH_FASTCALL, nullptr},
    {"kv4_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_append)), METH_FASTCALL, nullptr},
    {"dequant_i4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequant_i4)), METH_FASTCALL, nullptr},
    {"kv4_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
