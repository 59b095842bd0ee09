// bind.cpp — the Python side of the calls that a decode step makes for every layer (rotary positions, the 4-bit cache's
// append and reading, the attention over it, 8-bit products, routing and the experts' sum): the tensors' checks, the outputs'
// allocation and the C call.
//
// Why not in Python over ctypes as elsewhere: these kernels take 2 to 10 us for one token, and there the same checks took
// 5 us, the arguments' conversion 2 and the outputs 1.4 to 2.4 each. One token's rotation takes 5.6 us a call here and took
// 11.4, an append 5.2 and 15.3, an attention 7.6 and 18.6. (Quantisation takes 4.0, the experts' sum 4.1, routing 5.0, an 8-bit product 5.9.) The entry points of ops.py are the names and the documentation.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <initializer_list>

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

// ---- 8-bit products and experts ----
int float_kind(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? (int)UP_EK_F32 : half_kind(t); }

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& beside_it, at::ScalarType type) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return at::empty(sizes, beside_it.options().dtype(type));
}

// A tensor over part of another's memory: one allocation (1.3 us of the host) serves several outputs.
at::Tensor carve(const at::Tensor& all, int64_t byte, at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
  c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  impl->set_sizes_and_strides(sizes, strides);
  impl->set_storage_offset((all.storage_offset() + byte) / (int64_t)c10::elementSize(type));
  return t;
}
constexpr int64_t up_to(int64_t bytes) { return (bytes + 31) / 32 * 32; }

// The stream's workspace of this kind (ops.workspace's), or a captured graph's own, of which the first `counters` bytes are
// zero-filled within the graph.
at::Tensor workspace_of(const char* kind, PyObject* beside_it, int dev, void* stream, size_t bytes, size_t counters) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    at::Tensor ws = empty({(int64_t)bytes}, THPVariable_Unpack(beside_it), at::kByte);
    if (counters > 0) ws.narrow(0, 0, (int64_t)counters).zero_();
    return ws;
  }
  PyObject* key = Py_BuildValue("siK", kind, dev, (unsigned long long)reinterpret_cast<uintptr_t>(stream));
  if (!key) throw Raised();
  PyObject* held = PyDict_GetItemWithError(g_cache, key);
  Py_DECREF(key);
  if (held && (size_t)tensor(held, "workspace").nbytes() >= bytes) return tensor(held, "workspace");
  if (PyErr_Occurred()) throw Raised();
  PyObject* device = PyObject_GetAttrString(beside_it, "device");
  PyObject* made = device ? PyObject_CallFunction(g_workspace, "snO", kind, (Py_ssize_t)bytes, device) : nullptr;
  Py_XDECREF(device);
  if (!made) throw Raised();
  at::Tensor ws = tensor(made, "workspace");
  Py_DECREF(made);
  return ws;
}

PyObject* tuple_of(std::initializer_list<at::Tensor*> items) {
  PyObject* all = PyTuple_New((Py_ssize_t)items.size());
  if (!all) throw Raised();
  Py_ssize_t i = 0;
  for (at::Tensor* t : items) {
    PyObject* o = THPVariable_Wrap(std::move(*t));
    if (!o) {
      Py_DECREF(all);
      throw Raised();
    }
    PyTuple_SET_ITEM(all, i++, o);
  }
  return all;
}

// f8_quantise(x, rows, gate)
PyObject* f8_quantise(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 3);
    const at::Tensor& x = cuda_tensor(a[0], "x");
    const int kind = float_kind(x);
    need(kind >= 0 && x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1),
         "x is float32, float16 or bfloat16 [tokens, k] with contiguous rows");
    const int dev = current_device_of(x);
    const int gate = PyObject_IsTrue(a[2]);
    if (gate < 0) throw Raised();
    need(!gate || x.size(1) % 2 == 0, "with a gate, x holds 2k values a row");
    const int64_t k = gate ? x.size(1) / 2 : x.size(1);
    const int32_t* rows = nullptr;
    int64_t n_rows = x.size(0);
    if (given(a[1])) {
      const at::Tensor& r = tensor(a[1], "rows");
      need(r.scalar_type() == at::kInt && r.dim() == 1 && r.is_contiguous(), "rows is contiguous int32 [n]");
      beside(dev, r);
      rows = r.data_ptr<int32_t>(), n_rows = r.size(0);
    }
    const int64_t blocks = (k + 127) / 128;
    const int64_t q_bytes = up_to(n_rows * k);
    const at::Tensor all = empty({q_bytes + 4 * n_rows * blocks}, x, at::kByte);
    at::Tensor q = carve(all, 0, {n_rows, k}, {k, 1}, at::kFloat8_e4m3fn);
    at::Tensor scale = carve(all, q_bytes, {n_rows, blocks}, {1, n_rows}, at::kFloat);
    check(unlocked([&] {
            return up_sm100_f8_quantise(x.data_ptr(), kind, x.size(0), x.stride(0), rows, n_rows, k, gate,
                                        static_cast<uint8_t*>(q.data_ptr()), scale.data_ptr<float>(), 1, n_rows, stream_of(dev));
          }),
          "f8_quantise");
    return tuple_of({&q, &scale});
  });
}

// f8_quantise_weight(w)
PyObject* f8_quantise_weight(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 1);
    const at::Tensor& w = cuda_tensor(a[0], "w");
    const int kind = float_kind(w);
    const bool many = w.dim() == 3;
    need(kind >= 0 && (many || w.dim() == 2) && (w.stride(-1) == 1 || w.size(-1) <= 1),
         "w is float32, float16 or bfloat16 [n, k] or [experts, n, k] with contiguous rows");
    const int dev = current_device_of(w);
    const int64_t experts = many ? w.size(0) : 1, rows = w.size(-2), k = w.size(-1), bn = (rows + 127) / 128, bk = (k + 127) / 128;
    at::Tensor q, scale;
    if (many)
      q = empty({experts, rows, k}, w, at::kFloat8_e4m3fn), scale = empty({experts, bn, bk}, w, at::kFloat);
    else
      q = empty({rows, k}, w, at::kFloat8_e4m3fn), scale = empty({bn, bk}, w, at::kFloat);
    check(unlocked([&] {
            return up_sm100_f8_quantise_weight(w.data_ptr(), kind, experts, rows, k, many ? w.stride(0) : 0, w.stride(-2),
                                               static_cast<uint8_t*>(q.data_ptr()), scale.data_ptr<float>(), stream_of(dev));
          }),
          "f8_quantise_weight");
    return tuple_of({&q, &scale});
  });
}

// f8_matmul(x, x_scale, w, w_scale, offsets, dtype, out, ws): offsets None for one matrix
PyObject* f8_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 8);
    const bool many = given(a[4]);
    const char* name = many ? "f8_expert_matmul" : "f8_matmul";
    const at::Tensor &x = cuda_tensor(a[0], "x"), &xs = tensor(a[1], "x_scale"), &w = tensor(a[2], "w"), &ws = tensor(a[3], "w_scale");
    const int dev = current_device_of(x);
    need(x.scalar_type() == at::kFloat8_e4m3fn && x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1),
         "x is float8_e4m3fn [rows, k] with contiguous rows");
    const int64_t m = x.size(0), k = x.size(1), kb = (k + 127) / 128;
    need(w.scalar_type() == at::kFloat8_e4m3fn && w.dim() == (many ? 3 : 2) && w.size(-1) == k && w.is_contiguous(),
         many ? "w is float8_e4m3fn [experts, n, k] of x's k, contiguous" : "w is float8_e4m3fn [n, k] of x's k, contiguous");
    const int64_t experts = many ? w.size(0) : 1, cols = w.size(-2), nb = (cols + 127) / 128;
    need(xs.scalar_type() == at::kFloat && xs.dim() == 2 && xs.size(0) == m && xs.size(1) == kb,
         "x_scale is float32 [rows, ceil(k / 128)]");
    need(ws.scalar_type() == at::kFloat && ws.dim() == w.dim() && ws.size(-2) == nb && ws.size(-1) == kb &&
             (!many || ws.size(0) == experts) && ws.is_contiguous(),
         "w_scale is float32 [ceil(n / 128), ceil(k / 128)], for each expert, contiguous");
    beside(dev, xs), beside(dev, w), beside(dev, ws);
    const int32_t* offsets = nullptr;
    if (many) {
      const at::Tensor& o = tensor(a[4], "offsets");
      need(o.scalar_type() == at::kInt && o.dim() == 1 && o.size(0) == experts + 1 && o.is_contiguous(),
           "offsets is contiguous int32 [experts + 1]");
      beside(dev, o);
      offsets = o.data_ptr<int32_t>();
    }
    at::Tensor out;
    if (given(a[6])) {
      out = tensor(a[6], "out");
      need(out.dim() == 2 && out.size(0) == m && out.size(1) == cols && (out.stride(1) == 1 || cols <= 1),
           "out is [rows, n] with contiguous rows");
      beside(dev, out);
    } else {
      need(THPDtype_Check(a[5]), "dtype is a torch dtype");
      const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
      need(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, "dtype is float32, float16 or bfloat16");
      out = empty({m, cols}, x, type);
    }
    const int kind = float_kind(out);
    need(kind >= 0, "out is float32, float16 or bfloat16");
    void* stream = stream_of(dev);
    at::Tensor space;
    if (given(a[7])) {
      space = tensor(a[7], "ws");
      beside(dev, space);
      need(space.is_contiguous(), "ws is contiguous");
    } else {
      space = workspace_of("f8", a[0], dev, stream, up_sm100_f8_matmul_workspace_bytes(m, experts, cols, k), UP_F8_COUNTER_BYTES);
    }
    check(unlocked([&] {
            return up_sm100_f8_matmul(static_cast<const uint8_t*>(x.data_ptr()), m, x.stride(0), xs.data_ptr<float>(), xs.stride(0),
                                      xs.stride(1), static_cast<const uint8_t*>(w.data_ptr()), ws.data_ptr<float>(), experts, cols, k,
                                      offsets, out.data_ptr(), kind, out.stride(0), space.data_ptr(), space.nbytes(), stream);
          }),
          name);
    if (given(a[6])) {
      Py_INCREF(a[6]);
      return a[6];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// expert_route(logits, k, score, renormalise, gain)
PyObject* expert_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 5);
    const at::Tensor& l = cuda_tensor(a[0], "logits");
    const int kind = float_kind(l);
    need(kind >= 0 && l.dim() == 2 && (l.stride(1) == 1 || l.size(1) <= 1),
         "logits is float32, float16 or bfloat16 [tokens, experts] with contiguous rows");
    const int dev = current_device_of(l);
    const int64_t tokens = l.size(0), experts = l.size(1), k = PyLong_AsLongLong(a[1]);
    if (k == -1 && PyErr_Occurred()) throw Raised();
    need(k >= 1 && k <= experts, "k is from 1 to the number of experts");
    int score = -1;
    if (PyUnicode_Check(a[2])) {
      if (PyUnicode_CompareWithASCIIString(a[2], "softmax") == 0) score = UP_EXPERT_SOFTMAX;
      if (PyUnicode_CompareWithASCIIString(a[2], "sigmoid") == 0) score = UP_EXPERT_SIGMOID;
    }
    need(score >= 0, "score is \"softmax\" or \"sigmoid\"");
    const int renormalise = PyObject_IsTrue(a[3]);
    if (renormalise < 0) throw Raised();
    const double gain = PyFloat_AsDouble(a[4]);
    if (gain == -1.0 && PyErr_Occurred()) throw Raised();
    const int64_t pairs = up_to(4 * tokens * k);
    const at::Tensor all = empty({4 * pairs + 4 * (experts + 1)}, l, at::kByte);
    at::Tensor ids = carve(all, 0, {tokens, k}, {k, 1}, at::kInt), weights = carve(all, pairs, {tokens, k}, {k, 1}, at::kFloat),
               rows = carve(all, 2 * pairs, {tokens * k}, {1}, at::kInt), slots = carve(all, 3 * pairs, {tokens, k}, {k, 1}, at::kInt),
               offsets = carve(all, 4 * pairs, {experts + 1}, {1}, at::kInt);
    void* stream = stream_of(dev);
    const at::Tensor ws = workspace_of("route", a[0], dev, stream, up_sm100_expert_route_workspace_bytes(tokens, experts), 0);
    check(unlocked([&] {
            return up_sm100_expert_route(l.data_ptr(), kind, tokens, experts, l.stride(0), k, score, renormalise, (float)gain,
                                         ids.data_ptr<int32_t>(), weights.data_ptr<float>(), rows.data_ptr<int32_t>(),
                                         slots.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), ws.data_ptr(), ws.nbytes(), stream);
          }),
          "expert_route");
    return tuple_of({&ids, &weights, &rows, &slots, &offsets});
  });
}

// expert_combine(y, slots, weights, add, out)
PyObject* expert_combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 5);
    const at::Tensor &y = cuda_tensor(a[0], "y"), &slots = tensor(a[1], "slots"), &weights = tensor(a[2], "weights");
    const int kind = float_kind(y);
    need(kind >= 0 && y.dim() == 2 && (y.stride(1) == 1 || y.size(1) <= 1), "y is float32, float16 or bfloat16 [rows, n] with contiguous rows");
    const int dev = current_device_of(y);
    need(slots.scalar_type() == at::kInt && slots.dim() == 2 && slots.is_contiguous(), "slots is contiguous int32 [tokens, k]");
    need(weights.scalar_type() == at::kFloat && weights.sizes() == slots.sizes() && weights.is_contiguous(),
         "weights is contiguous float32 of slots' shape");
    beside(dev, slots), beside(dev, weights);
    const int64_t tokens = slots.size(0), cols = y.size(1);
    const void* add = nullptr;
    int64_t add_stride = 0;
    if (given(a[3])) {
      const at::Tensor& t = tensor(a[3], "add");
      need(t.dim() == 2 && t.size(0) == tokens && t.size(1) == cols && t.scalar_type() == y.scalar_type() && (t.stride(1) == 1 || cols <= 1),
           "add is [tokens, n] of y's type with contiguous rows");
      beside(dev, t);
      add = t.data_ptr(), add_stride = t.stride(0);
    }
    at::Tensor out;
    if (given(a[4])) {
      out = tensor(a[4], "out");
      need(out.dim() == 2 && out.size(0) == tokens && out.size(1) == cols && out.scalar_type() == y.scalar_type() &&
               (out.stride(1) == 1 || cols <= 1),
           "out is [tokens, n] of y's type with contiguous rows");
      beside(dev, out);
    } else {
      out = empty({tokens, cols}, y, y.scalar_type());
    }
    check(unlocked([&] {
            return up_sm100_expert_combine(y.data_ptr(), kind, y.size(0), y.stride(0), cols, slots.data_ptr<int32_t>(),
                                           weights.data_ptr<float>(), tokens, slots.size(1), add, add_stride, out.data_ptr(),
                                           out.stride(0), stream_of(dev));
          }),
          "expert_combine");
    if (given(a[4])) {
      Py_INCREF(a[4]);
      return a[4];
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
    {"f8_quantise", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f8_quantise)), METH_FASTCALL, nullptr},
    {"f8_quantise_weight", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f8_quantise_weight)), METH_FASTCALL, nullptr},
    {"f8_matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f8_matmul)), METH_FASTCALL, nullptr},
    {"expert_route", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(expert_route)), METH_FASTCALL, nullptr},
    {"expert_combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(expert_combine)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
