// CPython bindings that take torch tensors, for calls that a decode step makes once per layer.
//
// The Python wrappers of engine/hip_attn.py and kv/quant_cache.py read some forty attributes of their
// tensors, at a tenth of a microsecond each, which is most of a small call's time.  These functions
// read them in C++ and make the call where every argument is as the library takes it; where one is not
// (another type or layout, a CPU tensor, a bad value) they return None, having done nothing, and the
// wrapper goes on with its own checks, conversions and messages.  The stream and whether the tensors'
// device is the current one come from the wrapper.  The library's entry points are called through the
// addresses that dispec_amd._lib hands to bind(), as in fastcall.c.  Built with g++ (no device code).
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>
#include <limits>

#include "../../include/dispec_hip.h"

namespace {

decltype(&dsp_paged_window_attention) p_window;
decltype(&dsp_paged_window_workspace_bytes) p_window_bytes;
decltype(&dsp_kv_append_quant) p_append;
decltype(&dsp_kv_gather_quant) p_gather;

// An argument that is not as the library takes it.
struct Slow {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw Slow{};
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  if (!PyLong_CheckExact(o)) throw Slow{};
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Slow{};
  }
  return v;
}
int32_t integer32(PyObject* o) {
  const int64_t v = integer(o);
  if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max()) throw Slow{};
  return int32_t(v);
}
void need(bool ok) {
  if (!ok) throw Slow{};
}
int32_t dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return DSP_BF16;
  if (t == at::kHalf) return DSP_F16;
  need(t == at::kFloat);
  return DSP_F32;
}
// A dense int32 vector or matrix on `device`.
const int32_t* ints(const at::Tensor& t, at::Device device, int64_t dim) {
  need(t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous() && t.device() == device);
  return static_cast<const int32_t*>(t.const_data_ptr());
}
int32_t* counter(PyObject* o, at::Device device) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o);
  need(t.scalar_type() == at::kInt && t.numel() >= 1 && t.device() == device);
  return static_cast<int32_t*>(t.data_ptr());
}

// window(q, k_cache, k_scale, v_cache, v_scale, block_table, cu_q, ctx_lens, kv_groups, window, sinks,
//        block_size, scale, max_q_len, max_ctx, out, err, workspace, stream) -> out or None
PyObject* window(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[3]);
  const at::Device device = q.device();
  need(device.is_cuda() && k.device() == device && v.device() == device);
  need(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.strides() == v.strides());
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), S = k.size(0), KVH = k.size(1);
  need(q.stride(2) == 1 && k.stride(2) == 1 && Hq == KVH * integer(a[8]));
  const int32_t dtype = dtype_code(q.scalar_type());
  int32_t format = DSP_KV_PLAIN;
  const uint8_t *ks = nullptr, *vs = nullptr;
  int64_t s_slot = 0, s_head = 0;
  if (a[2] == Py_None) {
    need(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.size(2) == D);
  } else {
    const at::Tensor &x = tensor(a[2]), &y = tensor(a[4]);
    need(D == 64 || D == 128 || D == 256);
    need(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte &&
         x.scalar_type() == at::kByte && y.scalar_type() == at::kByte);
    need(k.size(2) == D || 2 * k.size(2) == D);
    need(x.dim() == 3 && x.size(0) == S && x.size(1) == KVH && x.size(2) * 32 == D &&
         x.sizes() == y.sizes() && x.strides() == y.strides() && x.stride(2) == 1 &&
         x.device() == device && y.device() == device);
    format = k.size(2) == D ? DSP_KV_FP8 : DSP_KV_FP4;
    ks = static_cast<const uint8_t*>(x.const_data_ptr());
    vs = static_cast<const uint8_t*>(y.const_data_ptr());
    s_slot = x.stride(0);
    s_head = x.stride(1);
  }
  const at::Tensor &table = tensor(a[5]), &lens = tensor(a[7]);
  const int32_t *bt = ints(table, device, 2), *ctx_lens = ints(lens, device, 1), *cu = nullptr;
  const int64_t B = lens.numel();
  need(table.size(0) == B && B > 0 && B <= 65535 && T > 0);
  int32_t max_q_len = 1;
  if (a[6] == Py_None) {
    need(T == B);
  } else {
    const at::Tensor& c = tensor(a[6]);
    cu = ints(c, device, 1);
    need(c.numel() == B + 1);
    max_q_len = integer32(a[13]);
    need(max_q_len > 0);
  }
  const int32_t win = integer32(a[9]), sinks = integer32(a[10]), bs = integer32(a[11]);
  need(win >= 0 && sinks >= 0 && (win > 0 || sinks == 0) && bs > 0);
  const int64_t most = table.size(1) * int64_t(bs);
  const int64_t max_ctx = a[14] == Py_None ? most : integer(a[14]);
  need(max_ctx >= 0 && max_ctx <= most && max_ctx <= std::numeric_limits<int32_t>::max());
  double scale = 1.0 / std::sqrt(double(D));
  if (a[12] != Py_None) {
    need(PyFloat_CheckExact(a[12]));
    scale = PyFloat_AS_DOUBLE(a[12]);
    need(a[2] == Py_None || (scale > 0 && std::isfinite(scale)));
  }
  int32_t* const err = counter(a[16], device);
  at::Tensor out;
  if (a[15] == Py_None) {
    out = at::empty_like(q);
  } else {
    out = tensor(a[15]);
    need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1 &&
         out.device() == device);
  }
  need(S <= std::numeric_limits<int64_t>::max() / 2 && Hq <= 65535 && D <= 256);
  const size_t bytes = p_window_bytes(int32_t(B), int32_t(Hq), int32_t(KVH), int32_t(D), max_q_len,
                                      int32_t(max_ctx), win, sinks, format, dtype);
  at::Tensor ws;
  if (bytes) {
    if (a[17] != Py_None) {
      ws = tensor(a[17]);
      need(ws.device() == device && ws.is_contiguous());
    }
    if (!ws.defined() || size_t(ws.nbytes()) < bytes)  // (from the stream-ordered allocator)
      ws = at::empty({int64_t(bytes / 4)}, q.options().dtype(at::kFloat));
  }
  void* const stream = PyLong_AsVoidPtr(a[18]);
  const int64_t es = k.element_size();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = p_window(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(),
                    v.const_data_ptr(), S, k.stride(0) * es, k.stride(1) * es, ks, vs, s_slot, s_head,
                    format, bt, table.size(1), bs, cu, ctx_lens, int32_t(B), int32_t(Hq), int32_t(KVH),
                    int32_t(D), float(scale), win, sinks, max_q_len, int32_t(max_ctx),
                    bytes ? ws.data_ptr() : nullptr, bytes, out.data_ptr(), out.stride(0),
                    out.stride(1), dtype, err, stream);
  Py_END_ALLOW_THREADS
  need(status == DSP_OK);  // (nothing was launched: the wrapper finds the same and says so)
  return THPVariable_Wrap(out);
}

// The pools of a quantised cache, of one layer (S, KVH, width) or all.
struct Pools {
  const at::Tensor &kc, &ks, &vc, &vs;
  at::Device device;
  int64_t L, S, KVH, D, code_layer, code_slot, scale_layer, scale_slot;
  int32_t format;
  bool layers;
  explicit Pools(PyObject* const* a)
      : kc(tensor(a[0])), ks(tensor(a[1])), vc(tensor(a[2])), vs(tensor(a[3])), device(kc.device()) {
    for (const at::Tensor* t : {&kc, &ks, &vc, &vs})
      need(t->scalar_type() == at::kByte && t->device() == device);
    const int64_t n = kc.dim();
    need(device.is_cuda() && (n == 3 || n == 4) && ks.dim() == n && vc.sizes() == kc.sizes() &&
         vs.sizes() == ks.sizes() && vc.strides() == kc.strides() && vs.strides() == ks.strides());
    layers = n == 4;
    const int64_t i = n - 3, width = kc.size(i + 2), groups = ks.size(i + 2);
    S = kc.size(i);
    KVH = kc.size(i + 1);
    D = 32 * groups;
    L = layers ? kc.size(0) : 1;
    need(ks.size(i) == S && ks.size(i + 1) == KVH && ks.size(0) == kc.size(0) &&
         (width == D || 2 * width == D));
    need(kc.stride(i + 2) == 1 && ks.stride(i + 2) == 1 &&
         (KVH == 1 || (kc.stride(i + 1) == width && ks.stride(i + 1) == groups)));
    code_layer = layers ? kc.stride(0) : 0;
    scale_layer = layers ? ks.stride(0) : 0;
    code_slot = kc.stride(i);
    scale_slot = ks.stride(i);
    format = width == D ? DSP_KV_FP8 : DSP_KV_FP4;
    need(L > 0 && KVH > 0 && KVH <= 65535 && D > 0 && D <= 65536);
  }
};

const int64_t* slots_of(const at::Tensor& t, const Pools& p) {
  need(t.scalar_type() == at::kLong && t.is_contiguous() && t.device() == p.device && t.numel() > 0);
  return static_cast<const int64_t*>(t.const_data_ptr());
}

// append(k_cache, k_scale, v_cache, v_scale, slots, k, v, err, stream) -> True or None
PyObject* append(PyObject* const* a) {
  const Pools p(a);
  const at::Tensor &slots = tensor(a[4]), &k = tensor(a[5]), &v = tensor(a[6]);
  const int64_t* s = slots_of(slots, p);
  const int64_t T = slots.numel(), i = p.layers ? 1 : 0;
  need(k.device() == p.device && v.device() == p.device && k.dim() == 3 + i && k.sizes() == v.sizes() &&
       k.scalar_type() == v.scalar_type() && k.size(i) == T && k.size(i + 1) == p.KVH &&
       k.size(i + 2) == p.D && (!p.layers || k.size(0) == p.L) && k.stride(i + 2) == 1 &&
       v.stride(i + 2) == 1);
  const int32_t dtype = dtype_code(k.scalar_type());
  int32_t* const err = counter(a[7], p.device);
  void* const stream = PyLong_AsVoidPtr(a[8]);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = p_append(p.kc.data_ptr(), p.ks.data_ptr(), p.vc.data_ptr(), p.vs.data_ptr(), p.L,
                    p.code_layer, p.code_slot, p.scale_layer, p.scale_slot, p.S, k.const_data_ptr(),
                    p.layers ? k.stride(0) : 0, k.stride(i), k.stride(i + 1), v.const_data_ptr(),
                    p.layers ? v.stride(0) : 0, v.stride(i), v.stride(i + 1), s, T, int32_t(p.KVH),
                    int32_t(p.D), p.format, dtype, err, stream);
  Py_END_ALLOW_THREADS
  need(status == DSP_OK);
  Py_RETURN_TRUE;
}

// gather(k_cache, k_scale, v_cache, v_scale, slots, like, err, stream) -> (k, v) or None; like: a tensor
// of the values' type
PyObject* gather(PyObject* const* a) {
  const Pools p(a);
  const at::Tensor& slots = tensor(a[4]);
  const int64_t* s = slots_of(slots, p);
  const int64_t T = slots.numel();
  need(Py_TYPE(a[5]) == reinterpret_cast<PyTypeObject*>(&THPDtypeType));
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const int32_t dtype = dtype_code(type);
  int32_t* const err = counter(a[6], p.device);
  void* const stream = PyLong_AsVoidPtr(a[7]);
  const auto options = p.kc.options().dtype(type);
  const at::Tensor k = p.layers ? at::empty({p.L, T, p.KVH, p.D}, options)
                                : at::empty({T, p.KVH, p.D}, options);
  const at::Tensor v = at::empty_like(k);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = p_gather(p.kc.const_data_ptr(), p.ks.const_data_ptr(), p.vc.const_data_ptr(),
                    p.vs.const_data_ptr(), p.L, p.code_layer, p.code_slot, p.scale_layer, p.scale_slot,
                    p.S, s, T, int32_t(p.KVH), int32_t(p.D), p.format, k.data_ptr(), v.data_ptr(), dtype,
                    err, stream);
  Py_END_ALLOW_THREADS
  need(status == DSP_OK);
  PyObject* const x = THPVariable_Wrap(k);
  PyObject* const y = THPVariable_Wrap(v);
  PyObject* const both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

// No C++ exception leaves a binding: what torch throws becomes the Python exception that torch makes of it
// (of a failed allocation an OutOfMemoryError).
template <PyObject* (*F)(PyObject* const*), int kArgs>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", kArgs, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Slow&) {
    Py_RETURN_NONE;
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// bind(window, window_bytes, append, gather): the addresses of the library's entry points.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long at[4];
  if (!PyArg_ParseTuple(args, "KKKK", at, at + 1, at + 2, at + 3)) return nullptr;
  p_window = reinterpret_cast<decltype(p_window)>(uintptr_t(at[0]));
  p_window_bytes = reinterpret_cast<decltype(p_window_bytes)>(uintptr_t(at[1]));
  p_append = reinterpret_cast<decltype(p_append)>(uintptr_t(at[2]));
  p_gather = reinterpret_cast<decltype(p_gather)>(uintptr_t(at[3]));
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int kArgs>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F, kArgs>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {{"bind", bind, METH_VARARGS, "bind(window, window_bytes, append, gather)"},
                          method<window, 19>("window"),
                          method<append, 9>("append"),
                          method<gather, 8>("gather"),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&kModule); }
