// torch_calls.cpp — the dense operators' calls from Python without ctypes.
//
// A decode step makes many small calls, whose cost is the host's: through ctypes, Python-side
// checks and torch.empty a 2048 x 2048 product takes 11.7 us to issue, of which the launch is
// 2.7. These functions make the same checks, allocate the output and the workspace from
// torch's allocator on the current stream, and call the same C entry points. A call that does
// not fit their checks returns None: ops.py then makes it, or says what is wrong with it.
// Contexts are per thread and device, so that no other call can bind another stream in
// between; they own no device memory here.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/moe_b200.h"

namespace {

PyObject* g_error = nullptr;  // MlxError

struct Contexts {
  moe_ctx* at[64] = {};
  ~Contexts() {
    for (moe_ctx* c : at) moe_ctx_destroy(c);
  }
};
moe_ctx* context_for(int device) {
  thread_local Contexts contexts;
  if (device < 0 || device >= 64) return nullptr;
  moe_ctx*& c = contexts.at[device];
  if (!c && moe_ctx_create(device, nullptr, &c) != MOE_OK) c = nullptr;
  if (c) moe_ctx_set_stream(c, c10::cuda::getCurrentCUDAStream(device).stream());
  return c;
}

PyObject* raise(const char* fn, int rc, const char* detail) {
  PyObject* e = PyObject_CallFunction(g_error, "sis", fn, rc, detail);
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  return nullptr;
}

// A plain CUDA tensor, or null.
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}
// The same for an input: not one that torch would look for a gradient of (no graph is recorded here;
// ops.py refuses it).
const at::Tensor* input(PyObject* o) {
  const at::Tensor* t = tensor(o);
  return t && !(t->requires_grad() && c10::GradMode::is_enabled()) ? t : nullptr;
}
bool contiguous_on(const at::Tensor* t, c10::ScalarType type, int device) {
  return t && t->scalar_type() == type && t->get_device() == device && t->is_contiguous();
}
int dtype_of(c10::ScalarType t) {
  return t == at::kBFloat16 ? MOE_DTYPE_BF16 : t == at::kHalf ? MOE_DTYPE_F16 : t == at::kFloat ? MOE_DTYPE_F32 : -1;
}
at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

// Runs f, turning a C++ exception (an allocation that failed, for one) into a Python one.
template <class F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* m = PyImport_ImportModule("torch");
    PyObject* type = m ? PyObject_GetAttrString(m, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(m);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// quantized_matmul(x, w, scales, biases, transpose, group_size)
PyObject* quantized_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "6 arguments expected");
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = input(a[0]), *w = tensor(a[1]), *s = tensor(a[2]);
    const at::Tensor* b = a[3] == Py_None ? nullptr : tensor(a[3]);
    const int transpose = PyObject_IsTrue(a[4]);
    const long g = PyLong_AsLong(a[5]);
    if (transpose < 0 || (g == -1 && PyErr_Occurred())) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    if (!x || !w || !s || (a[3] != Py_None && !b) || x->dim() < 1 || w->dim() != 2 || (g != 32 && g != 64 && g != 128))
      Py_RETURN_NONE;
    const int type = dtype_of(x->scalar_type()), dev = x->get_device();
    const int64_t K = x->size(-1), rows = w->size(0), cols = w->size(1) * 8, N = transpose ? rows : cols;
    if ((type != MOE_DTYPE_BF16 && type != MOE_DTYPE_F16) || !x->is_contiguous() || K == 0 ||
        (transpose ? cols : rows) != K || cols % g)
      Py_RETURN_NONE;
    if (!contiguous_on(w, at::kInt, dev) && !contiguous_on(w, at::kUInt32, dev)) Py_RETURN_NONE;
    for (const at::Tensor* q : {s, b})
      if (q && (!contiguous_on(q, x->scalar_type(), dev) || q->dim() != 2 || q->size(0) != rows || q->size(1) != cols / g))
        Py_RETURN_NONE;
    const int64_t M = x->numel() / K;
    size_t need = 0;
    const char* fn = "mlx_quantized_matmul";
    int rc = moe_quantized_matmul_workspace(type, M, K, N, transpose, (int)g, 4, &need);
    if (rc) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = N;
    at::Tensor out = at::empty(shape, x->options());
    at::Tensor ws;
    if (need) ws = scratch(need, *x);
    moe_ctx* ctx = context_for(dev);
    if (!ctx) return raise("moe_ctx_create", MOE_ERR_CUDA, "");
    rc = moe_quantized_matmul_ex(ctx, type, x->data_ptr(), M, K, static_cast<const uint32_t*>(w->data_ptr()),
                                 s->data_ptr(), b ? b->data_ptr() : nullptr, N, transpose, (int)g, 4, out.data_ptr(),
                                 need ? ws.data_ptr() : nullptr, need);
    if (rc) return raise(fn, rc, moe_last_error(ctx));
    return THPVariable_Wrap(std::move(out));
  });
}

// The block's weights from a tuple (w, scales, biases of gate, of up, of down), on the device and of
// the type of `like`; false where one does not fit the config. Pointers are taken anew in every
// call: a tensor of the block may have been replaced since the last.
bool ffn_weights(PyObject* o, const moe_ffn_config* cfg, const at::Tensor& like, moe_ffn_weights& out) {
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 9 || cfg->group_size <= 0) return false;
  moe_qweight* q[3] = {&out.gate, &out.up, &out.down};
  const int dev = like.get_device();
  for (int i = 0; i < 3; ++i) {
    const int64_t rows = i < 2 ? cfg->inter : cfg->hidden, cols = i < 2 ? cfg->hidden : cfg->inter;
    const void* at[3] = {};
    for (int j = 0; j < 3; ++j) {
      PyObject* p = PyTuple_GET_ITEM(o, 3 * i + j);
      if (j == 2 && p == Py_None) continue;
      if (!THPVariable_Check(p)) return false;
      const at::Tensor& t = THPVariable_Unpack(p);
      if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.dim() != 2 || t.size(0) != rows ||
          t.size(1) != cols / (j ? cfg->group_size : 8))
        return false;
      if (j ? !contiguous_on(&t, like.scalar_type(), dev)
            : !contiguous_on(&t, at::kInt, dev) && !contiguous_on(&t, at::kUInt32, dev))
        return false;
      at[j] = t.data_ptr();
    }
    *q[i] = {static_cast<const uint32_t*>(at[0]), at[1], at[2]};
  }
  return true;
}

// ffn_forward(config address, weights, x, residual, save): the config is ops.py's struct.
PyObject* ffn_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "5 arguments expected");
  return guarded([&]() -> PyObject* {
    const auto* cfg = static_cast<const moe_ffn_config*>(PyLong_AsVoidPtr(a[0]));
    moe_ffn_weights wts;
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* x = input(a[2]);
    const at::Tensor* r = a[3] == Py_None ? nullptr : input(a[3]);
    const bool save = a[4] == Py_True;
    if (!cfg || !x || (a[3] != Py_None && !r) || dtype_of(x->scalar_type()) != cfg->dtype || !x->is_contiguous() ||
        x->dim() < 1 || x->size(-1) != cfg->hidden || !ffn_weights(a[1], cfg, *x, wts))
      Py_RETURN_NONE;
    const int dev = x->get_device();
    if (r && (!contiguous_on(r, x->scalar_type(), dev) || r->sizes() != x->sizes())) Py_RETURN_NONE;
    const int64_t T = x->numel() / cfg->hidden;
    size_t need = 0;
    if (moe_gated_ffn_workspace(cfg, T, 0, &need)) Py_RETURN_NONE;
    at::Tensor out = at::empty(x->sizes(), x->options()), g, u, ws;
    if (save) {
      c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
      shape.back() = cfg->inter;
      g = at::empty(shape, x->options());
      u = at::empty(shape, x->options());
    }
    if (need) ws = scratch(need, *x);
    moe_ctx* ctx = context_for(dev);
    if (!ctx) return raise("moe_ctx_create", MOE_ERR_CUDA, "");
    const int rc = moe_gated_ffn_forward(ctx, cfg, &wts, x->data_ptr(), T, r ? r->data_ptr() : nullptr,
                                         save ? g.data_ptr() : nullptr, save ? u.data_ptr() : nullptr, out.data_ptr(),
                                         need ? ws.data_ptr() : nullptr, need);
    if (rc) return raise("moe_gated_ffn_forward", rc, moe_last_error(ctx));
    if (!save) return THPVariable_Wrap(std::move(out));
    return Py_BuildValue("NNN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(g)),
                         THPVariable_Wrap(std::move(u)));
  });
}

// ffn_backward(config address, weights, g, u, dy)
PyObject* ffn_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "5 arguments expected");
  return guarded([&]() -> PyObject* {
    const auto* cfg = static_cast<const moe_ffn_config*>(PyLong_AsVoidPtr(a[0]));
    moe_ffn_weights wts;
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *g = input(a[2]), *u = input(a[3]), *dy = input(a[4]);
    if (!cfg || !g || !u || !dy || dtype_of(dy->scalar_type()) != cfg->dtype || !dy->is_contiguous() ||
        dy->dim() < 1 || dy->size(-1) != cfg->hidden || !ffn_weights(a[1], cfg, *dy, wts))
      Py_RETURN_NONE;
    const int dev = dy->get_device();
    c10::SmallVector<int64_t, 6> shape(dy->sizes().begin(), dy->sizes().end());
    shape.back() = cfg->inter;
    for (const at::Tensor* t : {g, u})
      if (!contiguous_on(t, dy->scalar_type(), dev) || t->sizes() != c10::IntArrayRef(shape)) Py_RETURN_NONE;
    const int64_t T = dy->numel() / cfg->hidden;
    size_t need = 0;
    if (moe_gated_ffn_workspace(cfg, T, 1, &need)) Py_RETURN_NONE;
    at::Tensor dx = at::empty(dy->sizes(), dy->options()), dg = at::empty(shape, dy->options()),
               du = at::empty(shape, dy->options()), ws;
    if (need) ws = scratch(need, *dy);
    moe_ctx* ctx = context_for(dev);
    if (!ctx) return raise("moe_ctx_create", MOE_ERR_CUDA, "");
    const int rc = moe_gated_ffn_backward(ctx, cfg, &wts, g->data_ptr(), u->data_ptr(), dy->data_ptr(), T, dg.data_ptr(),
                                          du.data_ptr(), dx.data_ptr(), need ? ws.data_ptr() : nullptr, need);
    if (rc) return raise("moe_gated_ffn_backward", rc, moe_last_error(ctx));
    return Py_BuildValue("NNN", THPVariable_Wrap(std::move(dx)), THPVariable_Wrap(std::move(dg)),
                         THPVariable_Wrap(std::move(du)));
  });
}

// fast_rope(x [B, H, L, D], dims, traditional, base, scale, offset, freqs, mscale, inverse):
// into a new contiguous tensor.
PyObject* fast_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "9 arguments expected");
  return guarded([&]() -> PyObject* {
    const at::Tensor* x = input(a[0]);
    const at::Tensor* f = a[6] == Py_None ? nullptr : tensor(a[6]);
    if (!x || x->dim() != 4 || (a[6] != Py_None && !f)) Py_RETURN_NONE;
    const int type = dtype_of(x->scalar_type()), dev = x->get_device();
    if (type < 0 || (x->size(3) > 1 && x->stride(3) != 1)) Py_RETURN_NONE;
    moe_rope_config cfg{};
    cfg.dtype = type;
    const long dims = PyLong_AsLong(a[1]);
    if (dims < 0 || dims > x->size(3)) {  // an error of the conversion too
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    cfg.dims = (int32_t)dims;
    cfg.traditional = PyObject_IsTrue(a[2]);
    cfg.inverse = PyObject_IsTrue(a[8]);
    cfg.base = a[3] == Py_None ? 0.0 : PyFloat_AsDouble(a[3]);
    cfg.scale = PyFloat_AsDouble(a[4]);
    cfg.mscale = PyFloat_AsDouble(a[7]);
    const at::Tensor* offs = nullptr;
    int64_t offset = 0;
    if (THPVariable_Check(a[5])) {
      offs = tensor(a[5]);
      if (!offs || (offs->scalar_type() != at::kInt && offs->scalar_type() != at::kLong) || offs->get_device() != dev ||
          !offs->is_contiguous() || offs->dim() > 1 || offs->numel() != x->size(0))
        Py_RETURN_NONE;
    } else {
      offset = PyLong_AsLongLong(a[5]);
    }
    if (PyErr_Occurred()) {  // not the numbers expected here: ops.py says so
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    if (f && (!contiguous_on(f, at::kFloat, dev) || f->dim() != 1 || f->size(0) != cfg.dims / 2)) Py_RETURN_NONE;
    at::Tensor out = at::empty(x->sizes(), x->options());
    moe_ctx* ctx = context_for(dev);
    if (!ctx) return raise("moe_ctx_create", MOE_ERR_CUDA, "");
    const int rc = moe_fast_rope(ctx, &cfg, x->data_ptr(), x->strides().data(), x->size(0), x->size(1), x->size(2),
                                 x->size(3), offset, offs ? offs->data_ptr() : nullptr,
                                 offs ? (offs->scalar_type() == at::kInt ? 32 : 64) : 0,
                                 f ? static_cast<const float*>(f->data_ptr()) : nullptr, out.data_ptr(),
                                 out.strides().data());
    if (rc) return raise("mlx_fast_rope", rc, moe_last_error(ctx));
    return THPVariable_Wrap(std::move(out));
  });
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"set_error", set_error, METH_O, "The class raised for a failed call."},
    {"quantized_matmul", reinterpret_cast<PyCFunction>(quantized_matmul), METH_FASTCALL, nullptr},
    {"ffn_forward", reinterpret_cast<PyCFunction>(ffn_forward), METH_FASTCALL, nullptr},
    {"ffn_backward", reinterpret_cast<PyCFunction>(ffn_backward), METH_FASTCALL, nullptr},
    {"fast_rope", reinterpret_cast<PyCFunction>(fast_rope), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "The dense operators' calls (see ops.py).", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
