// The short way from Python to the entry points whose calls last a few microseconds (routing, grouped products, products with an epilogue, combining).
//
// Each function takes its arguments as the Python function of the same name does, and where all is well (plain tensors on one CUDA device, of the types, shapes and strides that the kernels
// take, nothing that would need a gradient) allocates the result, queues the kernels on the current stream and returns it.  Everywhere else it returns None and has done nothing: the Python
// function then says what is wrong, or makes the copy that it takes.  Results are the same either way; a call takes half the time.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/tcq_b200.h"

namespace {

// The library's entry points, by address (bind): the same instance that the rest of the package has loaded.
decltype(&tcq_ms_grouped_linear_workspace_bytes) grouped_bytes = nullptr;
decltype(&tcq_ms_grouped_linear) grouped_linear = nullptr;
decltype(&tcq_route_workspace_bytes) route_bytes = nullptr;
decltype(&tcq_route) route = nullptr;
decltype(&tcq_combine) combine = nullptr;
decltype(&tcq_ms_linear_workspace_bytes) linear_bytes = nullptr;
decltype(&tcq_ms_linear) ms_linear = nullptr;
decltype(&tcq_ms_epilogue) epilogue = nullptr;

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return TCQ_F32;
        case at::kHalf: return TCQ_F16;
        case at::kBFloat16: return TCQ_BF16;
        default: return -1;
    }
}

// A tensor that can be taken as it is, or NULL.
const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_conj() || t.is_neg() || at::isTensorSubclassLike(t)) return nullptr;
    if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
    if (t._fw_grad(0).defined()) return nullptr;
    return &t;
}
bool on(const at::Tensor* t, int dev) { return t != nullptr && t->get_device() == dev; }
bool is(const at::Tensor* t, at::ScalarType type, int dev) { return on(t, dev) && t->scalar_type() == type && t->is_contiguous(); }

// Rows of `k` columns: a matrix with unit column stride whose rows do not overlap, or anything contiguous.
struct Rows {
    int64_t rows, ld;
    bool ok;
};
Rows rows_of(const at::Tensor& t, int64_t k) {
    if (t.dim() == 0 || t.size(-1) != k) return {0, 0, false};
    if (t.is_contiguous()) return {k ? t.numel() / k : 0, k, k > 0};
    if (t.dim() != 2 || (t.stride(1) != 1 && k > 1) || (t.stride(0) < k && t.size(0) > 1)) return {0, 0, false};
    return {t.size(0), t.size(0) > 1 ? t.stride(0) : k, true};
}

bool text(PyObject* o, const char* s) { return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, s) == 0; }

int activation_of(PyObject* o) {
    static const char* const names[] = {nullptr, "relu", "gelu", "gelu_tanh", "silu", "geglu", "swiglu"};
    if (o == Py_None) return 0;
    for (int i = 1; i < 7; ++i)
        if (text(o, names[i])) return i;
    return -1;
}
bool gated(int act) { return act >= TCQ_ACT_GEGLU; }

// Matrices in 4 bits: (codes, scales, row_scale, shape, fmt), of shape (n, k), or (e, n, k) with one more axis in front.
struct Matrices {
    const at::Tensor *codes, *scales, *row;
    int64_t e, n, k;
    int fmt, dev;
};
bool matrices(PyObject* w, bool many, Matrices& m) {
    if (!PyTuple_Check(w) || PyTuple_GET_SIZE(w) != 5) return false;
    PyObject *shape = PyTuple_GET_ITEM(w, 3), *fmt = PyTuple_GET_ITEM(w, 4), *row = PyTuple_GET_ITEM(w, 2);
    if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != (many ? 3 : 2)) return false;
    int64_t size[3] = {1, 0, 0};
    for (int i = 0; i < (many ? 3 : 2); ++i) {
        size[i + !many] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
        if (PyErr_Occurred()) { PyErr_Clear(); return false; }
        if (size[i + !many] < 0) return false;
    }
    m.e = size[0]; m.n = size[1]; m.k = size[2];
    m.fmt = text(fmt, "nvfp4") ? TCQ_MS_NVFP4 : text(fmt, "mxfp4") ? TCQ_MS_MXFP4 : -1;
    if (m.fmt < 0) return false;
    m.codes = plain(PyTuple_GET_ITEM(w, 0));
    if (m.codes == nullptr) return false;
    m.dev = m.codes->get_device();
    m.scales = plain(PyTuple_GET_ITEM(w, 1));
    if (!is(m.codes, at::kByte, m.dev) || !is(m.scales, at::kByte, m.dev)) return false;
    const int64_t codes[3] = {m.e, m.n, (m.k + 31) / 32 * 16}, scales[6] = {m.e, (m.n + 127) / 128, (m.fmt == TCQ_MS_NVFP4 ? 4 : 2) * ((m.k + 255) / 256), 32, 4, 4}, rows[2] = {m.e, m.n};
    const int skip = many ? 0 : 1;
    if (m.codes->sizes() != at::IntArrayRef(codes + skip, 3 - skip) || m.scales->sizes() != at::IntArrayRef(scales + skip, 6 - skip)) return false;
    m.row = nullptr;
    if (m.fmt == TCQ_MS_MXFP4) return row == Py_None;
    m.row = plain(row);
    return is(m.row, at::kFloat, m.dev) && m.row->sizes() == at::IntArrayRef(rows + skip, 2 - skip);
}

bool usual_mode() { return !c10::impl::dispatch_mode_enabled(); }
const void* address(const at::Tensor* t) { return t == nullptr ? nullptr : t->const_data_ptr(); }
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int dev) { return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, dev), std::nullopt); }

// The product, its workspace given back when the call is queued: the stream's later work comes after it.
bool queue_grouped(const at::Tensor& x, const Rows& r, const int32_t* tokens, const int32_t* offsets, int64_t rows, const Matrices& m, const at::Tensor* bias, int act,
                   const at::Tensor* residual, int64_t ldr, at::Tensor& y, int64_t out) {
    const int dt = type_of(x.scalar_type());
    const bool in_order = tokens == nullptr && reinterpret_cast<uintptr_t>(address(&x)) % 16 == 0 && r.ld % 8 == 0;
    const size_t size = grouped_bytes(rows, m.e, m.n, m.k, dt, m.fmt, in_order);
    at::Tensor ws;
    if (size) ws = empty({int64_t(size)}, at::kByte, m.dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(m.dev));
    return grouped_linear(address(&x), dt, r.rows, r.ld, tokens, offsets, m.e, rows, static_cast<const uint8_t*>(address(m.codes)), static_cast<const uint8_t*>(address(m.scales)),
                          static_cast<const float*>(address(m.row)), m.n, m.k, m.fmt, address(bias), bias ? type_of(bias->scalar_type()) : 0, act, address(residual), ldr,
                          y.mutable_data_ptr(), type_of(y.scalar_type()), out, size ? ws.mutable_data_ptr() : nullptr, size,
                          c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(m.dev)).stream()) == TCQ_OK;
}

// fp32 x: the product, then the epilogue behind it, in place where nothing is gated.
at::Tensor queue_fp32(const at::Tensor& x, const Rows& r, const Matrices& m, const at::Tensor* bias, int act, const at::Tensor* residual, int64_t ldr, at::IntArrayRef sizes, int64_t out) {
    at::Tensor y = empty(sizes, at::kFloat, m.dev), h = out == m.n ? y : empty({r.rows, m.n}, at::kFloat, m.dev), ws;
    const size_t size = linear_bytes(r.rows, m.n, m.k, TCQ_F32, m.fmt);
    if (r.rows > 8) ws = empty({int64_t(size)}, at::kByte, m.dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(m.dev));
    void* const stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(m.dev)).stream();
    if (ms_linear(address(&x), TCQ_F32, r.rows, r.ld, static_cast<const uint8_t*>(address(m.codes)), static_cast<const uint8_t*>(address(m.scales)), static_cast<const float*>(address(m.row)),
                  m.n, m.k, m.fmt, h.mutable_data_ptr(), m.n, r.rows > 8 ? ws.mutable_data_ptr() : nullptr, size, stream) != TCQ_OK ||
        epilogue(h.const_data_ptr<float>(), r.rows, m.n, address(bias), bias ? type_of(bias->scalar_type()) : 0, act, address(residual), ldr, y.mutable_data_ptr(), TCQ_F32, out, stream) != TCQ_OK)
        return {};
    return y;
}

// linear(x, w, bias, activation, residual)
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Matrices m;
    const int act = count == 5 ? activation_of(a[3]) : -1;
    if (act < 0 || !usual_mode() || !matrices(a[1], false, m) || (gated(act) && m.n % 2)) Py_RETURN_NONE;
    const at::Tensor* const x = plain(a[0]);
    if (!on(x, m.dev) || type_of(x->scalar_type()) < 0) Py_RETURN_NONE;
    const Rows r = rows_of(*x, m.k);
    if (!r.ok || r.rows == 0 || m.n == 0) Py_RETURN_NONE;
    const int64_t out = gated(act) ? m.n / 2 : m.n;
    const at::Tensor* bias = nullptr;
    if (a[2] != Py_None) {
        bias = plain(a[2]);
        if (!on(bias, m.dev) || type_of(bias->scalar_type()) < 0 || bias->dim() != 1 || bias->size(0) != m.n || !bias->is_contiguous()) Py_RETURN_NONE;
    }
    const at::Tensor* residual = nullptr;
    int64_t ldr = 0;
    if (a[4] != Py_None) {
        residual = plain(a[4]);
        if (!on(residual, m.dev) || residual->scalar_type() != x->scalar_type() || residual->dim() != x->dim()) Py_RETURN_NONE;
        for (int64_t i = 0; i + 1 < x->dim(); ++i)
            if (residual->size(i) != x->size(i)) Py_RETURN_NONE;
        const Rows rr = rows_of(*residual, out);
        if (!rr.ok) Py_RETURN_NONE;
        ldr = rr.ld;
    }
    c10::SmallVector<int64_t, 4> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() = out;
    if (x->scalar_type() == at::kFloat) {
        at::Tensor y = queue_fp32(*x, r, m, bias, act, residual, ldr, sizes, out);
        if (!y.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(y));
    }
    at::Tensor y = empty(sizes, x->scalar_type(), m.dev);
    if (!queue_grouped(*x, r, nullptr, nullptr, r.rows, m, bias, act, residual, ldr, y, out)) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// grouped_linear(x, w, offsets, tokens, bias, activation, dtype)
PyObject* py_grouped(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Matrices m;
    const int act = count == 7 ? activation_of(a[5]) : -1;
    if (act < 0 || !usual_mode() || !matrices(a[1], true, m) || (gated(act) && m.n % 2) || m.e < 1 || m.n == 0 || m.k == 0) Py_RETURN_NONE;
    const at::Tensor *const x = plain(a[0]), *const offsets = plain(a[2]);
    if (!on(x, m.dev) || x->dim() != 2 || (x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    const Rows r = rows_of(*x, m.k);
    if (!r.ok || !is(offsets, at::kInt, m.dev) || offsets->dim() != 1 || offsets->size(0) != m.e + 1) Py_RETURN_NONE;
    const at::Tensor *tokens = nullptr, *bias = nullptr;
    int64_t rows = r.rows;
    if (a[3] != Py_None) {
        tokens = plain(a[3]);
        if (!is(tokens, at::kInt, m.dev) || tokens->dim() != 1) Py_RETURN_NONE;
        rows = tokens->size(0);
    }
    if (rows == 0) Py_RETURN_NONE;
    if (a[4] != Py_None) {
        bias = plain(a[4]);
        if (!on(bias, m.dev) || type_of(bias->scalar_type()) < 0 || bias->dim() != 2 || bias->size(0) != m.e || bias->size(1) != m.n || !bias->is_contiguous()) Py_RETURN_NONE;
    }
    at::ScalarType type = x->scalar_type();
    if (a[6] != Py_None) {
        if (!THPDtype_Check(a[6])) Py_RETURN_NONE;
        type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
        if (type_of(type) < 0) Py_RETURN_NONE;
    }
    const int64_t out = gated(act) ? m.n / 2 : m.n;
    at::Tensor y = empty({rows, out}, type, m.dev);
    if (!queue_grouped(*x, r, tokens ? tokens->const_data_ptr<int32_t>() : nullptr, offsets->const_data_ptr<int32_t>(), rows, m, bias, act, nullptr, 0, y, out)) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// route(logits, top_k, score, normalize) -> (weights, experts, places, tokens, offsets)
PyObject* py_route(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 4 || !usual_mode() || !PyLong_CheckExact(a[1]) || !PyBool_Check(a[3])) Py_RETURN_NONE;
    const at::Tensor* const logits = plain(a[0]);
    const int score = text(a[2], "softmax") ? TCQ_SCORE_SOFTMAX : text(a[2], "sigmoid") ? TCQ_SCORE_SIGMOID : -1;
    if (logits == nullptr || score < 0 || logits->dim() != 2 || type_of(logits->scalar_type()) < 0) Py_RETURN_NONE;
    const int64_t t = logits->size(0), e = logits->size(1);
    const long long top = PyLong_AsLongLong(a[1]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const Rows r = rows_of(*logits, e);
    if (!r.ok || t == 0 || top < 1 || top > 32 || top > e || e > 1024) Py_RETURN_NONE;
    const int dev = logits->get_device();
    at::Tensor weights = empty({t, top}, at::kFloat, dev), chosen = empty({t, top}, at::kInt, dev), places = empty({t, top}, at::kInt, dev), tokens = empty({t * top}, at::kInt, dev),
               offsets = empty({e + 1}, at::kInt, dev), ws;
    const size_t size = route_bytes(t, e);
    if (size) ws = empty({int64_t(size)}, at::kByte, dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    if (route(address(logits), type_of(logits->scalar_type()), t, r.ld, e, top, score, a[3] == Py_True, weights.mutable_data_ptr<float>(), chosen.mutable_data_ptr<int32_t>(),
              places.mutable_data_ptr<int32_t>(), tokens.mutable_data_ptr<int32_t>(), offsets.mutable_data_ptr<int32_t>(), size ? ws.mutable_data_ptr() : nullptr, size,
              c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream()) != TCQ_OK)
        Py_RETURN_NONE;
    at::Tensor* const all[5] = {&weights, &chosen, &places, &tokens, &offsets};
    PyObject* const result = PyTuple_New(5);
    if (result == nullptr) return nullptr;
    for (int i = 0; i < 5; ++i) {
        PyObject* const o = THPVariable_Wrap(std::move(*all[i]));
        if (o == nullptr) { Py_DECREF(result); return nullptr; }
        PyTuple_SET_ITEM(result, i, o);
    }
    return result;
    END_HANDLE_TH_ERRORS
}

// combine(y, routing, residual, dtype)
PyObject* py_combine(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 4 || !usual_mode() || !PyTuple_Check(a[1]) || PyTuple_GET_SIZE(a[1]) != 5) Py_RETURN_NONE;
    const at::Tensor *const y = plain(a[0]), *const weights = plain(PyTuple_GET_ITEM(a[1], 0)), *const places = plain(PyTuple_GET_ITEM(a[1], 2));
    if (y == nullptr || y->dim() != 2 || type_of(y->scalar_type()) < 0) Py_RETURN_NONE;
    const int dev = y->get_device();
    const int64_t n = y->size(1);
    const Rows r = rows_of(*y, n);
    if (!r.ok || !is(weights, at::kFloat, dev) || !is(places, at::kInt, dev) || weights->dim() != 2 || places->sizes() != weights->sizes()) Py_RETURN_NONE;
    const int64_t t = weights->size(0), top = weights->size(1);
    if (t == 0 || top < 1 || top > 32) Py_RETURN_NONE;
    at::ScalarType type = y->scalar_type();
    if (a[3] != Py_None) {
        if (!THPDtype_Check(a[3])) Py_RETURN_NONE;
        type = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    }
    const at::Tensor* residual = nullptr;
    int64_t ldr = 0;
    if (a[2] != Py_None) {
        residual = plain(a[2]);
        if (!on(residual, dev) || residual->dim() != 2 || residual->size(0) != t || (a[3] != Py_None && residual->scalar_type() != type)) Py_RETURN_NONE;
        const Rows rr = rows_of(*residual, n);
        if (!rr.ok) Py_RETURN_NONE;
        ldr = rr.ld;
        type = residual->scalar_type();
    }
    if (type_of(type) < 0) Py_RETURN_NONE;
    at::Tensor out = empty({t, n}, type, dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    if (combine(address(y), type_of(y->scalar_type()), r.rows, r.ld, n, weights->const_data_ptr<float>(), places->const_data_ptr<int32_t>(), t, top, address(residual), ldr,
                out.mutable_data_ptr(), type_of(type), n, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream()) != TCQ_OK)
        Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(addresses of tcq_ms_grouped_linear_workspace_bytes, tcq_ms_grouped_linear, tcq_route_workspace_bytes, tcq_route, tcq_combine, tcq_ms_linear_workspace_bytes, tcq_ms_linear,
// tcq_ms_epilogue)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 8) {
        PyErr_SetString(PyExc_TypeError, "eight addresses expected");
        return nullptr;
    }
    void* at[8];
    for (int i = 0; i < 8; ++i)
        if ((at[i] = PyLong_AsVoidPtr(a[i])) == nullptr) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is NULL");
            return nullptr;
        }
    grouped_bytes = reinterpret_cast<decltype(grouped_bytes)>(at[0]);
    grouped_linear = reinterpret_cast<decltype(grouped_linear)>(at[1]);
    route_bytes = reinterpret_cast<decltype(route_bytes)>(at[2]);
    route = reinterpret_cast<decltype(route)>(at[3]);
    combine = reinterpret_cast<decltype(combine)>(at[4]);
    linear_bytes = reinterpret_cast<decltype(linear_bytes)>(at[5]);
    ms_linear = reinterpret_cast<decltype(ms_linear)>(at[6]);
    epilogue = reinterpret_cast<decltype(epilogue)>(at[7]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_bind)), METH_FASTCALL, nullptr},
                         {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_linear)), METH_FASTCALL, nullptr},
                         {"grouped_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_grouped)), METH_FASTCALL, nullptr},
                         {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_route)), METH_FASTCALL, nullptr},
                         {"combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_combine)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tcq_torch", "The short way to the library's small calls.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: what it was compiled against, (ABI of the library, torch, Python); whoever loads it looks before any other call.
PyMODINIT_FUNC PyInit_tcq_torch() {
    PyObject* const m = PyModule_Create(&module);
    if (m == nullptr) return nullptr;
    PyObject* const built_for = Py_BuildValue("(isi)", TCQ_ABI_VERSION, TORCH_VERSION, PY_VERSION_HEX >> 16);
    if (built_for == nullptr || PyModule_AddObject(m, "built_for", built_for) < 0) {
        Py_XDECREF(built_for);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
