// Torch side of the int8 and norm entries: checks of tensors, the device and its current stream, then the C ABI.
//
// A call of these takes the GPU a few microseconds, so the way to the launch counts.  Host time of a call in us, with the checks in Python and
// ctypes / here: int8_gemm 7.1 / 3.0, int8_quantize 5.5 / 3.0, rms_norm 6.2 / 3.0, block_norm (21 arguments) 9.8 / 4.0; a launch alone takes 2.5.
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cstdarg>
#include <cstdint>
#include <exception>
#include <limits>
#include <stdexcept>
#include <string>
#include "../../include/tkb200.h"

namespace {

typedef uint64_t Types;       // a bit for each dtype
constexpr Types one(at::ScalarType s) { return Types(1) << int(s); }
constexpr Types kHalf = one(at::kBFloat16) | one(at::kHalf), kFp32 = one(at::kFloat), kOut = kHalf | kFp32, kInt8 = one(at::kChar);

[[noreturn]] void fail(const char* fmt, ...) {
    char text[512];
    va_list args;
    va_start(args, fmt);
    vsnprintf(text, sizeof(text), fmt, args);
    va_end(args);
    throw std::runtime_error(text);
}

std::string shape_text(at::IntArrayRef sizes) {
    std::string s = "(";
    for (int64_t n : sizes) s += (s.size() > 1 ? ", " : "") + (n < 0 ? std::string("any") : std::to_string(n));
    return s + ")";
}

int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? TKB_DTYPE_BF16 : (t.scalar_type() == at::kHalf ? TKB_DTYPE_FP16 : TKB_DTYPE_FP32); }

// A CUDA tensor of one of `types`, on `device` (any if negative), of the given sizes (any where negative)
const at::Tensor& tensor(PyObject* o, const char* name, Types types, int device, at::IntArrayRef shape) {
    if (!THPVariable_Check(o)) fail("%s must be a torch.Tensor", name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) fail("%s must be a CUDA tensor", name);
    if (!(one(t.scalar_type()) & types)) {
        std::string want;
        for (at::ScalarType s : {at::kBFloat16, at::kHalf, at::kFloat, at::kChar})
            if (one(s) & types) want += (want.empty() ? "" : ", ") + std::string(c10::toString(s));
        fail("%s has dtype %s, expected one of (%s)", name, c10::toString(t.scalar_type()), want.c_str());
    }
    if (device >= 0 && t.get_device() != device) fail("%s is on device %d, the first operand on device %d", name, int(t.get_device()), device);
    const at::IntArrayRef sizes = t.sizes();
    bool fits = sizes.size() == shape.size();
    for (size_t i = 0; i < sizes.size(); i++) {
        // (sizes are passed as C ints, which would keep the low 32 bits of a larger one)
        if (sizes[i] > std::numeric_limits<int>::max())
            fail("%s has shape %s, of which the library takes sizes up to %d", name, shape_text(sizes).c_str(), std::numeric_limits<int>::max());
        fits = fits && (shape[i] < 0 || shape[i] == sizes[i]);
    }
    if (!fits) fail("%s has shape %s, expected %s", name, shape_text(sizes).c_str(), shape_text(shape).c_str());
    return t;
}

struct Matrix {
    void* data;
    int64_t pitch;            // elements
    int n, k, device, dtype;
};
// A row-strided matrix (a single row has no pitch that anything reads)
Matrix matrix(PyObject* o, const char* name, Types types, int device, int64_t n, int64_t k) {
    const at::Tensor& t = tensor(o, name, types, device, {n, k});
    n = t.size(0); k = t.size(1);
    const int64_t pitch = n <= 1 ? k : t.stride(0);
    if (pitch < k || (t.stride(1) != 1 && k > 1)) fail("%s must have a contiguous last dimension and rows that do not overlap", name);
    return {t.data_ptr(), pitch, int(n), int(k), int(t.get_device()), dtype_code(t)};
}
void* vector(PyObject* o, const char* name, Types types, int device, int64_t n) {
    const at::Tensor& t = tensor(o, name, types, device, {n});
    if (n > 1 && t.stride(0) != 1) fail("%s must be contiguous", name);
    return t.data_ptr();
}
Types only(int dtype) { return one(dtype == TKB_DTYPE_BF16 ? at::kBFloat16 : at::kHalf); }

double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        fail("%s must be a number", name);
    }
    return v;
}

// Makes `device` current, hands its current stream to `call`, and returns the entry's code
template <typename F>
PyObject* launch(int device, F call) {
    int code;
    {
        const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
        void* const stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
        PyThreadState* const state = PyEval_SaveThread();      // (a launch waits where the queue is full)
        code = call(stream);
        PyEval_RestoreThread(state);
    }
    return PyLong_FromLong(code);
}

// The optional outputs of a norm
struct Outputs {
    void* y = nullptr; int64_t ldy = 0;
    void* codes = nullptr; int64_t ldc = 0;
    float* sc = nullptr;
};
Outputs outputs(PyObject* Y, PyObject* Y_int8, PyObject* Y_sc, Types types, int device, int M, int K) {
    Outputs out;
    if (Y != Py_None) {
        const Matrix y = matrix(Y, "Y", types, device, M, K);
        out.y = y.data; out.ldy = y.pitch;
    }
    if ((Y_int8 == Py_None) != (Y_sc == Py_None)) fail("Y_int8 and Y_sc come together");
    if (Y_int8 != Py_None) {
        const Matrix q = matrix(Y_int8, "Y_int8", kInt8, device, M, K);
        out.codes = q.data; out.ldc = q.pitch;
        out.sc = static_cast<float*>(vector(Y_sc, "Y_sc", kFp32, device, M));
    }
    return out;
}

// int8_quantize(A, A_int8, A_sc)
PyObject* int8_quantize(PyObject* const* o) {
    const Matrix a = matrix(o[0], "A", kHalf, -1, -1, -1);
    const Matrix q = matrix(o[1], "A_int8", kInt8, a.device, a.n, a.k);
    float* const sc = static_cast<float*>(vector(o[2], "A_sc", kFp32, a.device, a.n));
    return launch(a.device, [&](void* s) { return tkb_int8_quantize(a.data, a.pitch, a.dtype, q.data, q.pitch, sc, a.n, a.k, s); });
}

// int8_gemm(A, A_sc, B, B_sc, D, config)
PyObject* int8_gemm(PyObject* const* o) {
    const Matrix a = matrix(o[0], "A", kInt8, -1, -1, -1);
    const Matrix b = matrix(o[2], "B", kInt8, a.device, -1, a.k);
    const Matrix d = matrix(o[4], "D", kOut, a.device, a.n, b.n);
    const float* const a_sc = static_cast<float*>(vector(o[1], "A_sc", kFp32, a.device, a.n));
    const float* const b_sc = static_cast<float*>(vector(o[3], "B_sc", kFp32, a.device, b.n));
    const int config = int(number(o[5], "config"));
    return launch(a.device, [&](void* s) {
        return tkb_int8_gemm_ex(a.data, a.pitch, a_sc, b.data, b.pitch, b_sc, d.data, d.pitch, d.dtype, a.n, b.n, a.k, config, s);
    });
}

// rms_norm(X, W, Y, Y_int8, Y_sc, eps)
PyObject* rms_norm(PyObject* const* o) {
    const Matrix x = matrix(o[0], "X", kHalf, -1, -1, -1);
    const void* const w = vector(o[1], "W", only(x.dtype), x.device, x.k);
    if (o[2] == Py_None && o[3] == Py_None) fail("rms_norm needs Y or Y_int8 and Y_sc");
    const Outputs out = outputs(o[2], o[3], o[4], only(x.dtype), x.device, x.n, x.k);
    const float eps = float(number(o[5], "eps"));
    return launch(x.device, [&](void* s) {
        return tkb_rms_norm(x.data, x.pitch, w, out.y, out.ldy, out.codes, out.ldc, out.sc, x.dtype, x.n, x.k, eps, s);
    });
}

// block_norm(H, X, X_out, W_post, gate, residual_scale, W_pre, Y, Y_int8, Y_sc, eps)
PyObject* block_norm(PyObject* const* o) {
    const Matrix h = matrix(o[0], "H", kHalf, -1, -1, -1);
    const int dev = h.device, M = h.n, K = h.k;
    const Matrix x = matrix(o[1], "X", only(h.dtype), dev, M, K), r = matrix(o[2], "X_out", only(h.dtype), dev, M, K);
    const void* const w_post = o[3] == Py_None ? nullptr : vector(o[3], "W_post", only(h.dtype), dev, K);
    const void* const w_pre = o[6] == Py_None ? nullptr : vector(o[6], "W_pre", only(h.dtype), dev, K);
    const void* gate = nullptr;
    int64_t ldg = 0;
    int per = 1;
    if (o[4] != Py_None) {
        if (THPVariable_Check(o[4]) && THPVariable_Unpack(o[4]).dim() == 1) {
            gate = vector(o[4], "gate", only(h.dtype), dev, K);
            ldg = K; per = M > 0 ? M : 1;
        } else {
            const at::Tensor& t = tensor(o[4], "gate", only(h.dtype), dev, {-1, K});
            const int n = int(t.size(0));
            if (n ? M % n != 0 || (M > 0 && M < n) : M > 0) fail("gate has %d rows, of which %d rows of H are no multiple", n, M);
            if (n > 1 && t.stride(0) == 0 && (t.stride(1) == 1 || K == 1)) {       // one row, expanded
                gate = t.data_ptr(); ldg = K; per = M > 0 ? M : 1;
            } else {
                const Matrix g = matrix(o[4], "gate", only(h.dtype), dev, n, K);
                gate = g.data; ldg = g.pitch; per = n && M >= n ? M / n : 1;
            }
        }
    }
    const bool second = o[7] != Py_None || o[8] != Py_None;
    if (!w_pre && second) fail("Y and Y_int8 need W_pre");
    if (w_pre && !second) fail("W_pre needs Y or Y_int8 and Y_sc");
    const Outputs out = outputs(o[7], o[8], o[9], only(h.dtype), dev, M, K);
    const float residual_scale = float(number(o[5], "residual_scale")), eps = float(number(o[10], "eps"));
    return launch(dev, [&](void* s) {
        return tkb_block_norm(h.data, h.pitch, x.data, x.pitch, r.data, r.pitch, w_post, gate, ldg, per, residual_scale, w_pre, out.y, out.ldy, out.codes,
                              out.ldc, out.sc, h.dtype, M, K, eps, s);
    });
}

// No C++ exception leaves for Python, whatever a tensor's accessors throw
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != N) fail("%d arguments expected, %d given", N, int(n));
        return F(args);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<int8_quantize, 3>("int8_quantize"), method<int8_gemm, 6>("int8_gemm"), method<rms_norm, 6>("rms_norm"),
                         method<block_norm, 11>("block_norm"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__torch_ops() {
    PyObject* const m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TKB_TORCH_VERSION) != 0) {      // that it was built with
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
