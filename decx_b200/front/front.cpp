// Python entry of the low-precision operators: checks the tensors and calls the C ABI of include/decx_b200.h.
//
// A call through ctypes, with the checks in Python, costs 8 to 12 us of host time; the small calls of this family take
// the GPU 2 to 6 us.  Here the checks read the tensors' own fields, and what remains is the launch.  Every function takes
// all of its arguments by position (None where there is none), raises TypeError / ValueError / RuntimeError for what does
// not fit, and returns the C ABI's code.  decx_b200/blas.py and gemm.py give them their names and documentation.
#include <Python.h>

#include <ATen/core/TensorBase.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>

#include "../../include/decx_b200.h"

namespace {

using at::TensorBase;

struct Refused {};          // a Python error has been set

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(type, format, args);
    va_end(args);
    throw Refused();
}

const TensorBase& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}
const TensorBase* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

void on_gpu(const TensorBase& t) {
    if (!t.is_cuda()) refuse(PyExc_RuntimeError, "decx_b200 works on CUDA tensors only (no CPU fallback)");
}

// elements between the rows of a row-major, pitched matrix
uint64_t pitch(const TensorBase& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    if (sizes.size() != 2 || (sizes[1] > 1 && strides[1] != 1))
        refuse(PyExc_ValueError, "matrices must be 2-D with unit column stride (row-major, pitched)");
    return uint64_t(sizes[0] > 1 ? strides[0] : (sizes[1] > strides[0] ? sizes[1] : strides[0]));
}
uint32_t extent(int64_t n) {
    if (n > 0xFFFFFFFFll) refuse(PyExc_ValueError, "extents are 32-bit");
    return uint32_t(n);
}

void is_matrix(const TensorBase& t, int64_t rows, int64_t cols, const char* what) {
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols) refuse(PyExc_ValueError, "%s", what);
}
void is_vector(const TensorBase& t, at::ScalarType type, int64_t n, const char* what) {
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1)) refuse(PyExc_ValueError, "%s", what);
}
void same_device(const TensorBase& a, const TensorBase& b) {
    if (a.device() != b.device()) refuse(PyExc_ValueError, "all operands must be on one device");
}

int float_type(const TensorBase& t) {
    return t.scalar_type() == at::kHalf ? DECXB200_FP16 : t.scalar_type() == at::kFloat ? DECXB200_FP32 : 0;
}

void need(Py_ssize_t given, Py_ssize_t wanted) {
    if (given != wanted) refuse(PyExc_TypeError, "takes %zd arguments", wanted);
}

float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return float(v);
}
long integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}

// Makes `device` current while the call lasts, if it is not: switching costs more than a small launch.
struct Current {
    c10::DeviceIndex before, device;
    explicit Current(c10::DeviceIndex d) : before(c10::cuda::current_device()), device(d) {
        if (before != device) c10::cuda::set_device(device);
    }
    ~Current() {
        if (before != device) c10::cuda::MaybeSetDevice(before);
    }
};

template <typename F>
PyObject* launch(const TensorBase& t, F&& call) {
    const c10::DeviceIndex device = t.get_device();
    const Current current(device);
    return PyLong_FromLong(call(static_cast<void*>(c10::cuda::getCurrentCUDAStream(device).stream())));
}

template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

struct Q8 {
    uint8_t* q;
    uint64_t ld;
    float* scales;
};
// the 8-bit matrix and the scales that a call writes
Q8 q8_result(const TensorBase& x, PyObject* out, PyObject* scales) {
    const TensorBase& q = tensor(out, "out");
    const TensorBase& s = tensor(scales, "scales");
    if (q.scalar_type() != at::kFloat8_e4m3fn) refuse(PyExc_ValueError, "out must be float8_e4m3fn");
    is_matrix(q, x.size(0), x.size(1), "out must have the input's shape");
    is_vector(s, at::kFloat, x.size(0), "scales must be a contiguous float32 vector with one entry per row");
    same_device(x, q);
    same_device(x, s);
    return {static_cast<uint8_t*>(q.data_ptr()), pitch(q), static_cast<float*>(s.data_ptr())};
}

// (src, out, scales)
PyObject* cast_q8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() {
        need(n, 3);
        const TensorBase& src = tensor(args[0], "src");
        on_gpu(src);
        const int type = float_type(src);
        if (type == 0) refuse(PyExc_TypeError, "cast_q8 takes float16 or float32");
        const uint64_t ld = pitch(src);
        const Q8 r = q8_result(src, args[1], args[2]);
        return launch(src, [&](void* stream) {
            return decxb200_cast_q8(type, stream, extent(src.size(0)), extent(src.size(1)), src.data_ptr(), ld, r.q, r.ld, r.scales);
        });
    });
}

// (x, weight, residual, eps, out, scales, sum_out)
PyObject* rmsnorm_q8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() {
        need(n, 7);
        const TensorBase& x = tensor(args[0], "x");
        const TensorBase& w = tensor(args[1], "weight");
        const TensorBase* r = maybe(args[2], "residual");
        const TensorBase* sum = maybe(args[6], "sum_out");
        on_gpu(x);
        const int type = float_type(x);
        if (type == 0 || w.scalar_type() != x.scalar_type() || (r != nullptr && r->scalar_type() != x.scalar_type()))
            refuse(PyExc_TypeError, "x, weight and residual must share one dtype out of float16, float32");
        const uint64_t ldx = pitch(x);
        const int64_t rows = x.size(0), cols = x.size(1);
        is_vector(w, x.scalar_type(), cols, "weight must be a contiguous vector with one entry per column of x");
        same_device(x, w);
        uint64_t ldr = 0, lds = 0;
        if (r != nullptr) {
            is_matrix(*r, rows, cols, "residual must have the shape of x");
            same_device(x, *r);
            ldr = pitch(*r);
        }
        if (sum != nullptr) {
            if (r == nullptr) refuse(PyExc_ValueError, "sum_out without a residual");
            is_matrix(*sum, rows, cols, "sum_out must have the shape and type of x");
            if (sum->scalar_type() != x.scalar_type()) refuse(PyExc_ValueError, "sum_out must have the shape and type of x");
            same_device(x, *sum);
            lds = pitch(*sum);
        }
        const float eps = number(args[3]);
        const Q8 q = q8_result(x, args[4], args[5]);
        return launch(x, [&](void* stream) {
            return decxb200_rmsnorm_q8(type, stream, extent(rows), extent(cols), x.data_ptr(), ldx, r ? r->data_ptr() : nullptr, ldr,
                                       sum ? sum->data_ptr() : nullptr, lds, w.data_ptr(), eps, q.q, q.ld, q.scales);
        });
    });
}

// (A, scale_a, B, scale_b, C, alpha, beta, out, status, tile)
PyObject* gemm_q8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() {
        need(n, 10);
        const TensorBase& A = tensor(args[0], "A");
        const TensorBase& sa = tensor(args[1], "scale_a");
        const TensorBase& B = tensor(args[2], "B");
        const TensorBase& sb = tensor(args[3], "scale_b");
        const TensorBase* C = maybe(args[4], "C");
        const TensorBase& D = tensor(args[7], "out");
        const TensorBase* status = maybe(args[8], "status");
        on_gpu(A);
        if (A.scalar_type() != at::kFloat8_e4m3fn || B.scalar_type() != at::kFloat8_e4m3fn)
            refuse(PyExc_TypeError, "A and B must be float8_e4m3fn");
        const uint64_t lda = pitch(A), ldb = pitch(B);
        const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
        if (B.size(1) != K) refuse(PyExc_ValueError, "A is %lldx%lld but B is %lldx%lld", (long long)M, (long long)K, (long long)N, (long long)B.size(1));
        is_vector(sa, at::kFloat, M, "scale_a must be a contiguous float32 vector with one entry per row of A");
        is_vector(sb, at::kFloat, N, "scale_b must be a contiguous float32 vector with one entry per row of B");
        const int type = float_type(D);
        if (type == 0 || (C != nullptr && C->scalar_type() != D.scalar_type()))
            refuse(PyExc_TypeError, "C and the result must share one dtype out of float16, float32");
        is_matrix(D, M, N, "C and out must be M x N");
        if (C != nullptr) is_matrix(*C, M, N, "C and out must be M x N");
        same_device(A, B);
        same_device(A, sa);
        same_device(A, sb);
        same_device(A, D);
        if (C != nullptr) same_device(A, *C);
        if (status != nullptr) {
            if (status->scalar_type() != at::kInt || status->numel() < 1) refuse(PyExc_TypeError, "status must be an int32 tensor");
            same_device(A, *status);
        }
        const float alpha = args[5] == Py_None ? 1.f : number(args[5]);
        const float beta = args[6] == Py_None || C == nullptr ? 0.f : number(args[6]);
        const long tile = integer(args[9]);
        const uint64_t ldc = C != nullptr ? pitch(*C) : 0, ldd = pitch(D);
        return launch(A, [&](void* stream) {
            return decxb200_gemm_q8(type, stream, extent(M), extent(N), extent(K), A.data_ptr(), lda,
                                    static_cast<const float*>(sa.data_ptr()), B.data_ptr(), ldb,
                                    static_cast<const float*>(sb.data_ptr()), C ? C->data_ptr() : nullptr, ldc, D.data_ptr(), ldd,
                                    &alpha, &beta, status ? static_cast<unsigned*>(status->data_ptr()) : nullptr,
                                    tile >= 0 && tile <= 0xFFFF ? int(tile) : -1);
        });
    });
}

// (W, scales, x, group, zeros, x_scales, out); x and out of one vector may be 1-D
PyObject* gemv_q4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() {
        need(n, 7);
        const TensorBase& W = tensor(args[0], "W");
        const TensorBase& s = tensor(args[1], "scales");
        const TensorBase& x = tensor(args[2], "x");
        const long asked = integer(args[3]);
        const uint32_t group = asked > 0 && asked <= 128 ? uint32_t(asked) : 0u;     // 0: refused below
        const TensorBase* z = maybe(args[4], "zeros");
        const TensorBase* xs = maybe(args[5], "x_scales");
        const TensorBase& y = tensor(args[6], "out");
        on_gpu(W);
        if (W.scalar_type() != at::kByte || s.scalar_type() != at::kHalf || (z != nullptr && z->scalar_type() != at::kByte))
            refuse(PyExc_TypeError, "gemv_q4 takes uint8 W, float16 scales and uint8 zeros");
        const int xt = x.scalar_type() == at::kHalf ? DECXB200_FP16 : x.scalar_type() == at::kFloat8_e4m3fn ? DECXB200_E4M3 : 0;
        if (xt == 0) refuse(PyExc_TypeError, "x must be float16 or float8_e4m3fn");
        const bool single = x.dim() == 1;
        const int64_t vectors = single ? 1 : x.size(0), cols = single ? x.size(0) : x.size(1), rows = W.size(0);
        if (single && cols > 1 && x.stride(0) != 1) refuse(PyExc_ValueError, "x must be contiguous");
        const uint64_t ldx = single ? uint64_t(cols) : pitch(x), ldw = pitch(W), lds = pitch(s), ldz = z != nullptr ? pitch(*z) : 0;
        const int64_t groups = group != 0 ? (cols + group - 1) / group : 0;
        const char* const shapes = "W is rows x ceil(cols / 2), scales and zeros rows x ceil(cols / group), x vectors of cols entries";
        is_matrix(W, rows, (cols + 1) / 2, shapes);
        is_matrix(s, rows, groups, shapes);
        if (z != nullptr) is_matrix(*z, rows, groups, shapes);
        if (xs != nullptr && (xs->scalar_type() != at::kFloat || xs->numel() != vectors || !xs->is_contiguous()))
            refuse(PyExc_ValueError, "x_scales must be contiguous float32 with one entry per vector");
        const int yt = float_type(y);
        const bool fits = y.dim() == 1 ? single && y.size(0) == rows && (rows <= 1 || y.stride(0) == 1)
                                       : y.dim() == 2 && !single && y.size(0) == vectors && y.size(1) == rows;
        if (yt == 0 || !fits) refuse(PyExc_ValueError, "the result is float16 or float32, one entry per row of W for each vector");
        const uint64_t ldy = y.dim() == 1 ? uint64_t(rows) : pitch(y);
        same_device(W, s);
        same_device(W, x);
        same_device(W, y);
        if (z != nullptr) same_device(W, *z);
        if (xs != nullptr) same_device(W, *xs);
        return launch(W, [&](void* stream) {
            return decxb200_gemv_q4(xt, yt, stream, extent(rows), extent(cols), extent(vectors), group, W.data_ptr(),
                                    ldw, s.data_ptr(), lds, z ? z->data_ptr() : nullptr, ldz, x.data_ptr(), ldx,
                                    xs ? static_cast<const float*>(xs->data_ptr()) : nullptr, y.data_ptr(), ldy);
        });
    });
}

template <typename F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"cast_q8", fast(cast_q8), METH_FASTCALL, "(src, out, scales) -> code"},
    {"rmsnorm_q8", fast(rmsnorm_q8), METH_FASTCALL, "(x, weight, residual, eps, out, scales, sum_out) -> code"},
    {"gemm_q8", fast(gemm_q8), METH_FASTCALL, "(A, scale_a, B, scale_b, C, alpha, beta, out, status, tile) -> code"},
    {"gemv_q4", fast(gemv_q4), METH_FASTCALL, "(W, scales, x, group, zeros, x_scales, out) -> code"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", "Checked calls of the low-precision operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front() {
    PyObject* const m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", DECXB200_TORCH) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
