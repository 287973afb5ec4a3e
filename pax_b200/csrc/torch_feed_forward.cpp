// torch_feed_forward.cpp -- the feed-forward products on torch tensors, as a
// CPython module (pax_b200/_feed_forward).
//
// feed_forward.py's functions end here: argument checks, outputs from torch's
// allocator, the stream, and the call of the C entry.  A decoding step calls
// these operators dozens of times with a few microseconds of GPU work each.
// Host time of a call at 1x64x64: glu 4.7 us, quantize_rows 4.7, glu_backward
// 10.5, of which the C entry takes 3.5, 3 and 6.3; with checks, allocations
// and descriptors in Python it was 11, 12 and 24.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "../../include/pax.h"

namespace {

// An error to be raised as the given Python exception.
struct Raise {
    PyObject* type;
    std::string what;
};
// The Python error is already set.
struct Raised {};

// Raises module.cls(*args); takes args.
void raise_from(const char* module, const char* cls, PyObject* args) {
    PyObject* m = args ? PyImport_ImportModule(module) : nullptr;
    PyObject* c = m ? PyObject_GetAttrString(m, cls) : nullptr;
    PyObject* e = c ? PyObject_CallObject(c, args) : nullptr;
    if (e) PyErr_SetObject(c, e);
    Py_XDECREF(e);
    Py_XDECREF(c);
    Py_XDECREF(m);
    Py_XDECREF(args);
}

[[noreturn]] void value_error(const std::string& s) { throw Raise{PyExc_ValueError, s}; }
[[noreturn]] void type_error(const std::string& s) { throw Raise{PyExc_TypeError, s}; }

const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return "float16";
        case at::kFloat: return "float32";
        case at::kChar: return "int8";
        default: return "?";
    }
}

std::string shape_text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

bool given(PyObject* o) { return o != Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const at::Tensor& matrix2d(PyObject* o, const char* name) {
    if (!THPVariable_Check(o) || THPVariable_Unpack(o).dim() != 2)
        value_error(std::string(name) + " must be a 2-D tensor");
    return THPVariable_Unpack(o);
}

void same_place(const at::Tensor& t, const char* name, c10::Device dev) {
    if (t.device() != dev) value_error(std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
}

// Checks a matrix operand; its leading dimension in elements (0 where it is
// never used).
int64_t matrix(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, at::ScalarType dtype,
               c10::Device dev) {
    if (t.scalar_type() != dtype) type_error(std::string(name) + " must be " + type_name(dtype));
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
        value_error(std::string(name) + " has shape " + shape_text(t.sizes()) + ", expected " +
                    shape_text({rows, cols}));
    same_place(t, name, dev);
    if (rows == 0 || cols == 0) return 0;
    if (cols > 1 && t.stride(1) != 1) value_error(std::string(name) + " must be a 2-D tensor with unit column stride");
    if (rows == 1) return 0;
    if (t.stride(0) < cols) value_error(std::string(name) + " must have rows that do not overlap");
    return t.stride(0);
}

void vector(const at::Tensor& t, const char* name, int64_t n, at::ScalarType dtype, c10::Device dev) {
    if (t.scalar_type() != dtype) type_error(std::string(name) + " must be a " + type_name(dtype) + " tensor");
    if (t.dim() != 1 || t.size(0) != n)
        value_error(std::string(name) + " has shape " + shape_text(t.sizes()) + ", expected " + shape_text({n}));
    same_place(t, name, dev);
    if (n > 1 && t.stride(0) != 1) value_error(std::string(name) + " must be contiguous");
}

int64_t attribute(PyObject* o, const char* name) {
    PyObject* v = PyObject_GetAttrString(o, name);
    if (!v) throw Raised{};
    const int64_t r = PyLong_AsLongLong(v);
    Py_DECREF(v);
    if (r == -1 && PyErr_Occurred()) throw Raised{};
    return r;
}

// The device and stream of one call.  Outputs are allocated on the call's
// stream, so that neither their memory's earlier use nor its reuse after them
// can overlap the call, and stay reserved for the caller's current stream as
// well.  What the caller gives stays reserved for the call's stream until it is
// done there, also where the caller frees it right after the call.
class Call {
public:
    Call(c10::Device dev, PyObject* stream)
        : dev_(cuda(dev)), guard_(dev_), current_(c10::cuda::getCurrentCUDAStream(dev_.index())), stream_(current_) {
        if (!given(stream)) return;
        const c10::Device on(c10::kCUDA, (c10::DeviceIndex)attribute(stream, "device_index"));
        if (on != dev_) value_error("stream is on " + on.str() + ", expected " + dev_.str());
        stream_ = c10::cuda::CUDAStream::unpack3(attribute(stream, "stream_id"), on.index(), c10::kCUDA);
    }
    at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, bool scratch = false) const {
        if (stream_ == current_) return at::detail::empty_cuda(shape, dtype, dev_, std::nullopt);
        c10::cuda::CUDAStreamGuard on(stream_);
        at::Tensor t = at::detail::empty_cuda(shape, dtype, dev_, std::nullopt);
        if (!scratch && t.numel()) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), current_);
        return t;
    }
    void uses(std::initializer_list<const at::Tensor*> given) const {
        if (stream_ == current_) return;
        for (const at::Tensor* t : given)
            if (t->defined() && t->numel())
                c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), stream_);
    }
    // Runs f(stream), a C entry, and raises PaxError for its status.
    template <typename F>
    void run(const char* name, F f) const {
        PyThreadState* const held = PyEval_SaveThread();
        const pax_status_t st = f(stream_.stream());
        PyEval_RestoreThread(held);
        if (st == PAX_OK) return;
        raise_from("pax_b200.api", "PaxError", Py_BuildValue("(is)", (int)st, name));
        throw Raised{};
    }

private:
    static c10::Device cuda(c10::Device d) {
        if (!d.is_cuda()) value_error("tensors must be on a CUDA device");
        return d;
    }
    c10::Device dev_;
    c10::cuda::CUDAGuard guard_;
    c10::cuda::CUDAStream current_, stream_;
};

// Counts outputs as written, as torch's own writes do: autograd refuses
// a backward pass through a saved tensor that was overwritten.  Tensors made in
// inference mode have no count.
void written(std::initializer_list<const at::Tensor*> outs) {
    for (const at::Tensor* t : outs)
        if (t->defined() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// A given output as it is, or a new tensor.
PyObject* wrap(PyObject* out, const at::Tensor& t) {
    if (given(out)) {
        Py_INCREF(out);
        return out;
    }
    return THPVariable_Wrap(t);
}

PyObject* tuple(std::initializer_list<PyObject*> items) {
    PyObject* r = PyTuple_New((Py_ssize_t)items.size());
    Py_ssize_t i = 0;
    for (PyObject* o : items) {
        if (r && o)
            PyTuple_SET_ITEM(r, i, o);
        else
            Py_XDECREF(o);
        ++i;
    }
    return r;
}

PyObject* none() { Py_RETURN_NONE; }

// X, Wg, Wu, activation, save, out, G, U, stream, w_const -> H or (H, G, U)
PyObject* glu(PyObject* const* a) {
    const at::Tensor &X = matrix2d(a[0], "X"), &Wg = matrix2d(a[1], "Wg"), &Wu = tensor(a[2], "Wu");
    const int64_t M = X.size(0), D = X.size(1), F = Wg.size(1);
    PyObject *out = a[5], *g = a[6], *u = a[7];
    if (given(g) != given(u)) value_error("G and U go together");
    const c10::Device dev = X.device();
    pax_glu_desc_t d = {};
    d.M = M, d.D = D, d.F = F;
    d.act = (pax_activation_t)PyLong_AsLong(a[3]);
    d.w_const = a[9] == Py_True;
    d.ldx = matrix(X, "X", M, D, at::kHalf, dev);
    d.ldwg = matrix(Wg, "Wg", D, F, at::kHalf, dev);
    d.ldwu = matrix(Wu, "Wu", D, F, at::kHalf, dev);
    at::Tensor H, G, U;
    if (given(out)) d.ldh = matrix(H = tensor(out, "out"), "out", M, F, at::kHalf, dev);
    if (given(g)) {
        d.ldg = matrix(G = tensor(g, "G"), "G", M, F, at::kHalf, dev);
        d.ldu = matrix(U = tensor(u, "U"), "U", M, F, at::kHalf, dev);
    }
    const bool save = given(g) || a[4] == Py_True;
    const Call call(dev, a[8]);
    call.uses({&X, &Wg, &Wu, &H, &G, &U});
    if (!given(out)) H = call.empty({M, F}, at::kHalf);
    if (save && !given(g)) {
        G = call.empty({M, F}, at::kHalf);
        U = call.empty({M, F}, at::kHalf);
    }
    d.X = X.data_ptr(), d.Wg = Wg.data_ptr(), d.Wu = Wu.data_ptr(), d.H = H.data_ptr();
    if (save) d.G = G.data_ptr(), d.U = U.data_ptr();
    call.run("pax_glu_ex", [&](cudaStream_t s) { return pax_glu_ex(&d, s); });
    written({&H, &G, &U});
    if (!save) return wrap(out, H);
    return tuple({wrap(out, H), wrap(g, G), wrap(u, U)});
}

// dH, X, Wg, Wu, G, U, activation, need_dX, need_dW, dX, dWg, dWu, dW dtype
// (0 float32, 1 float16), accumulate, dG, dU, stream -> (dX, dWg, dWu)
PyObject* glu_backward(PyObject* const* a) {
    const at::Tensor &X = matrix2d(a[1], "X"), &Wg = matrix2d(a[2], "Wg"), &dH = tensor(a[0], "dH"),
                     &Wu = tensor(a[3], "Wu"), &G = tensor(a[4], "G"), &U = tensor(a[5], "U");
    const int64_t M = X.size(0), D = X.size(1), F = Wg.size(1);
    const bool need_x = a[7] == Py_True, need_w = a[8] == Py_True, accumulate = a[13] == Py_True;
    PyObject *px = a[9], *pg = a[10], *pu = a[11];
    at::ScalarType wt = PyLong_AsLong(a[12]) == PAX_DT_F16 ? at::kHalf : at::kFloat;
    if (given(pg) != given(pu)) value_error("dWg and dWu go together");
    if (given(pg)) {
        if (!need_w) value_error("dWg and dWu are given, but need_dW is false");
        wt = tensor(pg, "dWg").scalar_type();
        if (wt != at::kHalf && wt != at::kFloat) type_error("weight gradients must be float32 or float16");
    }
    if (given(px) && !need_x) value_error("dX is given, but need_dX is false");
    if (accumulate && (!given(pg) || wt != at::kFloat)) value_error("accumulate needs given float32 dWg and dWu");
    const c10::Device dev = X.device();
    pax_glu_grad_desc_t d = {};
    d.M = M, d.D = D, d.F = F;
    d.act = (pax_activation_t)PyLong_AsLong(a[6]);
    d.lddh = matrix(dH, "dH", M, F, at::kHalf, dev);
    d.ldx = matrix(X, "X", M, D, at::kHalf, dev);
    d.ldwg = matrix(Wg, "Wg", D, F, at::kHalf, dev);
    d.ldwu = matrix(Wu, "Wu", D, F, at::kHalf, dev);
    d.ldg = matrix(G, "G", M, F, at::kHalf, dev);
    d.ldu = matrix(U, "U", M, F, at::kHalf, dev);
    at::Tensor dX, dWg, dWu, dG, dU;
    if (given(a[14])) d.lddg = matrix(dG = tensor(a[14], "dG"), "dG", M, F, at::kHalf, dev);
    if (given(a[15])) d.lddu = matrix(dU = tensor(a[15], "dU"), "dU", M, F, at::kHalf, dev);
    if (given(px)) d.lddx = matrix(dX = tensor(px, "dX"), "dX", M, D, at::kHalf, dev);
    if (given(pg)) {
        d.lddwg = matrix(dWg = tensor(pg, "dWg"), "dWg", D, F, wt, dev);
        d.lddwu = matrix(dWu = tensor(pu, "dWu"), "dWu", D, F, wt, dev);
    }
    const Call call(dev, a[16]);
    call.uses({&dH, &X, &Wg, &Wu, &G, &U, &dX, &dWg, &dWu, &dG, &dU});
    if (need_x && !given(px)) dX = call.empty({M, D}, at::kHalf);
    if (need_w && !given(pg)) {
        dWg = call.empty({D, F}, wt);
        dWu = call.empty({D, F}, wt);
    }
    if (!given(a[14])) dG = call.empty({M, F}, at::kHalf, true);
    if (!given(a[15])) dU = call.empty({M, F}, at::kHalf, true);
    d.dH = dH.data_ptr(), d.X = X.data_ptr(), d.Wg = Wg.data_ptr(), d.Wu = Wu.data_ptr();
    d.G = G.data_ptr(), d.U = U.data_ptr(), d.dG = dG.data_ptr(), d.dU = dU.data_ptr();
    if (need_x) d.dX = dX.data_ptr();
    if (need_w) d.dWg = dWg.data_ptr(), d.dWu = dWu.data_ptr();
    d.dw_dtype = wt == at::kHalf ? PAX_DT_F16 : PAX_DT_F32;
    d.accumulate = accumulate;
    call.run("pax_glu_backward_ex", [&](cudaStream_t s) { return pax_glu_backward_ex(&d, s); });
    written({&dX, &dWg, &dWu, &dG, &dU});
    return tuple({need_x ? wrap(px, dX) : none(), need_w ? wrap(pg, dWg) : none(), need_w ? wrap(pu, dWu) : none()});
}

// X, out, scale, stream -> (Q, scale)
PyObject* quantize_rows(PyObject* const* a) {
    const at::Tensor& X = matrix2d(a[0], "X");
    const int64_t M = X.size(0), K = X.size(1);
    const c10::Device dev = X.device();
    const int64_t ldx = matrix(X, "X", M, K, at::kHalf, dev);
    int64_t ldq = 0;
    at::Tensor Q, scale;
    if (given(a[1])) ldq = matrix(Q = tensor(a[1], "out"), "out", M, K, at::kChar, dev);
    if (given(a[2])) vector(scale = tensor(a[2], "scale"), "scale", M, at::kFloat, dev);
    const Call call(dev, a[3]);
    call.uses({&X, &Q, &scale});
    if (!given(a[1])) Q = call.empty({M, K}, at::kChar);
    if (!given(a[2])) scale = call.empty({M}, at::kFloat);
    call.run("pax_quantize_rows", [&](cudaStream_t s) {
        return pax_quantize_rows(X.data_ptr(), ldx, Q.data_ptr(), ldq, static_cast<float*>(scale.data_ptr()), M, K, s);
    });
    written({&Q, &scale});
    return tuple({wrap(a[1], Q), wrap(a[2], scale)});
}

// A, B, a_scale, b_scale, bias, out, out dtype (0 float32, 1 float16), stream,
// b_const -> C
PyObject* gemm_i8(PyObject* const* a) {
    const at::Tensor &A = matrix2d(a[0], "A"), &B = matrix2d(a[1], "B"), &sa = tensor(a[2], "a_scale"),
                     &sb = tensor(a[3], "b_scale");
    const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
    const c10::Device dev = A.device();
    pax_gemm_i8_desc_t d = {};
    d.M = M, d.N = N, d.K = K;
    d.b_const = a[8] == Py_True;
    d.lda = matrix(A, "A", M, K, at::kChar, dev);
    d.ldb = matrix(B, "B", N, K, at::kChar, dev);
    vector(sa, "a_scale", M, at::kFloat, dev);
    vector(sb, "b_scale", N, at::kFloat, dev);
    at::ScalarType ct = PyLong_AsLong(a[6]) == PAX_DT_F16 ? at::kHalf : at::kFloat;
    at::Tensor bias, C;
    if (given(a[4])) vector(bias = tensor(a[4], "bias"), "bias", N, at::kHalf, dev);
    if (given(a[5])) {
        C = tensor(a[5], "out");
        ct = C.scalar_type();
        if (ct != at::kHalf && ct != at::kFloat) type_error("out must be float32 or float16");
        d.ldc = matrix(C, "out", M, N, ct, dev);
    }
    const Call call(dev, a[7]);
    call.uses({&A, &B, &sa, &sb, &bias, &C});
    if (!given(a[5])) C = call.empty({M, N}, ct);
    d.A = A.data_ptr(), d.B = B.data_ptr(), d.C = C.data_ptr();
    d.a_scale = static_cast<const float*>(sa.data_ptr());
    d.b_scale = static_cast<const float*>(sb.data_ptr());
    if (given(a[4])) d.bias = bias.data_ptr();
    d.c_dtype = ct == at::kHalf ? PAX_DT_F16 : PAX_DT_F32;
    call.run("pax_gemm_i8_ex", [&](cudaStream_t s) { return pax_gemm_i8_ex(&d, s); });
    written({&C});
    return wrap(a[5], C);
}

// Entry of each function: positional arguments only, every C++ exception
// turned into a Python one.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Raise& e) {
        PyErr_SetString(e.type, e.what.c_str());
    } catch (const Raised&) {
    } catch (const c10::OutOfMemoryError& e) {
        raise_from("torch", "OutOfMemoryError", Py_BuildValue("(s)", e.what_without_backtrace()));
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define PAX_ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {PAX_ENTRY(glu, 10), PAX_ENTRY(glu_backward, 17), PAX_ENTRY(quantize_rows, 4),
                          PAX_ENTRY(gemm_i8, 9), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_feed_forward", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__feed_forward(void) { return PyModule_Create(&kModule); }
