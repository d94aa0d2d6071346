// ptxstd._ffn: the feed-forward operators' argument checks, output tensors and C calls in one
// extension module. The operators take a few microseconds at serving sizes; checking a dozen
// tensors, allocating five or six and converting twenty arguments from Python takes 15 to 20 us a
// call, from here 5 to 8. It computes nothing: every result comes from libptxstd.so's entry points
// (include/ptxstd.h), which check sizes, alignment and types again.
//
// Functions take positional arguments only (ptxstd/ffn.py has the public signatures). Type errors
// raise TypeError, shapes and devices ValueError, a status of the library ptxstd.PtxStdError, and
// what torch throws meanwhile is raised as torch raises it.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <optional>
#include <string>

#include "ptxstd.h"

namespace {

struct PythonError {};  // the Python error is set

[[noreturn]] void raise(PyObject* type, const std::string& what) {
    PyErr_SetString(type, what.c_str());
    throw PythonError();
}

constexpr auto kBf16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;
constexpr auto kU8 = at::kByte;

// ---- arguments ------------------------------------------------------------------------------
const at::Tensor* optional_tensor(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, std::string(name) + ": expected a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* name) {
    const at::Tensor* t = optional_tensor(o, name);
    if (!t) raise(PyExc_TypeError, std::string(name) + ": expected a tensor");
    return *t;
}
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError();
    return v;
}

std::string str(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

// Type and shape of one argument (a missing one passes).
void want(const at::Tensor* t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
    if (!t) return;
    if (t->scalar_type() != type)
        raise(PyExc_TypeError, std::string(name) + ": expected " + at::toString(type) + ", got " +
                                   at::toString(t->scalar_type()));
    if (t->sizes() != shape)
        raise(PyExc_ValueError, std::string(name) + ": expected shape " + str(shape) + ", got " +
                                    str(t->sizes()));
}
void want_matrix(const at::Tensor& t) {
    if (t.scalar_type() != kBf16 || t.dim() != 2)
        raise(PyExc_TypeError, "expected a 2-D bfloat16 tensor");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t sf_numel(int64_t rows, int64_t cols) {
    return ceil_div(rows, 128) * ceil_div(cols, 128) * 512;
}

// An MX operand: a payload and its padded blocked scales, checked against each other.
struct Mx {
    const at::Tensor *q, *sf;
    int64_t rows, cols;
};
Mx operand(PyObject* q, PyObject* sf, const char* name, int64_t cols = -1) {
    Mx m = {&tensor(q, name), &tensor(sf, name), 0, 0};
    if (m.q->scalar_type() != kU8 || m.sf->scalar_type() != kU8 || m.q->dim() != 2)
        raise(PyExc_TypeError,
              std::string(name) + ": expected a 2-D uint8 payload and uint8 scales");
    m.rows = m.q->size(0);
    m.cols = m.q->size(1);
    if (cols >= 0 && m.cols != cols)
        raise(PyExc_ValueError, std::string(name) + ": K mismatch (" + std::to_string(m.cols) +
                                    ", expected " + std::to_string(cols) + ")");
    if (m.sf->numel() != sf_numel(m.rows, m.cols))
        raise(PyExc_ValueError, std::string(name) + ": the blocked scales of " +
                                    str(m.q->sizes()) + " have " +
                                    std::to_string(sf_numel(m.rows, m.cols)) + " bytes, got " +
                                    std::to_string(m.sf->numel()));
    return m;
}

// Device and stream of a call: every input has to be contiguous and on the current device.
struct Call {
    int device = -1;
    ptxstd_stream stream = nullptr;
    std::optional<c10::cuda::CUDAStreamGuard> guard;

    template <class T>
    T* in(const at::Tensor* t) {
        if (!t) return nullptr;
        if (!t->is_cuda()) raise(PyExc_TypeError, "expected a CUDA tensor");
        if (t->get_device() != device) {
            const int current = c10::cuda::current_device();
            if (t->get_device() != current)
                raise(PyExc_ValueError, "tensor on cuda:" + std::to_string(t->get_device()) +
                                            ", but the current device is cuda:" +
                                            std::to_string(current));
            device = current;
        }
        if (!t->is_contiguous()) raise(PyExc_ValueError, "expected a contiguous tensor");
        return static_cast<T*>(t->data_ptr());
    }
    // A torch.cuda.Stream, or None for the current stream; after the inputs. A stream that is given
    // is the current one until the call returns, so that the allocator keeps what is allocated
    // here (results, and workspaces that are dropped before the kernels end) in its order.
    void set_stream(PyObject* s) {
        const auto dev = static_cast<c10::DeviceIndex>(device);
        if (s == Py_None) {
            stream = c10::cuda::getCurrentCUDAStream(dev).stream();
            return;
        }
        PyObject* h = PyObject_GetAttrString(s, "cuda_stream");
        if (!h) throw PythonError();
        stream = PyLong_AsVoidPtr(h);
        Py_DECREF(h);
        if (PyErr_Occurred()) throw PythonError();
        guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), dev));
    }
    at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
        return at::detail::empty_cuda(
            shape, type, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)),
            std::nullopt);
    }
};

const uint16_t* bf16_in(Call& c, const at::Tensor* t) { return c.in<const uint16_t>(t); }
const uint8_t* u8_in(Call& c, const at::Tensor* t) { return c.in<const uint8_t>(t); }
const float* f32_in(Call& c, const at::Tensor* t) { return c.in<const float>(t); }

template <class T>
T* out(const at::Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// ---- results ----------------------------------------------------------------------------------
void check(int status, const char* what) {
    if (status == PTXSTD_OK) return;
    PyObject* m = PyImport_ImportModule("ptxstd");
    if (m) {
        PyObject* r = PyObject_CallMethod(m, "check", "is", status, what);
        Py_XDECREF(r);
        Py_DECREF(m);
    }
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    throw PythonError();
}

PyObject* wrap(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
// A tuple of new references.
template <class... P>
PyObject* tuple(P*... items) {
    PyObject* all[] = {items...};
    bool ok = true;
    for (PyObject* p : all) ok = ok && p;
    PyObject* t = ok ? PyTuple_New(sizeof...(items)) : nullptr;
    for (size_t i = 0; i < sizeof...(items); ++i) {
        if (t) PyTuple_SET_ITEM(t, static_cast<Py_ssize_t>(i), all[i]);
        else Py_XDECREF(all[i]);
    }
    return t;
}
PyObject* keep(PyObject* o) {
    Py_INCREF(o);
    return o;
}

// ---- operators --------------------------------------------------------------------------------
// x, w, y, w_post, gate, scale, eps, out_type (-1: bf16), sf_layout, stream
PyObject* rmsnorm_residual(PyObject* const* a) {
    const at::Tensor& x = tensor(a[0], "x");
    want_matrix(x);
    const int64_t rows = x.size(0), cols = x.size(1);
    const at::Tensor *w = &tensor(a[1], "w"), *y = optional_tensor(a[2], "y"),
                     *w_post = optional_tensor(a[3], "w_post"),
                     *gate = optional_tensor(a[4], "gate");
    want(w, "w", kBf16, {cols});
    want(y, "y", kBf16, {rows, cols});
    want(w_post, "w_post", kBf16, {cols});
    if (!y && (w_post || gate)) raise(PyExc_ValueError, "w_post and gate belong to y");
    int64_t gate_rows = 1;
    if (gate && gate->dim() == 2) {
        want(gate, "gate", kBf16, {rows, cols});
        gate_rows = rows;
    } else {
        want(gate, "gate", kBf16, {cols});
    }
    const float scale = static_cast<float>(real(a[5])), eps = static_cast<float>(real(a[6]));
    const int type = static_cast<int>(integer(a[7])), layout = static_cast<int>(integer(a[8]));
    Call c;
    const uint16_t *px = bf16_in(c, &x), *py = bf16_in(c, y), *pwp = bf16_in(c, w_post),
                   *pg = bf16_in(c, gate), *pw = bf16_in(c, w);
    c.set_stream(a[9]);
    at::Tensor x_out, n, q, sf, rstd, rstd_post;
    if (y) x_out = c.empty({rows, cols}, kBf16);
    if (type < 0) {
        n = c.empty({rows, cols}, kBf16);
    } else {
        q = c.empty({rows, cols}, kU8);
        sf = layout == 1 ? c.empty({sf_numel(rows, cols)}, kU8) : c.empty({rows, cols / 32}, kU8);
    }
    rstd = c.empty({rows}, kF32);
    if (w_post) rstd_post = c.empty({rows}, kF32);
    check(ptxstd_rmsnorm_residual(px, py, pwp, pg, gate_rows, scale, pw, eps, rows, cols,
                                  out<uint16_t>(x_out), out<uint16_t>(n), type < 0 ? 0 : type,
                                  out<uint8_t>(q), out<uint8_t>(sf), layout, out<float>(rstd),
                                  out<float>(rstd_post), c.stream),
          "rmsnorm_residual");
    return tuple(y ? wrap(x_out) : keep(a[0]), type < 0 ? wrap(n) : tuple(wrap(q), wrap(sf)),
                 tuple(wrap(rstd), wrap(rstd_post)));
}

// dn, x_out, w, rstd, rstd_post, dx_out, y, w_post, gate, scale, stream
PyObject* rmsnorm_residual_backward(PyObject* const* a) {
    const at::Tensor& dn = tensor(a[0], "dn");
    want_matrix(dn);
    const int64_t rows = dn.size(0), cols = dn.size(1);
    const at::Tensor *x = &tensor(a[1], "x_out"), *w = &tensor(a[2], "w"),
                     *rstd = &tensor(a[3], "rstd"), *rstd_post = optional_tensor(a[4], "rstd_post"),
                     *du = optional_tensor(a[5], "dx_out"), *y = optional_tensor(a[6], "y"),
                     *w_post = optional_tensor(a[7], "w_post"),
                     *gate = optional_tensor(a[8], "gate");
    want(x, "x_out", kBf16, {rows, cols});
    want(du, "dx_out", kBf16, {rows, cols});
    want(y, "y", kBf16, {rows, cols});
    want(w, "w", kBf16, {cols});
    want(w_post, "w_post", kBf16, {cols});
    want(rstd, "rstd", kF32, {rows});
    want(rstd_post, "rstd_post", kF32, {rows});
    if (!y && (w_post || gate)) raise(PyExc_ValueError, "w_post and gate belong to y");
    if (!w_post != !rstd_post)
        raise(PyExc_ValueError, "w_post and its statistics belong together");
    const bool per_row = gate && gate->dim() == 2;
    if (per_row) want(gate, "gate", kBf16, {rows, cols});
    else want(gate, "gate", kBf16, {cols});
    // one row: a gate of all rows, whose gradient is f32 [cols]; given back as it was asked for
    const bool as_row = per_row && rows > 1;
    const float scale = static_cast<float>(real(a[9]));
    Call c;
    const uint16_t *pdn = bf16_in(c, &dn), *pdu = bf16_in(c, du), *px = bf16_in(c, x),
                   *pw = bf16_in(c, w), *py = bf16_in(c, y), *pwp = bf16_in(c, w_post),
                   *pg = bf16_in(c, gate);
    const float *pr = f32_in(c, rstd), *prp = f32_in(c, rstd_post);
    c.set_stream(a[10]);
    at::Tensor dx = c.empty({rows, cols}, kBf16), dw = c.empty({cols}, kF32), dy, dwp, dg;
    if (y) dy = c.empty({rows, cols}, kBf16);
    if (w_post) dwp = c.empty({cols}, kF32);
    if (gate) dg = as_row ? c.empty({rows, cols}, kBf16) : c.empty({cols}, kF32);
    const size_t bytes = ptxstd_rmsnorm_residual_backward_workspace_bytes(rows, cols);
    at::Tensor ws = c.empty({static_cast<int64_t>(bytes ? bytes : 16)}, kU8);
    check(ptxstd_rmsnorm_residual_backward(
              pdn, pdu, px, pw, pr, py, pwp, prp, pg, as_row ? rows : 1, scale, rows, cols,
              out<uint16_t>(dx), out<float>(dw), out<uint16_t>(dy), out<float>(dwp), out<void>(dg),
              ws.data_ptr(), bytes, c.stream),
          "rmsnorm_residual_backward");
    if (per_row && !as_row) dg = dg.to(kBf16).view({1, cols});
    return tuple(wrap(dx), wrap(dw), wrap(dy), wrap(dwp), wrap(dg));
}

// a, a_type, sfa, b, b_type, sfb, bias, act, residual, out_type (-1: bf16), save_pre, stream
PyObject* gemm_mx_epilogue(PyObject* const* a) {
    const Mx A = operand(a[0], a[2], "a"), B = operand(a[3], a[5], "b", A.cols);
    const int64_t M = A.rows, N = B.rows, K = A.cols;
    const at::Tensor *bias = optional_tensor(a[6], "bias"),
                     *residual = optional_tensor(a[8], "residual");
    want(bias, "bias", kBf16, {N});
    want(residual, "residual", kBf16, {M, N});
    const int type = static_cast<int>(integer(a[9]));
    const bool save = integer(a[10]) != 0;
    Call c;
    const uint8_t *pa = u8_in(c, A.q), *psa = u8_in(c, A.sf), *pb = u8_in(c, B.q),
                  *psb = u8_in(c, B.sf);
    const uint16_t *pbias = bf16_in(c, bias), *pres = bf16_in(c, residual);
    c.set_stream(a[11]);
    at::Tensor r, q, sf, pre;
    if (type < 0) {
        r = c.empty({M, N}, kBf16);
    } else {
        q = c.empty({M, N}, kU8);
        sf = c.empty({sf_numel(M, N)}, kU8);
    }
    if (save) pre = c.empty({M, N}, kBf16);
    check(ptxstd_gemm_mx_epilogue(pa, static_cast<int>(integer(a[1])), psa, pb,
                                  static_cast<int>(integer(a[4])), psb, pbias,
                                  static_cast<int>(integer(a[7])), pres, out<uint16_t>(r),
                                  out<uint16_t>(pre), type < 0 ? 0 : type, out<uint8_t>(q),
                                  out<uint8_t>(sf), M, N, K, c.stream),
          "gemm_mx_epilogue");
    PyObject* result = type < 0 ? wrap(r) : tuple(wrap(q), wrap(sf));
    return save ? tuple(result, wrap(pre)) : result;
}

// a, a_type, sfa, w_gate, sf_gate, w_up, sf_up, w_type, act, out_type (-1: bf16), save, stream
PyObject* gemm_mx_gated(PyObject* const* a) {
    const Mx A = operand(a[0], a[2], "a"), W = operand(a[3], a[4], "w_gate", A.cols),
             U = operand(a[5], a[6], "w_up", A.cols);
    if (W.rows != U.rows)
        raise(PyExc_ValueError, "w_gate and w_up have different numbers of rows");
    const int64_t M = A.rows, F = W.rows, K = A.cols;
    const int type = static_cast<int>(integer(a[9]));
    const bool save = integer(a[10]) != 0;
    Call c;
    const uint8_t *pa = u8_in(c, A.q), *psa = u8_in(c, A.sf), *pg = u8_in(c, W.q),
                  *psg = u8_in(c, W.sf), *pu = u8_in(c, U.q), *psu = u8_in(c, U.sf);
    c.set_stream(a[11]);
    at::Tensor h, q, sf, gate, up;
    if (type < 0) {
        h = c.empty({M, F}, kBf16);
    } else {
        q = c.empty({M, F}, kU8);
        sf = c.empty({sf_numel(M, F)}, kU8);
    }
    if (save) {
        gate = c.empty({M, F}, kBf16);
        up = c.empty({M, F}, kBf16);
    }
    check(ptxstd_gemm_mx_gated(pa, static_cast<int>(integer(a[1])), psa, pg, psg, pu, psu,
                               static_cast<int>(integer(a[7])), static_cast<int>(integer(a[8])),
                               out<uint16_t>(h), out<uint16_t>(gate), out<uint16_t>(up),
                               type < 0 ? 0 : type, out<uint8_t>(q), out<uint8_t>(sf), M, F, K,
                               c.stream),
          "gemm_mx_gated");
    PyObject* result = type < 0 ? wrap(h) : tuple(wrap(q), wrap(sf));
    return save ? tuple(result, tuple(wrap(gate), wrap(up))) : result;
}

// dh, gate, up, act, out_type, bias_grad, stream
PyObject* act_backward_mx(PyObject* const* a) {
    const at::Tensor& dh = tensor(a[0], "dh");
    want_matrix(dh);
    const int64_t rows = dh.size(0), cols = dh.size(1);
    const at::Tensor *gate = &tensor(a[1], "gate"), *up = optional_tensor(a[2], "up");
    want(gate, "gate", kBf16, {rows, cols});
    want(up, "up", kBf16, {rows, cols});
    const int act = static_cast<int>(integer(a[3])), type = static_cast<int>(integer(a[4]));
    const bool bias = integer(a[5]) != 0;
    Call c;
    const uint16_t *pdh = bf16_in(c, &dh), *pg = bf16_in(c, gate), *pu = bf16_in(c, up);
    c.set_stream(a[6]);
    const int64_t W = cols * (up ? 2 : 1), R = ceil_div(rows, 32) * 32;
    at::Tensor q = c.empty({rows, W}, kU8), sf = c.empty({sf_numel(rows, W)}, kU8),
               qt = c.empty({W, R}, kU8), sft = c.empty({sf_numel(W, R)}, kU8), db, ws;
    size_t bytes = 0;
    if (bias) {
        db = c.empty({W}, kF32);
        bytes = ptxstd_act_backward_mx_workspace_bytes(rows, cols, up != nullptr, 1);
        ws = c.empty({static_cast<int64_t>(bytes ? bytes : 16)}, kU8);
    }
    check(ptxstd_act_backward_mx(act, pdh, pg, pu, rows, cols, type, out<uint8_t>(q),
                                 out<uint8_t>(sf), out<uint8_t>(qt), out<uint8_t>(sft),
                                 out<float>(db), out<void>(ws), bytes, c.stream),
          "act_backward_mx");
    PyObject *row = tuple(wrap(q), wrap(sf)), *col = tuple(wrap(qt), wrap(sft));
    return bias ? tuple(row, col, wrap(db)) : tuple(row, col);
}

// x, out_type, stream
PyObject* quantize_mx_t(PyObject* const* a) {
    const at::Tensor& x = tensor(a[0], "x");
    want_matrix(x);
    const int64_t rows = x.size(0), cols = x.size(1), R = ceil_div(rows, 32) * 32;
    Call c;
    const uint16_t* px = bf16_in(c, &x);
    c.set_stream(a[2]);
    at::Tensor qt = c.empty({cols, R}, kU8), sft = c.empty({sf_numel(cols, R)}, kU8);
    check(ptxstd_quantize_mx_t(px, rows, cols, static_cast<int>(integer(a[1])), out<uint8_t>(qt),
                               out<uint8_t>(sft), c.stream),
          "quantize_mx_t");
    return tuple(wrap(qt), wrap(sft));
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %zd positional arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const PythonError&) {
        return nullptr;
    } catch (...) {  // torch's own errors as torch raises them (torch.OutOfMemoryError, say)
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)),
            METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {
    method<rmsnorm_residual, 10>("rmsnorm_residual"),
    method<rmsnorm_residual_backward, 11>("rmsnorm_residual_backward"),
    method<gemm_mx_epilogue, 12>("gemm_mx_epilogue"),
    method<gemm_mx_gated, 12>("gemm_mx_gated"),
    method<act_backward_mx, 7>("act_backward_mx"),
    method<quantize_mx_t, 3>("quantize_mx_t"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ffn", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ffn() { return PyModule_Create(&kModule); }
