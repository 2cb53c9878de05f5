// The scoring, loss and 4-bit lm_head calls for torch tensors: argument checks,
// output and workspace tensors, and the C ABI call on the current stream of the
// tensors' device (qwen600_engine_b200/losses.py and w4.py hold the public
// functions).  Small calls of these operators take a few microseconds on the
// GPU; made from Python through ctypes, the checks and allocations took 10 to
// 13 of a call's 20.
#include <Python.h>

#include <ATen/Functions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>

#include "qwen600_sampler.h"

namespace {

// A refused call, raised as SamplerError.
struct Refused {
    int code;
    std::string msg;
};

[[noreturn]] void invalid(const std::string& msg) { throw Refused{QS_ERR_INVALID, msg}; }

void check(int rc) {
    if (rc != QS_OK) throw Refused{rc, qs_last_error()};
}

const char* name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return c10::toString(t);
    }
}

std::string shape_of(const at::Tensor& t) {
    std::ostringstream s;
    s << "(";
    for (int64_t i = 0; i < t.dim(); i++) s << (i ? ", " : "") << t.size(i);
    s << (t.dim() == 1 ? ",)" : ")");
    return s.str();
}

std::string told(const at::Tensor& t) {
    return std::string(name_of(t.scalar_type())) + " " + shape_of(t) + " on " + t.device().str();
}

const at::Tensor& tensor(const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) invalid(std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{0, ""};  // the error is set
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused{0, ""};
    return v != 0;
}

int count(const char* name, int64_t n) {
    if (n > INT32_MAX) throw Refused{QS_ERR_UNSUPPORTED, std::string(name) + ": " + std::to_string(n) + " above 2^31 - 1"};
    return (int)n;
}

// A [rows, vocab] tensor whose columns are contiguous.
struct Matrix {
    int rows, vocab, dtype;
    long long ld;
    Matrix(const char* name, const at::Tensor& t) {
        if (t.dim() != 2) invalid(std::string(name) + " must be [rows, vocab], got " + shape_of(t));
        if (t.scalar_type() == at::kFloat) dtype = QS_F32;
        else if (t.scalar_type() == at::kBFloat16) dtype = QS_BF16;
        else invalid(std::string(name) + " dtype " + name_of(t.scalar_type()) + " (want float32 or bfloat16)");
        rows = count(name, t.size(0));
        vocab = count(name, t.size(1));
        ld = t.stride(0);
        if ((vocab > 1 && t.stride(1) != 1) || (rows > 1 && ld < vocab))
            invalid(std::string(name) + " columns must be contiguous and its rows apart, got strides (" + std::to_string(ld) +
                    ", " + std::to_string(t.stride(1)) + ")");
        if (ld < vocab) ld = vocab;
    }
};

template <typename T>
const T* vector(const char* name, PyObject* o, at::ScalarType type, int64_t n, const at::Tensor& with) {
    const at::Tensor& t = tensor(name, o);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || t.device() != with.device())
        invalid(std::string(name) + " must be a contiguous " + name_of(type) + " tensor [" + std::to_string(n) + "] on " +
                with.device().str() + ", got " + told(t));
    return static_cast<const T*>(t.data_ptr());
}

template <typename T>
const T* vector_or_none(const char* name, PyObject* o, at::ScalarType type, int64_t n, const at::Tensor& with) {
    return o == Py_None ? nullptr : vector<T>(name, o, type, n, with);
}

// The device and current stream of a call.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = nullptr;
    explicit On(const at::Tensor& t) {
        if (!t.is_cuda()) invalid("the tensors must be on a GPU");
        guard.set_device(t.device());
        stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
    }
};

// Where the gradient of `logits` goes: the caller's buffer, or a new one.
struct Gradient {
    PyObject* given = nullptr;
    at::Tensor made;
    void* ptr = nullptr;
    long long ld = 0;
    Gradient(PyObject* out, const at::Tensor& logits, bool wanted) {
        if (out == Py_None) return;
        if (!wanted) invalid("a buffer for the gradient without a gradient");
        const at::Tensor& t = tensor("the gradient's buffer", out);
        if (t.scalar_type() != logits.scalar_type() || t.sizes() != logits.sizes() || t.device() != logits.device())
            invalid(std::string("the gradient's buffer must be ") + told(logits) + ", got " + told(t));
        ld = Matrix("the gradient's buffer", t).ld;
        given = out;
        ptr = t.data_ptr();
    }
    void make(const at::Tensor& logits) {
        if (given) return;
        made = at::empty(logits.sizes(), logits.options().requires_grad(false));
        ptr = made.data_ptr();
        ld = logits.size(1);
    }
    PyObject* object() {  // a new reference, after the call
        if (given) {
            // autograd may hold the buffer (the logits themselves) for a backward: that has to fail now
            const at::Tensor& t = THPVariable_Unpack(given);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
            Py_INCREF(given);
            return given;
        }
        if (!made.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(made);
    }
};

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& with) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(with.device()));
}

void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor workspace(size_t bytes, const at::Tensor& with) {
    return bytes ? fresh({(int64_t)bytes}, at::kByte, with) : at::Tensor();
}

PyObject* pack(std::initializer_list<PyObject*> items) {  // steals the references
    PyObject* t = PyTuple_New((Py_ssize_t)items.size());
    Py_ssize_t i = 0;
    for (PyObject* o : items) {
        if (t) PyTuple_SET_ITEM(t, i++, o);
        else Py_XDECREF(o);
    }
    return t;
}

PyObject* raise(const Refused& r) {
    if (!r.code) return nullptr;  // a Python error is set
    PyObject* mod = PyImport_ImportModule("qwen600_engine_b200._lib");
    PyObject* cls = mod ? PyObject_GetAttrString(mod, "SamplerError") : nullptr;
    PyObject* e = cls ? PyObject_CallFunction(cls, "is", r.code, r.msg.c_str()) : nullptr;
    if (e) PyErr_SetObject(cls, e);
    Py_XDECREF(e);
    Py_XDECREF(cls);
    Py_XDECREF(mod);
    return nullptr;
}

template <typename F>
PyObject* call(Py_ssize_t n, Py_ssize_t want, F body) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, want);
        return nullptr;
    }
    try {
        return body();
    } catch (const Refused& r) {
        return raise(r);
    } catch (const std::exception& e) {  // torch's errors, out of memory among them
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (logits, tokens, temperature) -> (logprobs, stats)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 3, [&] {
        const at::Tensor& x = tensor("logits", a[0]);
        const Matrix m("logits", x);
        const int* tok = vector<int>("tokens", a[1], at::kInt, m.rows, x);
        const double T = number(a[2]);
        const On on(x);
        at::Tensor lp = fresh({m.rows}, at::kFloat, x), stats = fresh({m.rows, 2}, at::kFloat, x);
        const size_t size = qs_token_logprobs_workspace(m.dtype, m.rows, m.vocab);
        at::Tensor work = workspace(size, x);
        check(qs_token_logprobs(x.data_ptr(), m.dtype, m.rows, m.vocab, m.ld, tok, T, (float*)lp.data_ptr(),
                                (float*)stats.data_ptr(), pointer(work), size, on.stream));
        return pack({THPVariable_Wrap(lp), THPVariable_Wrap(stats)});
    });
}

// (logits, tokens, stats, grad_logprobs, temperature, out) -> gradient
PyObject* token_logprobs_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 6, [&] {
        const at::Tensor& x = tensor("logits", a[0]);
        const Matrix m("logits", x);
        const int* tok = vector<int>("tokens", a[1], at::kInt, m.rows, x);
        const at::Tensor& st = tensor("stats", a[2]);
        if (st.scalar_type() != at::kFloat || st.dim() != 2 || st.size(0) != m.rows || st.size(1) != 2 ||
            !st.is_contiguous() || st.device() != x.device())
            invalid("stats must be a contiguous float32 tensor [" + std::to_string(m.rows) + ", 2] on " + x.device().str());
        const float* g = vector<float>("grad_logprobs", a[3], at::kFloat, m.rows, x);
        const double T = number(a[4]);
        Gradient grad(a[5], x, true);
        const On on(x);
        grad.make(x);
        check(qs_token_logprobs_backward(x.data_ptr(), m.dtype, m.rows, m.vocab, m.ld, tok, (const float*)st.data_ptr(), g,
                                         T, grad.ptr, grad.ld, on.stream));
        return grad.object();
    });
}

// (logits, tokens, old_logprobs, advantages, ref_logprobs, weights, clip_low, clip_high, kl_coef, temperature, grad, out)
//   -> (loss, logprobs, gradient)
PyObject* policy_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 12, [&] {
        const at::Tensor& x = tensor("logits", a[0]);
        const Matrix m("logits", x);
        const int* tok = vector<int>("tokens", a[1], at::kInt, m.rows, x);
        const float* old = vector<float>("old_logprobs", a[2], at::kFloat, m.rows, x);
        const float* adv = vector<float>("advantages", a[3], at::kFloat, m.rows, x);
        const float* ref = vector_or_none<float>("ref_logprobs", a[4], at::kFloat, m.rows, x);
        const float* w = vector_or_none<float>("weights", a[5], at::kFloat, m.rows, x);
        const qs_policy_params p{number(a[6]), number(a[7]), number(a[8]), number(a[9])};
        const bool wanted = truth(a[10]);
        Gradient grad(a[11], x, wanted);
        const On on(x);
        if (wanted) grad.make(x);
        at::Tensor loss = fresh({}, at::kFloat, x), lp = fresh({m.rows}, at::kFloat, x);
        const size_t size = qs_policy_loss_workspace(m.rows);
        at::Tensor work = workspace(size, x);
        check(qs_policy_loss(x.data_ptr(), m.dtype, m.rows, m.vocab, m.ld, tok, old, ref, adv, w, &p, (float*)loss.data_ptr(),
                             (float*)lp.data_ptr(), grad.ptr, grad.ld, pointer(work), size, on.stream));
        return pack({THPVariable_Wrap(loss), THPVariable_Wrap(lp), grad.object()});
    });
}

// (logits, tokens, seq_offsets, ref_logprobs, weights, beta, label_smoothing, grad, out) -> (loss, seq_logprobs, gradient)
PyObject* preference_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 9, [&] {
        const at::Tensor& x = tensor("logits", a[0]);
        const Matrix m("logits", x);
        const int* tok = vector<int>("tokens", a[1], at::kInt, m.rows, x);
        const at::Tensor& offsets = tensor("seq_offsets", a[2]);
        if (offsets.dim() != 1 || offsets.size(0) % 2 != 1)
            invalid("seq_offsets must be [2 * pairs + 1], got " + shape_of(offsets));
        const int pairs = count("seq_offsets", offsets.size(0) / 2);
        const int* off = vector<int>("seq_offsets", a[2], at::kInt, 2 * (int64_t)pairs + 1, x);
        const float* ref = vector<float>("ref_logprobs", a[3], at::kFloat, 2 * (int64_t)pairs, x);
        const float* w = vector_or_none<float>("weights", a[4], at::kFloat, pairs, x);
        const qs_preference_params p{number(a[5]), number(a[6])};
        const bool wanted = truth(a[7]);
        Gradient grad(a[8], x, wanted);
        const On on(x);
        if (wanted) grad.make(x);
        at::Tensor loss = fresh({}, at::kFloat, x), seq = fresh({2 * (int64_t)pairs}, at::kFloat, x);
        const size_t size = qs_preference_loss_workspace(m.dtype, m.rows, m.vocab);
        at::Tensor work = workspace(size, x);
        check(qs_preference_loss(x.data_ptr(), m.dtype, m.rows, m.vocab, m.ld, tok, off, pairs, ref, w, &p,
                                 (float*)loss.data_ptr(), (float*)seq.data_ptr(), grad.ptr, grad.ld, pointer(work), size,
                                 on.stream));
        return pack({THPVariable_Wrap(loss), THPVariable_Wrap(seq), grad.object()});
    });
}

// (hidden [B, hidden_dim], norm_weight, codes, scales, zeros, vocab, hidden_dim, group, scale dtype) -> (normed, logits)
PyObject* lm_head_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 9, [&] {
        const at::Tensor& h = tensor("hidden", a[0]);
        const void* norm = a[1] == Py_None ? nullptr : tensor("norm_weight", a[1]).data_ptr();
        const at::Tensor& codes = tensor("codes", a[2]);
        const at::Tensor& scales = tensor("scales", a[3]);
        const void* zeros = a[4] == Py_None ? nullptr : tensor("zeros", a[4]).data_ptr();
        const qs_w4_weight w{codes.data_ptr(),          scales.data_ptr(),          zeros,
                             (int)PyLong_AsLong(a[5]), (int)PyLong_AsLong(a[6]), (int)PyLong_AsLong(a[7]),
                             (int)PyLong_AsLong(a[8])};
        if (PyErr_Occurred()) throw Refused{0, ""};
        const int batch = count("hidden", h.size(0));
        const On on(codes);
        at::Tensor normed = fresh({batch, w.hidden_dim}, at::kBFloat16, codes);
        at::Tensor logits = fresh({batch, w.vocab}, at::kBFloat16, codes);
        if (batch) {
            const size_t size = qs_lm_head_w4_workspace(batch, w.hidden_dim);
            at::Tensor work = workspace(size, codes);
            check(qs_lm_head_w4(h.data_ptr(), norm, &w, batch, normed.data_ptr(), logits.data_ptr(), pointer(work), size,
                                on.stream));
        }
        return pack({THPVariable_Wrap(normed), THPVariable_Wrap(logits)});
    });
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(token_logprobs), FAST(token_logprobs_backward), FAST(policy_loss), FAST(preference_loss),
                         FAST(lm_head_w4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch", "torch tensors to the C ABI of libqwen600_sampler.so", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch(void) { return PyModule_Create(&module); }
