// The device operators on torch tensors: argument checks and allocation for
// azb_ops.py, straight onto the C ABI (include/azb200.h). A small operator's
// call is mostly host time, so this is a plain extension module (vector call,
// no keyword parsing); azb_ops.py has the documented functions.
//
// Bad arguments raise ValueError, failures of the device azb200.CudaError; no
// C++ exception leaves a function of this module.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <string>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <azb200.h>

namespace {

PyObject* cuda_error = nullptr;   // azb200.CudaError

struct Refused {
    std::string what;
};
struct Raised {};   // a Python error is set

template <class Fn>
PyObject* guarded(Fn fn) {
    try {
        return fn();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what.c_str());
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "azb_torch: unknown error");
    }
    return nullptr;
}

void require(bool ok, const std::string& what) {
    if (!ok) throw Refused{what};
}

// A C entry's message buffer.
struct Err {
    char text[1024] = "";
    void check(int rc) const {
        if (rc == 0) return;
        if (std::strncmp(text, "cuda", 4) == 0 || std::strstr(text, ": cuda")) {
            PyErr_SetString(cuda_error, text);
            throw Raised{};
        }
        throw Refused{text};
    }
};

void want(Py_ssize_t n, Py_ssize_t wanted) {
    if (n != wanted) {
        PyErr_Format(PyExc_TypeError, "azb_torch: %zd arguments, not %zd", wanted, n);
        throw Raised{};
    }
}

long long whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

std::string name_of(const at::Device& d) { return d.str(); }

int elem_type(at::ScalarType t, const char* what) {
    if (t == at::kFloat) return AZB_ELEM_F32;
    if (t == at::kBFloat16) return AZB_ELEM_BF16;
    throw Refused{std::string(what) + ": float32 or bfloat16, not " + c10::toString(t)};
}

at::ScalarType scalar_type(long long code) { return code == AZB_ELEM_F32 ? at::kFloat : at::kBFloat16; }

const at::Tensor& tensor(PyObject* o, const char* what) {
    require(THPVariable_Check(o), std::string(what) + ": a CUDA tensor is needed");
    const at::Tensor& t = THPVariable_Unpack(o);
    require(t.is_cuda(), std::string(what) + ": a CUDA tensor is needed");
    return t;
}

// A two-dimensional source with adjacent columns.
struct Matrix {
    int type;
    long long rows, cols, ld;
    const void* at;
};

// That a tensor's memory holds its values, and that nothing follows them. A
// gradient, or a forward-mode tangent, would be lost: there is no backward pass.
void check_source(const at::Tensor& t, const char* what) {
    const auto refuse = [&](const char* why) { throw Refused{std::string(what) + why}; };
    if ((t.requires_grad() && c10::GradMode::is_enabled()) ||
        (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()))
        refuse(" requires a gradient, and there is no backward pass (detach it)");
    if (t.is_neg()) refuse(" is a view of negated memory (resolve_neg it)");
    if (t.key_set().has(c10::DispatchKey::Python))
        refuse(" is of a tensor subclass with a dispatch of its own, which these calls would bypass");
    if (!t.has_storage()) refuse(" stands for other tensors (a transform's, say) and has no memory to read");
}

// These calls run below torch's dispatcher: a trace would hold their results
// as constants.
void check_untraced() {
    using Mode = c10::impl::TorchDispatchModeKey;
    using Modes = c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing() || (Modes::any_modes_set() && (Modes::get_mode(Mode::FAKE) || Modes::get_mode(Mode::PROXY) ||
                                                                       Modes::get_mode(Mode::FUNCTIONAL))))
        throw Refused{"these calls cannot be traced (capture them into a CUDA graph instead)"};
}

Matrix matrix(const at::Tensor& t, const char* what) {
    Matrix m{};
    m.type = elem_type(t.scalar_type(), what);
    require(t.dim() == 2, std::string(what) + ": a matrix is needed, not " + std::to_string(t.dim()) + " dimensions");
    check_source(t, what);
    m.rows = t.size(0);
    m.cols = t.size(1);
    require(m.cols >= 1, std::string(what) + ": at least one column is needed");
    require(m.cols == 1 || t.stride(1) == 1,
            std::string(what) + ": columns must be adjacent (stride " + std::to_string(t.stride(1)) + ")");
    m.ld = t.stride(0);
    m.at = t.const_data_ptr();
    return m;
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Device& device) {
    return at::detail::empty_cuda(size, type, device, std::nullopt);
}

void* stream(const at::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

long long round_256(long long n) { return (n + 255) / 256 * 256; }

// A quantised matrix as azb_ops.Mx4 holds it: codes, then from the next
// multiple of 256 bytes the scales.
struct Quantised {
    long long rows, cols;
    long long code_bytes() const { return rows * ((cols + 31) / 32) * 16; }
    long long scale_bytes() const { return (rows + 127) / 128 * (((cols + 31) / 32 + 3) / 4) * 512; }
    long long scales_at() const { return round_256(code_bytes()); }
    long long bytes() const { return scales_at() + scale_bytes(); }
};

const uint8_t* quantised_data(const at::Tensor& data, const Quantised& q, const char* what) {
    require(data.scalar_type() == at::kByte && data.dim() == 1 && data.is_contiguous() && data.numel() == q.bytes(),
            std::string(what) + ": not the data of an Mx4 of " + std::to_string(q.rows) + " x " + std::to_string(q.cols));
    return static_cast<const uint8_t*>(data.const_data_ptr());
}

// mx4_quantise(x) -> (data, rows, cols)
PyObject* mx4_quantise(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 1);
        check_untraced();
        const at::Tensor& x = tensor(args[0], "x");
        const Matrix m = matrix(x, "x");
        const Quantised q{m.rows, m.cols};
        Err err;
        err.check(azb_mx4_sizes(m.rows, m.cols, nullptr, nullptr, err.text, sizeof err.text));
        const at::Device device = x.device();
        at::Tensor data = empty({q.bytes()}, at::kByte, device);
        uint8_t* p = static_cast<uint8_t*>(data.mutable_data_ptr());
        err.check(azb_mx4_quantise(device.index(), m.at, m.type, m.rows, m.cols, m.ld, p, p + q.scales_at(), stream(device),
                                   err.text, sizeof err.text));
        PyObject* made = PyTuple_New(3);
        if (!made) throw Raised{};
        PyTuple_SET_ITEM(made, 0, THPVariable_Wrap(std::move(data)));
        PyTuple_SET_ITEM(made, 1, PyLong_FromLongLong(m.rows));
        PyTuple_SET_ITEM(made, 2, PyLong_FromLongLong(m.cols));
        return made;
    });
}

// mx4_values(data, rows, cols, type) -> values
PyObject* mx4_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 4);
        check_untraced();
        const at::Tensor& data = tensor(args[0], "q");
        const Quantised q{whole(args[1]), whole(args[2])};
        const uint8_t* p = quantised_data(data, q, "q");
        const int type = int(whole(args[3]));
        const at::Device device = data.device();
        at::Tensor out = empty({q.rows, q.cols}, scalar_type(type), device);
        Err err;
        err.check(azb_mx4_values(device.index(), p, p + q.scales_at(), q.rows, q.cols, out.mutable_data_ptr(), type, q.cols,
                                 stream(device), err.text, sizeof err.text));
        return THPVariable_Wrap(std::move(out));
    });
}

// mx4_product(x, x rows or -1: plain, x cols, w data, w rows, w cols, bias or
// None, relu, type or -1: x's) -> out
PyObject* mx4_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 9);
        check_untraced();
        const long long x_rows = whole(args[1]);
        const bool plain = x_rows < 0;
        at::Tensor x = tensor(args[0], "x");
        const bool vector = plain && x.dim() == 1;
        if (vector) x = x.unsqueeze(0);
        Matrix m{};
        if (plain) m = matrix(x, "x");
        else m.rows = x_rows, m.cols = whole(args[2]);
        const at::Tensor& w_data = tensor(args[3], "w");
        const Quantised w{whole(args[4]), whole(args[5])};
        require(m.cols == w.cols, "x has " + std::to_string(m.cols) + " columns, w " + std::to_string(w.cols));
        const long long asked = whole(args[8]);
        const int type = asked >= 0 ? int(asked) : m.type;
        const at::Device device = x.device();
        require(w_data.device() == device, "x is on " + name_of(device) + ", w on " + name_of(w_data.device()));
        const float* bias = nullptr;
        if (args[6] != Py_None) {
            const bool fits = THPVariable_Check(args[6]) && [&] {
                const at::Tensor& b = THPVariable_Unpack(args[6]);
                return b.scalar_type() == at::kFloat && b.dim() == 1 && b.size(0) == w.rows && b.is_contiguous();
            }();
            require(fits, "bias: " + std::to_string(w.rows) + " adjacent float32 numbers are needed");
            const at::Tensor& b = THPVariable_Unpack(args[6]);
            require(b.device() == device, "x is on " + name_of(device) + ", bias on " + name_of(b.device()));
            check_source(b, "bias");
            bias = static_cast<const float*>(b.const_data_ptr());
        }
        const int relu = PyObject_IsTrue(args[7]);
        if (relu < 0) throw Raised{};
        const uint8_t* wp = quantised_data(w_data, w, "w");
        at::Tensor out = empty({m.rows, w.rows}, scalar_type(type), device);
        Err err;
        if (plain) {
            const size_t need = azb_mx4_linear_workspace(m.rows, w.rows, m.cols);
            at::Tensor work;
            if (need) work = empty({static_cast<long long>(need)}, at::kByte, device);
            err.check(azb_mx4_linear(device.index(), m.at, m.type, m.rows, m.cols, m.ld, wp, wp + w.scales_at(), w.rows, bias,
                                     relu, out.mutable_data_ptr(), type, w.rows, need ? work.mutable_data_ptr() : nullptr, need,
                                     stream(device), err.text, sizeof err.text));
        } else {
            const Quantised xq{m.rows, m.cols};
            const uint8_t* xp = quantised_data(x, xq, "x");
            err.check(azb_mx4_product(device.index(), xp, xp + xq.scales_at(), m.rows, wp, wp + w.scales_at(), w.rows, m.cols,
                                      bias, relu, out.mutable_data_ptr(), type, w.rows, stream(device), err.text,
                                      sizeof err.text));
        }
        return THPVariable_Wrap(vector ? out.select(0, 0) : std::move(out));
    });
}

// A setting: one number, or one per row.
template <class T>
void setting(PyObject* o, const char* name, long long rows, const at::Device& device, at::ScalarType type, const char* type_name,
             T* one, const T** each) {
    *each = nullptr;
    if (!THPVariable_Check(o)) {
        if (type == at::kInt) *one = T(std::clamp<long long>(whole(o), INT_MIN, INT_MAX));
        else *one = T(number(o));
        return;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    require(t.scalar_type() == type && t.dim() == 1 && t.size(0) == rows && t.device() == device && t.is_contiguous(),
            std::string(name) + ": a number, or " + std::to_string(rows) + " adjacent " + type_name + " numbers on " +
                name_of(device));
    check_source(t, name);
    *one = T(0);
    *each = static_cast<const T*>(t.const_data_ptr());
}

// One of the sampler's arrays of logits' shape, or null for None.
const void* beside(PyObject* o, const char* name, const at::Tensor& logits, const char* types, bool (*fits)(at::ScalarType),
                   long long* ld) {
    *ld = 0;
    if (o == Py_None) return nullptr;
    require(THPVariable_Check(o), std::string(name) + ": " + types + " of logits' shape is needed");
    const at::Tensor& t = THPVariable_Unpack(o);
    require(fits(t.scalar_type()) && t.sizes() == logits.sizes(), std::string(name) + ": " + types + " of logits' shape is needed");
    require((t.size(1) == 1 || t.stride(1) == 1) && t.device() == logits.device(),
            std::string(name) + ": adjacent columns on " + name_of(logits.device()) + " are needed (stride " +
                std::to_string(t.stride(1)) + "; it is on " + name_of(t.device()) + ")");
    check_source(t, name);
    *ld = t.stride(0);
    return t.const_data_ptr();
}

// sample_moves(logits, noise or None, legal or None, temperature, top_k,
// top_p, min_p) -> (moves, logprob)
PyObject* sample_moves(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want(n, 7);
        check_untraced();
        const at::Tensor& logits = tensor(args[0], "logits");
        const Matrix m = matrix(logits, "logits");
        const at::Device device = logits.device();
        azb_sample_args a{};
        a.logits = m.at;
        a.type = m.type;
        a.rows = m.rows;
        a.cols = m.cols;
        a.ld = m.ld;
        a.noise = static_cast<const float*>(
            beside(args[1], "noise", logits, "float32", [](at::ScalarType t) { return t == at::kFloat; }, &a.noise_ld));
        a.legal = static_cast<const uint8_t*>(
            beside(args[2], "legal", logits, "bool or uint8", [](at::ScalarType t) { return t == at::kBool || t == at::kByte; },
                   &a.legal_ld));
        setting(args[3], "temperature", m.rows, device, at::kFloat, "float32", &a.temperature, &a.temperature_rows);
        setting(args[4], "top_k", m.rows, device, at::kInt, "int32", &a.top_k, &a.top_k_rows);
        setting(args[5], "top_p", m.rows, device, at::kFloat, "float32", &a.top_p, &a.top_p_rows);
        setting(args[6], "min_p", m.rows, device, at::kFloat, "float32", &a.min_p, &a.min_p_rows);
        at::Tensor moves = empty({m.rows}, at::kLong, device), logprob = empty({m.rows}, at::kFloat, device);
        a.moves = static_cast<int64_t*>(moves.mutable_data_ptr());
        a.logprob = static_cast<float*>(logprob.mutable_data_ptr());
        Err err;
        err.check(azb_sample_moves(device.index(), &a, stream(device), err.text, sizeof err.text));
        PyObject* pair = PyTuple_New(2);
        if (!pair) throw Raised{};
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(moves)));
        PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(logprob)));
        return pair;
    });
}

PyMethodDef methods[] = {
    {"mx4_quantise", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(mx4_quantise)), METH_FASTCALL, nullptr},
    {"mx4_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(mx4_values)), METH_FASTCALL, nullptr},
    {"mx4_product", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(mx4_product)), METH_FASTCALL, nullptr},
    {"sample_moves", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sample_moves)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_azb_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__azb_torch(void) {
    PyObject* engine = PyImport_ImportModule("azb200");
    if (!engine) return nullptr;
    cuda_error = PyObject_GetAttrString(engine, "CudaError");
    Py_DECREF(engine);
    return cuda_error ? PyModule_Create(&module) : nullptr;
}
