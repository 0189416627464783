// Python binding of the int8 operators on torch tensors: sigcomp_b200._int8, which sigcomp_b200.int8
// documents.  Checks the arguments, allocates results and workspace from torch's allocator (so that
// captured graphs and streams each have their own) and calls the C entry points.  It is compiled because
// a call's kernels take a few microseconds, and the same steps in Python took 14 to 25.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/sigcomp_b200.h"

namespace {

struct Refused {
    std::string text;
};

[[noreturn]] void refuse(const char *fmt, ...)
{
    char buf[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    throw Refused{buf};
}

// torch types <-> SC_TYPE_*, -1 for others
int sc_type(c10::ScalarType t)
{
    switch (t) {
    case c10::ScalarType::Float: return SC_TYPE_F32;
    case c10::ScalarType::Half: return SC_TYPE_F16;
    case c10::ScalarType::BFloat16: return SC_TYPE_BF16;
    case c10::ScalarType::Char: return SC_TYPE_I8;
    default: return -1;
    }
}
enum { F32 = 1 << SC_TYPE_F32, FLOATS = F32 | 1 << SC_TYPE_F16 | 1 << SC_TYPE_BF16, I8 = 1 << SC_TYPE_I8 };

const char *type_names(int types)
{
    return types == I8 ? "torch.int8" : types == F32 ? "torch.float32"
           : types == FLOATS ? "torch.float32, torch.float16 or torch.bfloat16"
                             : "torch.float32, torch.float16, torch.bfloat16 or torch.int8";
}

const at::Tensor &tensor(const char *name, PyObject *o, int types, const at::Tensor *beside = nullptr)
{
    if (!THPVariable_Check(o)) refuse("%s must be a torch tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    const int type = sc_type(t.scalar_type());
    if (type < 0 || !(types >> type & 1)) refuse("%s must be of type %s, not %s", name, type_names(types), c10::toString(t.scalar_type()));
    if (t.layout() != c10::kStrided || t.is_neg()) refuse("%s must be a dense tensor, not a lazily negated one", name);
    if (beside && t.device() != beside->device())
        refuse("%s is on %s, the other arrays are on %s", name, t.device().str().c_str(), beside->device().str().c_str());
    if (t.unsafeGetTensorImpl()->autograd_meta()) {                // without it a tensor has neither
        if (t.requires_grad() && c10::GradMode::is_enabled())
            refuse("%s asks for a gradient, which the int8 operators do not have", name);
        // a dual tensor: its tangent would be lost
        if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
            refuse("%s asks for a forward derivative, which the int8 operators do not have", name);
    }
    return t;
}

std::string shape_of(c10::IntArrayRef s)
{
    std::string o = "(";
    for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
    return o + (s.size() == 1 ? ",)" : ")");
}

void rows_there(const char *name, const at::Tensor &t)
{
    if (t.dim() == 0 || t.size(-1) == 0) refuse("%s must have rows of at least one element", name);
}

// t as rows: a view where its strides allow one, else a copy
at::Tensor as_rows(const at::Tensor &t)
{
    at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

void on_gpu(const at::Tensor &t)
{
    if (!t.is_cuda()) refuse("the int8 operators run on a GPU: move the arrays there");
}

at::Tensor vector_of(const char *name, PyObject *o, int64_t length, const at::Tensor &beside)
{
    const at::Tensor &t = tensor(name, o, F32, &beside);
    if (t.dim() != 1 || t.size(0) != length)
        refuse("%s must have %lld elements, not shape %s", name, (long long)length, shape_of(t.sizes()).c_str());
    return t;
}

at::Tensor row_scales(const char *name, PyObject *o, c10::IntArrayRef lead, const at::Tensor &beside)
{
    const at::Tensor &t = tensor(name, o, F32, &beside);
    if (t.sizes() != lead)
        refuse("%s must have shape %s, one scale for each row, not %s", name, shape_of(lead).c_str(), shape_of(t.sizes()).c_str());
    return t;
}

const float *floats_of(at::Tensor &t)
{
    if (!t.defined()) return nullptr;
    if (!t.is_contiguous()) t = t.contiguous();
    return (const float *)t.data_ptr();
}

at::Tensor empty(c10::IntArrayRef sizes, c10::ScalarType type, const at::Tensor &beside)
{
    return at::detail::empty_cuda(sizes, type, beside.device(), c10::nullopt);
}

// elements from row to row of results: a multiple of 16 bytes, as the kernels read and write whole vectors
int64_t padded(int64_t cols, c10::ScalarType type)
{
    const int64_t vec = 16 / (int64_t)c10::elementSize(type);
    return (cols + vec - 1) / vec * vec;
}

at::Tensor empty_rows(c10::IntArrayRef lead, int64_t cols, c10::ScalarType type, const at::Tensor &beside)
{
    c10::SmallVector<int64_t, 6> sizes(lead.begin(), lead.end()), strides(lead.size() + 1);
    sizes.push_back(cols);
    int64_t step = padded(cols, type);
    strides[lead.size()] = 1;
    for (size_t i = lead.size(); i-- > 0;) {
        strides[i] = step;
        step *= lead[i] > 0 ? lead[i] : 1;
    }
    return at::detail::empty_strided_cuda(sizes, strides, type, beside.device());
}

void *stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

c10::IntArrayRef leading(const at::Tensor &t) { return t.sizes().slice(0, t.dim() - 1); }

// the distance of rows; of a single row any distance will do, and its own length is always a valid one
int64_t row_stride(const at::Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : (rows.size(1) + 15) / 16 * 16; }

// Other Python threads run meanwhile, as they do during torch's own calls: an allocation can wait for the GPU, and so
// can a launch where the stream's queue is full, perhaps for work that another thread has yet to launch.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

struct Failed {
    int status;
};

void check(int status)
{
    if (status != SC_OK) throw Failed{status};
}

// float types only; `fallback` for None
c10::ScalarType float_type(PyObject *o, c10::ScalarType fallback, const char *more)
{
    if (o == Py_None) return fallback;
    if (THPDtype_Check(o)) {
        const c10::ScalarType t = reinterpret_cast<THPDtype *>(o)->scalar_type;
        const int type = sc_type(t);
        if (type >= 0 && (FLOATS >> type & 1)) return t;
    }
    refuse("dtype must be one of %s%s", type_names(FLOATS), more);
}

PyObject *pair(at::Tensor a, at::Tensor b)
{
    PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
    PyObject *r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, x);
    PyTuple_SET_ITEM(r, 1, y);
    return r;
}

PyObject *quantize(PyObject *const *a)
{
    const at::Tensor x = tensor("x", a[0], FLOATS);
    rows_there("x", x);
    on_gpu(x);
    at::Tensor q, s;
    {
        Unlocked unlocked;
        at::Tensor rows = as_rows(x);
        q = empty_rows(leading(x), x.size(-1), c10::ScalarType::Char, x);
        s = empty(leading(x), c10::ScalarType::Float, x);
        check(sc_quantize_tokens_device(x.device().index(), rows.data_ptr(), sc_type(x.scalar_type()), rows.size(0), rows.size(1),
                                        row_stride(rows), (int8_t *)q.data_ptr(), padded(x.size(-1), c10::ScalarType::Char),
                                        (float *)s.data_ptr(), stream_of(x)));
    }
    return pair(std::move(q), std::move(s));
}

PyObject *dequantize(PyObject *const *a)
{
    const at::Tensor q = tensor("q", a[0], I8);
    const c10::ScalarType type = float_type(a[2], c10::ScalarType::Float, "");
    rows_there("q", q);
    at::Tensor scales, y;
    double one = 0;
    if (THPVariable_Check(a[1])) {
        scales = row_scales("scales", a[1], leading(q), q);
    } else {
        one = PyFloat_AsDouble(a[1]);
        if (one == -1.0 && PyErr_Occurred()) return nullptr;
    }
    on_gpu(q);
    {
        Unlocked unlocked;
        at::Tensor rows = as_rows(q);
        y = empty_rows(leading(q), q.size(-1), type, q);
        check(sc_dequantize_tokens_device(q.device().index(), (const int8_t *)rows.data_ptr(), row_stride(rows),
                                          floats_of(scales), (float)one, rows.size(0), rows.size(1), y.data_ptr(),
                                          sc_type(type), padded(q.size(-1), type), stream_of(q)));
    }
    return THPVariable_Wrap(std::move(y));
}

// x, x_scales, weight, weight_scales, bias, relu, then as y_type says: the type's object, or output_scale
PyObject *linear(PyObject *const *a, bool int8_out)
{
    const at::Tensor x = tensor(int8_out ? "q" : "x", a[0], int8_out ? I8 : FLOATS | I8);
    const bool quantised = x.scalar_type() == c10::ScalarType::Char;
    c10::ScalarType type = c10::ScalarType::Char;
    double output_scale = 0;
    if (!int8_out) {
        type = float_type(a[6], quantised ? c10::ScalarType::Float : x.scalar_type(), "; int8_linear_requant gives int8");
    } else if (a[6] != Py_None) {
        output_scale = PyFloat_AsDouble(a[6]);
        if (output_scale == -1.0 && PyErr_Occurred()) return nullptr;
        if (!std::isfinite(output_scale) || !((float)output_scale > 0) || !std::isfinite((float)output_scale))
            refuse("output_scale must be a finite positive number");
    }
    const bool row_out = int8_out && a[6] == Py_None;
    const at::Tensor weight = tensor("weight", a[2], I8, &x);
    if (weight.dim() != 2 || weight.size(0) == 0 || weight.size(1) == 0) refuse("weight must be [out, in], both at least 1");
    const int64_t n = weight.size(0), k = weight.size(1);
    if (k > SC_INT8_MAX_K) refuse("rows of more than %d elements could overflow a 32-bit sum", SC_INT8_MAX_K);
    if (x.dim() == 0 || x.size(-1) != k)
        refuse("x has shape %s, weight takes rows of %lld", shape_of(x.sizes()).c_str(), (long long)k);
    at::Tensor ws = vector_of("weight_scales", a[3], n, x), bias, xs, y, y_scales;
    if (a[4] != Py_None) bias = vector_of("bias", a[4], n, x);
    if (quantised) {
        if (a[1] == Py_None) refuse("int8 rows need x_scales");
        xs = row_scales("x_scales", a[1], leading(x), x);
    } else if (a[1] != Py_None) {
        refuse("x_scales belong to int8 rows; float rows are quantised here");
    }
    const int relu = PyObject_IsTrue(a[5]);
    if (relu < 0) return nullptr;
    on_gpu(x);
    {
        Unlocked unlocked;
        at::Tensor rows = as_rows(x), w = as_rows(weight), work;
        if (n > 1 && w.stride(0) < k) w = w.contiguous();       // rows that overlap, as those of an expanded row do
        const int64_t m = rows.size(0), x_stride = row_stride(rows), w_stride = row_stride(w);
        const int xt = sc_type(x.scalar_type()), yt = sc_type(type);
        y = empty_rows(leading(x), n, type, x);
        const int64_t y_stride = padded(n, type);
        if (row_out) y_scales = empty(leading(x), c10::ScalarType::Float, x);
        const int x_packed = ((uintptr_t)rows.data_ptr() | (uintptr_t)x_stride) % 16 == 0 && x_stride >= k;
        const int w_packed = ((uintptr_t)w.data_ptr() | (uintptr_t)w_stride) % 16 == 0;
        const int64_t bytes = sc_int8_linear_workspace(xt, x_packed, w_packed, m, n, k, yt, row_out);
        if (bytes > 0) work = empty({bytes}, c10::ScalarType::Byte, x);
        if (m > 0)
            check(sc_int8_linear_device(x.device().index(), rows.data_ptr(), xt, x_stride, floats_of(xs),
                                        (const int8_t *)w.data_ptr(), w_stride, floats_of(ws), floats_of(bias), m, n, k, relu,
                                        y.data_ptr(), yt, y_stride, row_out ? (float *)y_scales.data_ptr() : nullptr,
                                        (float)output_scale, bytes > 0 ? work.data_ptr() : nullptr, bytes, stream_of(x)));
    }
    if (row_out) return pair(std::move(y), std::move(y_scales));
    return THPVariable_Wrap(std::move(y));
}

PyObject *failed(int status)
{
    // the exceptions of sigcomp_b200._lib.check
    PyObject *lib = PyImport_ImportModule("sigcomp_b200._lib");
    if (!lib) return nullptr;
    PyObject *r = PyObject_CallMethod(lib, "raise_status", "is", status, sc_last_error());
    Py_XDECREF(r);
    Py_DECREF(lib);
    return nullptr;
}

template <typename F>
PyObject *guarded(Py_ssize_t given, Py_ssize_t wanted, F &&f)
{
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments wanted, %zd given", wanted, given);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_ValueError, e.text.c_str());
    } catch (const Failed &e) {
        return failed(e.status);
    } catch (const c10::OutOfMemoryError &e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject *py_quantize(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 1, [&] { return quantize(a); });
}
PyObject *py_dequantize(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 3, [&] { return dequantize(a); });
}
PyObject *py_linear(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 7, [&] { return linear(a, false); });
}
PyObject *py_linear_requant(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 7, [&] { return linear(a, true); });
}

PyMethodDef methods[] = {
    {"quantize_tokens", (PyCFunction)(void (*)(void))py_quantize, METH_FASTCALL, nullptr},
    {"dequantize_tokens", (PyCFunction)(void (*)(void))py_dequantize, METH_FASTCALL, nullptr},
    {"int8_linear", (PyCFunction)(void (*)(void))py_linear, METH_FASTCALL, nullptr},
    {"int8_linear_requant", (PyCFunction)(void (*)(void))py_linear_requant, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "sigcomp_b200._int8", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__int8(void)
{
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", SC_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
