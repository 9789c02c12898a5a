// The Python module infmoe_b200._binding: checks of arguments, outputs and calls of the operators on torch tensors that stand in
// topk.py and adapters.py.  Through ctypes, torch.empty and shapes read in Python a call took 12 to 13 us of host time, here it
// takes 3.5 to 4.7 (4 to 9 on a slower host): what bounds a small batch, whose kernels take 2 to 3.  Everything else goes through ctypes (capi.py).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstring>
#include <string>

#include "infmoe_c.h"

namespace {

struct Refused {};   // a Python exception is set

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    PyErr_SetString(PyExc_ValueError, text);
    throw Refused{};
}

// InfMoEError for a status that is not 0 (capi.check)
void check(int status) {
    if (status == INFMOE_OK) return;
    PyObject* capi = PyImport_ImportModule("infmoe_b200.capi");
    PyObject* r = capi ? PyObject_CallMethod(capi, "check", "i", status) : nullptr;
    Py_XDECREF(r);
    Py_XDECREF(capi);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "capi.check accepted a status that is not 0");
    throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse("%s must be a torch tensor", what);
    return THPVariable_Unpack(o);
}
at::Tensor optional(PyObject* o, const char* what) { return o == Py_None ? at::Tensor() : tensor(o, what); }
const at::Tensor* given(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return INFMOE_F32;
        case at::kHalf: return INFMOE_F16;
        case at::kBFloat16: return INFMOE_BF16;
        default: refuse("tensors of %s are not supported: use float32, float16 or bfloat16", c10::toString(t.scalar_type()));
    }
}

// A size that the C ABI takes in 32 bits.
int32_t size32(int64_t n, const char* what) {
    if (n > INT32_MAX) refuse("%s is too large (%lld)", what, (long long)n);
    return (int32_t)n;
}

// Rows of a CUDA tensor [..., width] and the stride between them: any stride for [T, width], contiguous otherwise.
struct Rows {
    int64_t count, ld;
};
Rows rows_of(const at::Tensor& t, int64_t width, const char* what) {
    if (!t.is_cuda() || t.dim() < 1 || t.size(-1) != width || (width > 1 && t.stride(-1) != 1))
        refuse("%s must be a CUDA tensor [..., %lld] with consecutive elements in a row", what, (long long)width);
    Rows r{width ? t.numel() / width : 0, width};
    if (t.dim() == 2 && r.count > 1) {
        r.ld = t.stride(0);
        if (r.ld < width) refuse("the rows of %s overlap (stride %lld)", what, (long long)r.ld);
    } else if (t.dim() > 2 && !t.is_contiguous()) {
        refuse("%s must be contiguous (or two-dimensional)", what);
    }
    return r;
}

void check_array(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, const char* what) {
    if (t.scalar_type() != type || t.sizes() != shape || t.device() != device || !t.is_contiguous()) {
        std::string s;
        for (int64_t n : shape) s += (s.empty() ? "" : ", ") + std::to_string(n);
        refuse("%s must be a contiguous %s tensor of shape [%s] on %s", what, c10::toString(type), s.c_str(), device.str().c_str());
    }
}

// The caller's tensor for an output, or a new one.
at::Tensor output(PyObject* given, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, const char* what) {
    if (given == Py_None) return at::detail::empty_cuda(shape, type, device, std::nullopt);
    const at::Tensor& t = tensor(given, what);
    check_array(t, shape, type, device, what);
    return t;
}

void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Device and torch's current stream for the call.
struct On {
    explicit On(const at::Tensor& t) : guard(t.device()), current(c10::cuda::getCurrentCUDAStream(t.device().index())), stream(current.stream()) {}
    // Memory that a plan or a set allocated itself, on stream `home` (a handle; None: it is the caller's), is not given to others of that
    // stream before this one is done with it.
    void uses(const at::Tensor& t, PyObject* home) const {
        if (home == Py_None) return;
        void* const h = PyLong_AsVoidPtr(home);
        if (!h && PyErr_Occurred()) throw Refused{};
        if (h != stream) t.record_stream(current.unwrap());
    }
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream current;
    void* stream;
};

c10::SmallVector<int64_t, 6> with_last(const at::Tensor& t, int64_t last) {
    c10::SmallVector<int64_t, 6> shape(t.sizes().begin(), t.sizes().end());
    shape.back() = last;
    return shape;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject* t = PyTuple_New(2);
    if (!t) throw Refused{};
    PyTuple_SET_ITEM(t, 0, wrap(a));
    PyTuple_SET_ITEM(t, 1, wrap(b));
    return t;
}

// A structure of the C ABI that Python holds as bytes-like memory (a ctypes.Structure).
template <typename T>
struct Held {
    explicit Held(PyObject* o) {
        if (PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) != 0) throw Refused{};
        if (view.len != (Py_ssize_t)sizeof(T)) {
            PyBuffer_Release(&view);
            refuse("a structure of %zd bytes, %zu expected", view.len, sizeof(T));
        }
    }
    ~Held() { PyBuffer_Release(&view); }
    const T* operator->() const { return static_cast<const T*>(view.buf); }
    const T* get() const { return static_cast<const T*>(view.buf); }
    Py_buffer view;
};

template <PyObject* (*F)(PyObject* const*)>
struct Entry {
    template <int N>
    static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
        if (n != N) {
            PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
            return nullptr;
        }
        try {
            return F(args);
        } catch (const Refused&) {
            return nullptr;
        } catch (...) {
            torch::translate_exception_to_python(std::current_exception());     // torch's own, running out of memory among them
        }
        return nullptr;
    }
};

// (config, logits, bias, gate, weight, status) -> (gate, weight)
PyObject* select_topk(PyObject* const* a) {
    const Held<infmoe_topk_config> cfg(a[0]);
    const at::Tensor& logits = tensor(a[1], "logits");
    const at::Tensor bias = optional(a[2], "bias"), status = optional(a[5], "status");
    const Rows rows = rows_of(logits, cfg->expert_count, "logits");
    const int dtype = dtype_code(logits);
    const at::Device device = logits.device();
    if (bias.defined()) check_array(bias, {cfg->expert_count}, at::kFloat, device, "the router's bias");
    if (status.defined()) check_array(status, {1}, at::kInt, device, "status");
    const auto shape = with_last(logits, cfg->top_k);
    const at::Tensor gate = output(a[3], shape, at::kInt, device, "gate"), weight = output(a[4], shape, at::kFloat, device, "weight");
    const On on(logits);
    check(infmoe_expert_select_topk(cfg.get(), rows.count, logits.data_ptr(), dtype, rows.ld, (const float*)data(bias),
                                    (int32_t*)gate.data_ptr(), (float*)weight.data_ptr(), (int32_t*)data(status), on.stream));
    return pair(gate, weight);
}

// (x, pos, offset, top_k, out, row_of) -> (out, row_of)
PyObject* scatter_topk(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "x"), &pos = tensor(a[1], "pos"), &offset = tensor(a[2], "offset");
    const long long k = PyLong_AsLongLong(a[3]);
    if (k == -1 && PyErr_Occurred()) throw Refused{};
    if (x.dim() < 1) refuse("x must be [..., D]");
    if (k < 1 || k > INT32_MAX) refuse("top_k must be at least 1");
    const int64_t D = x.size(-1);
    const Rows rows = rows_of(x, D, "x");
    const at::Device device = x.device();
    check_array(pos, {rows.count * k}, at::kInt, device, "pos");
    if (offset.dim() != 1 || offset.numel() < 1) refuse("offset must hold expert_count + 1 row numbers");
    check_array(offset, offset.sizes(), at::kInt, device, "offset");
    const at::Tensor out = output(a[4], {rows.count * k, D}, x.scalar_type(), device, "out");
    const at::Tensor row_of = output(a[5], {rows.count, k}, at::kInt, device, "row_of");
    const On on(x);
    check(infmoe_expert_scatter_topk(rows.count, (int32_t)k, size32(D, "D"), dtype_code(x), x.data_ptr(), rows.ld, (const int32_t*)pos.data_ptr(),
                                     (const int32_t*)offset.data_ptr() + (offset.numel() - 1), out.data_ptr(), (int32_t*)row_of.data_ptr(),
                                     on.stream));
    return pair(out, row_of);
}

// (rows, weight, row_of, gate, residual, out) -> out
PyObject* combine_topk(PyObject* const* a) {
    const at::Tensor &rows = tensor(a[0], "rows"), &weight = tensor(a[1], "weight");
    const at::Tensor row_of = optional(a[2], "row_of"), gate = optional(a[3], "gate"), residual = optional(a[4], "residual");
    if (rows.dim() != 2 || !rows.is_cuda() || !rows.is_contiguous()) refuse("rows must be a contiguous CUDA tensor [n, D]");
    if (weight.dim() < 1 || weight.size(-1) < 1) refuse("weight must be [..., top_k]");
    const at::Device device = rows.device();
    const int64_t D = rows.size(1), k = weight.size(-1);
    check_array(weight, weight.sizes(), at::kFloat, device, "weight");
    if (row_of.defined()) check_array(row_of, weight.sizes(), at::kInt, device, "row_of");
    if (gate.defined()) check_array(gate, weight.sizes(), at::kInt, device, "gate");
    const auto shape = with_last(weight, D);
    if (residual.defined()) check_array(residual, shape, rows.scalar_type(), device, "residual");
    const int dtype = dtype_code(rows);
    const at::Tensor out = output(a[5], shape, rows.scalar_type(), device, "out");
    const On on(rows);
    check(infmoe_expert_combine_topk(weight.numel() / k, size32(k, "top_k"), size32(D, "D"), dtype, rows.data_ptr(), rows.size(0),
                                     (const float*)weight.data_ptr(), (const int32_t*)data(gate), (const int32_t*)data(row_of),
                                     data(residual), out.data_ptr(), on.stream));
    return wrap(out);
}

// (bytes of the set, a, b, scale, rank, x, y, plan buffer, plan tokens, plan adapters, out, status, scale's stream, plan's stream) -> out.  Where
// the weights lie is asked of the tensors at every call: a parameter's data may have been replaced since the set was made.
PyObject* apply_adapters(PyObject* const* args) {
    if (!PyBytes_Check(args[0]) || PyBytes_GET_SIZE(args[0]) != (Py_ssize_t)sizeof(infmoe_adapter_set)) refuse("not an adapter set");
    infmoe_adapter_set set;
    memcpy(&set, PyBytes_AS_STRING(args[0]), sizeof(set));
    const at::Tensor &a = tensor(args[1], "a"), &b = tensor(args[2], "b"), &x = tensor(args[5], "x"), &y = tensor(args[6], "y");
    const at::Tensor *scale = given(args[3], "scale"), *rank = given(args[4], "rank"), &plan = tensor(args[7], "plan");
    const long long tokens = PyLong_AsLongLong(args[8]), adapters = PyLong_AsLongLong(args[9]);
    if (PyErr_Occurred()) throw Refused{};
    const Rows rx = rows_of(x, set.d_in, "x"), ry = rows_of(y, set.d_out, "y");
    const at::Device device = a.device();
    const at::ScalarType type = set.dtype == INFMOE_F32 ? at::kFloat : set.dtype == INFMOE_F16 ? at::kHalf : at::kBFloat16;
    if (!a.is_cuda()) refuse("a must be a CUDA tensor");
    check_array(a, {set.adapter_count, set.rank, set.d_in}, type, device, "a");
    check_array(b, {set.adapter_count, set.d_out, set.rank}, type, device, "b");
    if (scale) check_array(*scale, {set.adapter_count}, at::kFloat, device, "scale");
    if (rank) check_array(*rank, {set.adapter_count}, at::kInt, device, "rank");
    set.d_a = a.data_ptr();
    set.d_b = b.data_ptr();
    set.d_scale = scale ? (const float*)scale->data_ptr() : nullptr;
    set.d_rank = rank ? (const int32_t*)rank->data_ptr() : nullptr;
    if (x.scalar_type() != type || y.scalar_type() != type || x.device() != device || y.device() != device)
        refuse("x and y must be %s tensors on %s, like the adapters", c10::toString(type), device.str().c_str());
    if (rx.count != ry.count || rx.count != tokens || adapters != set.adapter_count || plan.device() != device)
        refuse("x has %lld rows, y %lld; the plan is for %lld rows and %lld adapters on %s, the set has %d on %s", (long long)rx.count,
               (long long)ry.count, tokens, adapters, plan.device().str().c_str(), set.adapter_count, device.str().c_str());
    const at::Tensor status = optional(args[11], "status");
    if (status.defined()) check_array(status, {1}, at::kInt, device, "status");
    at::Tensor out;
    int64_t ldo = set.d_out;
    if (args[10] == Py_None) {
        out = at::detail::empty_cuda(y.sizes(), type, device, std::nullopt);
    } else {
        out = tensor(args[10], "out");
        ldo = rows_of(out, set.d_out, "out").ld;
        if (out.sizes() != y.sizes() || out.scalar_type() != type || out.device() != device) refuse("out must be a tensor like y");
    }
    const On on(x);
    size_t bytes = 0;
    check(infmoe_adapter_workspace_bytes(&set, rx.count, &bytes));
    const at::Tensor workspace = at::detail::empty_cuda({(int64_t)bytes}, at::kByte, device, std::nullopt);
    check(infmoe_adapter_apply(&set, rx.count, x.data_ptr(), rx.ld, y.data_ptr(), ry.ld, out.data_ptr(), ldo, plan.data_ptr(),
                               workspace.data_ptr(), bytes, (int32_t*)data(status), on.stream));
    if (scale) on.uses(*scale, args[12]);
    on.uses(plan, args[13]);
    return wrap(out);
}

PyMethodDef methods[] = {
    {"select_topk", (PyCFunction)(void (*)())Entry<select_topk>::call<6>, METH_FASTCALL, nullptr},
    {"scatter_topk", (PyCFunction)(void (*)())Entry<scatter_topk>::call<6>, METH_FASTCALL, nullptr},
    {"combine_topk", (PyCFunction)(void (*)())Entry<combine_topk>::call<6>, METH_FASTCALL, nullptr},
    {"apply_adapters", (PyCFunction)(void (*)())Entry<apply_adapters>::call<14>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
