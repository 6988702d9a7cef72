// The ordinary call of the 8-bit products and of drawing tokens, from Python to
// the C ABI without a way through Python: shapes, types and devices looked at,
// outputs and workspace taken from torch's caching allocator, one C call on the
// current stream.  A decoding step makes several of these calls a token, each
// shorter than its checks in Python.
//
// Each function returns None for whatever is not ordinary or is refused: kernels.py
// then takes its own way, which says what is wrong.  Nothing is kept between calls.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "soraku_b200.h"

namespace {

decltype(&skb_quantize_rows) quantize_rows;
decltype(&skb_int8_workspace) int8_workspace;
decltype(&skb_int8_linear) int8_linear;
decltype(&skb_int8_swiglu) int8_swiglu;
decltype(&skb_sample_tokens) sample_tokens;

int type_of(at::ScalarType t) {
    return t == at::kFloat ? SKB_F32 : t == at::kBFloat16 ? SKB_BF16 : t == at::kHalf ? SKB_F16 : t == at::kChar ? SKB_I8 : -1;
}
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// The device of a CUDA tensor, where it is the current one.
bool device_of(const at::Tensor* t, int* device) {
    return t && t->is_cuda() && (*device = t->get_device()) == c10::cuda::current_device();
}

// Rows [n, k] that are contiguous and apart.
struct Rows {
    int64_t n = 0, k = 0, ld = 0;
    int type = -1;
    void* data = nullptr;
    bool read(const at::Tensor* t, int device) {
        if (!t || t->dim() != 2 || !t->is_cuda() || t->get_device() != device) return false;
        n = t->size(0), k = t->size(1);
        if (n < 1 || k < 2 || t->stride(1) != 1 || (n > 1 && t->stride(0) < k) || n > (1 << 30) || k > (1 << 30)) return false;
        ld = n > 1 ? t->stride(0) : (k + 15) & ~int64_t(15);
        type = type_of(t->scalar_type());
        data = t->data_ptr();
        return type >= 0;
    }
};
// A contiguous vector [n].
bool vector(PyObject* o, int device, int64_t n, at::ScalarType type, void** p) {
    const at::Tensor* t = tensor(o);
    if (!t || t->dim() != 1 || !t->is_cuda() || t->get_device() != device || t->size(0) != n || t->scalar_type() != type ||
        !t->is_contiguous())
        return false;
    *p = t->data_ptr();
    return true;
}
bool optional_vector(PyObject* o, int device, int64_t n, at::ScalarType type, void** p) {
    *p = nullptr;
    return o == Py_None || vector(o, device, n, type, p);
}
// Other Python threads run while outputs are taken and kernels launched: a launch waits
// where a stream has as many before it as its queue holds, as long as they take.  No
// Python object is touched meanwhile.
struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
};
// 8-bit rows and their scales.
struct Codes {
    Rows q;
    void* scale = nullptr;
    bool read(PyObject* o, int device) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
        return q.read(tensor(PyTuple_GET_ITEM(o, 0)), device) && q.type == SKB_I8 &&
               vector(PyTuple_GET_ITEM(o, 1), device, q.n, at::kFloat, &scale);
    }
};
bool number(PyObject* o, float* f) {
    const double d = PyFloat_CheckExact(o) ? PyFloat_AS_DOUBLE(o) : PyLong_CheckExact(o) ? PyLong_AsDouble(o) : NAN;
    if (PyErr_Occurred()) PyErr_Clear();
    *f = (float)d;
    return d == d;
}

// (x, weight, up or None, norm_weight, eps, bias, residual, out_dtype, out)
PyObject* product(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    if (n_args != 9 ||
        !device_of(PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == 2 ? tensor(PyTuple_GET_ITEM(a[0], 0)) : tensor(a[0]), &device))
        Py_RETURN_NONE;
    const bool glu = a[2] != Py_None;
    Rows x;
    Codes xc, w, up;
    void *norm, *bias = nullptr;
    float eps;
    at::ScalarType type = at::kFloat;
    if (const at::Tensor* t = tensor(a[0])) {
        if (!x.read(t, device) || x.type == SKB_I8) Py_RETURN_NONE;
        type = t->scalar_type();
    } else {
        if (!xc.read(a[0], device) || a[3] != Py_None) Py_RETURN_NONE;
        x = xc.q;
    }
    if (!w.read(a[1], device) || w.q.k != x.k || (glu && (!up.read(a[2], device) || up.q.k != x.k || up.q.n != w.q.n)) ||
        !optional_vector(a[3], device, x.k, at::kFloat, &norm) || !number(a[4], &eps) ||
        !optional_vector(a[5], device, w.q.n, at::kFloat, &bias))
        Py_RETURN_NONE;
    const at::Tensor* out_given = a[8] == Py_None ? nullptr : tensor(a[8]);
    if (a[8] != Py_None) {
        if (!out_given) Py_RETURN_NONE;
        type = out_given->scalar_type();
    }
    if (a[7] != Py_None) {
        if (!THPDtype_Check(a[7])) Py_RETURN_NONE;
        const at::ScalarType asked = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
        if (out_given && asked != type) Py_RETURN_NONE;
        type = asked;
    }
    const int out_type = type_of(type);
    if (out_type < 0 || out_type == SKB_I8) Py_RETURN_NONE;
    Rows residual, o;
    if (a[6] != Py_None && (!residual.read(tensor(a[6]), device) || residual.type != out_type || residual.n != x.n || residual.k != w.q.n))
        Py_RETURN_NONE;
    if (w.q.n < 2) Py_RETURN_NONE;
    const at::TensorOptions on = at::TensorOptions().device(at::kCUDA, device);
    at::Tensor out;
    if (out_given) out = *out_given;
    int status = SKB_ERR_ARG;
    {
        const Released released;
        if (!out_given) out = at::empty({x.n, w.q.n}, on.dtype(type));
        if (o.read(&out, device) && o.n == x.n && o.k == w.q.n) {
            const int64_t need = int8_workspace((int)x.n, (int)x.k, x.type);
            at::Tensor work;
            if (need > 0) work = at::empty({need}, on.dtype(at::kByte));
            void* space = need > 0 ? work.data_ptr() : nullptr;
            const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
            const float *xs = static_cast<const float*>(xc.scale), *nw = static_cast<const float*>(norm);
            status = glu ? int8_swiglu(x.data, x.type, x.ld, xs, nw, eps, (int)x.n, (int)x.k, static_cast<const int8_t*>(w.q.data),
                                       w.q.ld, static_cast<const float*>(w.scale), static_cast<const int8_t*>(up.q.data), up.q.ld,
                                       static_cast<const float*>(up.scale), (int)w.q.n, o.data, out_type, o.ld, space, need, stream)
                         : int8_linear(x.data, x.type, x.ld, xs, nw, eps, (int)x.n, (int)x.k, static_cast<const int8_t*>(w.q.data),
                                       w.q.ld, static_cast<const float*>(w.scale), (int)w.q.n, static_cast<const float*>(bias),
                                       residual.data, residual.ld, o.data, out_type, o.ld, space, need, stream);
        }
    }
    if (status != SKB_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// (x, norm_weight, eps) to (q, scale)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    Rows x;
    void* norm;
    float eps;
    if (n_args != 3 || !device_of(tensor(a[0]), &device) || !x.read(tensor(a[0]), device) || x.type == SKB_I8 || x.k % 16 != 0 ||
        !optional_vector(a[1], device, x.k, at::kFloat, &norm) || !number(a[2], &eps))
        Py_RETURN_NONE;
    const at::TensorOptions on = at::TensorOptions().device(at::kCUDA, device);
    at::Tensor q, scale;
    int status;
    {
        const Released released;
        q = at::empty({x.n, x.k}, on.dtype(at::kChar)), scale = at::empty({x.n}, on.dtype(at::kFloat));
        status = quantize_rows(x.data, x.type, x.ld, (int)x.n, (int)x.k, static_cast<const float*>(norm), eps, q.data_ptr<int8_t>(),
                               x.k, scale.data_ptr<float>(), c10::cuda::getCurrentCUDAStream(device).stream());
    }
    if (status != SKB_OK) Py_RETURN_NONE;
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(q)).get(), THPObjectPtr(THPVariable_Wrap(scale)).get());
    END_HANDLE_TH_ERRORS
}

// (logits, uniform, temperature, top_k, top_p, min_p) to (tokens, logprob)
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    Rows x;
    void *u, *each[4] = {};
    float value[4] = {};
    int top_k = 0;
    if (n_args != 6 || !device_of(tensor(a[0]), &device) || !x.read(tensor(a[0]), device) || x.type == SKB_I8 ||
        !vector(a[1], device, x.n, at::kFloat, &u))
        Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i) {
        PyObject* o = a[2 + i];
        if (THPVariable_Check(o)) {
            if (!vector(o, device, x.n, i == 1 ? at::kInt : at::kFloat, &each[i])) Py_RETURN_NONE;
        } else if (i == 1) {
            if (!PyLong_CheckExact(o)) Py_RETURN_NONE;
            int over = 0;
            const long k = PyLong_AsLongAndOverflow(o, &over);
            if (over || k > INT32_MAX || k < -INT32_MAX) Py_RETURN_NONE;
            top_k = (int)k;
        } else if (!number(o, &value[i])) {
            Py_RETURN_NONE;
        }
    }
    const at::TensorOptions on = at::TensorOptions().device(at::kCUDA, device);
    at::Tensor tokens, logprob;
    int status;
    {
        const Released released;
        tokens = at::empty({x.n}, on.dtype(at::kLong)), logprob = at::empty({x.n}, on.dtype(at::kFloat));
        status = sample_tokens(x.data, x.type, x.ld, (int)x.n, (int)x.k, static_cast<const float*>(u), static_cast<const float*>(each[0]),
                               value[0], static_cast<const int32_t*>(each[1]), top_k, static_cast<const float*>(each[2]), value[2],
                               static_cast<const float*>(each[3]), value[3], tokens.data_ptr<int64_t>(), logprob.data_ptr<float>(),
                               c10::cuda::getCurrentCUDAStream(device).stream());
    }
    if (status != SKB_OK) Py_RETURN_NONE;
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(tokens)).get(), THPObjectPtr(THPVariable_Wrap(logprob)).get());
    END_HANDLE_TH_ERRORS
}

// Addresses of the C functions, in the order of the pointers above.
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    void* p[5];
    if (n_args != 5) {
        PyErr_SetString(PyExc_TypeError, "connect: five addresses expected");
        return nullptr;
    }
    for (int i = 0; i < 5; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "connect: null address");
            return nullptr;
        }
    }
    quantize_rows = reinterpret_cast<decltype(quantize_rows)>(p[0]);
    int8_workspace = reinterpret_cast<decltype(int8_workspace)>(p[1]);
    int8_linear = reinterpret_cast<decltype(int8_linear)>(p[2]);
    int8_swiglu = reinterpret_cast<decltype(int8_swiglu)>(p[3]);
    sample_tokens = reinterpret_cast<decltype(sample_tokens)>(p[4]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"connect", (PyCFunction)(void*)connect, METH_FASTCALL, nullptr},
                         {"product", (PyCFunction)(void*)product, METH_FASTCALL, nullptr},
                         {"quantize", (PyCFunction)(void*)quantize, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void*)sample, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", SKB_BIND_KEY) < 0) Py_CLEAR(m);
    return m;
}
