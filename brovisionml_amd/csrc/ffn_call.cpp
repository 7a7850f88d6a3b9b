// The usual call of a feed-forward operator from Python (brovisionml_amd/ffn.py):
// contiguous tensors of one type on the current device that autograd does not
// record, checked, given their outputs and launched in C.  Anything out of the ordinary returns None, and
// the Python function's own checks then take it or say what is wrong.  Against
// the same steps in Python, time per call: a product of one row, 5120 to 1280,
// 8.3-8.6 to 6.6-6.8 us; a norm of one row of 1280, 9.2-9.4 to 8.1-8.4 (both
// with residual and bias or weight, bfloat16; two runs).  What is left is the launch, 3 to 4 us, and
// the outputs' allocation, about 1 us each.
//
// Only the CPython API: tensors are asked through their Python methods, and
// torch's headers are not needed.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "bvml_ffn.h"

namespace {

// what setup() hands over, kept for the process
PyObject *g_f16, *g_bf16, *g_f32, *g_u8, *g_acts, *g_device, *g_stream, *g_recording;
// method and attribute names
PyObject *n_dtype, *n_device, *n_contiguous, *n_shape, *n_ptr, *n_empty, *n_grad;

struct Held {  // a reference that is given back
    PyObject* o;
    explicit Held(PyObject* p) : o(p) {}
    ~Held() { Py_XDECREF(o); }
    Held(const Held&) = delete;
    Held& operator=(const Held&) = delete;
};

// BVML_FFN_F32, F16 or BF16; -1: another
int type_of(PyObject* dtype) {
    return dtype == g_bf16  ? BVML_FFN_BF16
           : dtype == g_f16 ? BVML_FFN_F16
           : dtype == g_f32 ? BVML_FFN_F32
                            : -1;
}

// The output's type as asked for: not given, or x's, which it is by default.
bool default_type(PyObject* dtype, int x) { return dtype == Py_None || type_of(dtype) == x; }

constexpr int kMostDims = 8;

struct Tensor {
    int type = -1;  // as type_of
    long device = -1;
    bool contiguous = false, requires_grad = false;
    int dims = 0;
    Py_ssize_t shape[kMostDims];
    void* data = nullptr;

    // false: not a tensor of a known type and few dimensions (no error is left set)
    bool ask(PyObject* t) {
        if (read(t)) return true;
        PyErr_Clear();
        return false;
    }
    Py_ssize_t numel() const {
        Py_ssize_t n = 1;
        for (int i = 0; i < dims; ++i) n *= shape[i];
        return n;
    }

private:
    bool read(PyObject* t) {
        const Held dtype(PyObject_GetAttr(t, n_dtype));
        type = type_of(dtype.o);
        if (type < 0) return false;
        const Held dev(PyObject_CallMethodNoArgs(t, n_device));
        if (!dev.o) return false;
        device = PyLong_AsLong(dev.o);
        const Held whole(PyObject_CallMethodNoArgs(t, n_contiguous));
        contiguous = whole.o == Py_True;
        const Held sizes(PyObject_GetAttr(t, n_shape));
        if (!sizes.o || !PyTuple_Check(sizes.o) || PyTuple_GET_SIZE(sizes.o) > kMostDims)
            return false;
        dims = (int)PyTuple_GET_SIZE(sizes.o);
        for (int i = 0; i < dims; ++i)
            shape[i] = PyLong_AsSsize_t(PyTuple_GET_ITEM(sizes.o, i));
        const Held ptr(PyObject_CallMethodNoArgs(t, n_ptr));
        if (!ptr.o) return false;
        data = PyLong_AsVoidPtr(ptr.o);
        const Held grad(PyObject_GetAttr(t, n_grad));
        requires_grad = grad.o == Py_True;
        return !PyErr_Occurred();
    }
};

// Whether autograd is to record a call on tensors of which some require a
// gradient.
bool recorded(bool any) {
    if (!any) return false;
    const Held on(PyObject_CallNoArgs(g_recording));
    return on.o != Py_False;
}

// The current device is `index`, and its stream.
bool stream_of(long index, void** stream) {
    const Held now(PyObject_CallNoArgs(g_device));
    if (!now.o || PyLong_AsLong(now.o) != index) return false;
    const Held arg(PyLong_FromLong(index));
    const Held raw(PyObject_CallOneArg(g_stream, arg.o));
    if (!raw.o) return false;
    *stream = PyLong_AsVoidPtr(raw.o);
    return !PyErr_Occurred();
}

PyObject* unusual() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

PyObject* refused(const char* op, int status) {
    return PyErr_Format(PyExc_RuntimeError, "ffn ops: %s: %s (status %d)", op,
                        bvml_ffn_last_error(), status);
}

// the data pointer of a tensor this library has just made, nullptr with an error set
void* data_of(PyObject* t) {
    const Held ptr(PyObject_CallMethodNoArgs(t, n_ptr));
    return ptr.o ? PyLong_AsVoidPtr(ptr.o) : nullptr;
}

// product(x, w, bias, act, residual, gated, dtype): y, or None for an unusual call
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "product takes seven arguments");
        return nullptr;
    }
    const bool gated = args[5] == Py_True, has_bias = args[2] != Py_None;
    const bool has_residual = args[4] != Py_None;
    Tensor x, w, b, r;
    if (!x.ask(args[0]) || x.type == BVML_FFN_F32 || !x.contiguous || x.dims != 2 ||
        x.device < 0 || !default_type(args[6], x.type))
        return unusual();
    if (!w.ask(args[1]) || w.type != x.type || !w.contiguous || w.dims != 2 ||
        w.device != x.device || w.shape[1] != x.shape[1])
        return unusual();
    const Py_ssize_t M = x.shape[0], K = x.shape[1], R = w.shape[0], N = gated ? R / 2 : R;
    const Py_ssize_t most = 1 << 30;
    if (M < 1 || K < 1 || N < 1 || (gated && R % 2) || M > most || K > most || R > most)
        return unusual();
    if (has_bias && (!b.ask(args[2]) || b.type != x.type || b.device != x.device ||
                     !b.contiguous || b.numel() != R))
        return unusual();
    if (has_residual && (!r.ask(args[4]) || r.type != x.type || r.device != x.device ||
                         !r.contiguous || r.dims != 2 || r.shape[0] != M || r.shape[1] != N))
        return unusual();
    if (recorded(x.requires_grad || w.requires_grad || b.requires_grad || r.requires_grad))
        return unusual();
    PyObject* const code = PyDict_GetItemWithError(g_acts, args[3]);
    void* stream = nullptr;
    if (!code || !stream_of(x.device, &stream)) return unusual();
    const int act = (int)PyLong_AsLong(code);

    const Held shape(Py_BuildValue("(nn)", M, N));
    Held y(shape.o ? PyObject_CallMethodOneArg(args[0], n_empty, shape.o) : nullptr);
    if (!y.o) return nullptr;
    void* const yp = data_of(y.o);
    if (!yp) return nullptr;
    const int m = (int)M, c = (int)N, k = (int)K;
    const long long bytes = gated ? bvml_ffn_gated_workspace(m, c, k, x.type)
                                  : bvml_ffn_linear_workspace(m, c, k, x.type);
    Held space(nullptr);
    void* sp = nullptr;
    if (bytes > 0) {
        // (new_empty takes the size as a tuple and the type by keyword)
        const Held empty(PyObject_GetAttr(args[0], n_empty));
        const Held sizes(Py_BuildValue("((L))", bytes));
        const Held type(Py_BuildValue("{s:O}", "dtype", g_u8));
        if (!empty.o || !sizes.o || !type.o) return nullptr;
        space.o = PyObject_Call(empty.o, sizes.o, type.o);
        if (!space.o || !(sp = data_of(space.o))) return nullptr;
    }
    const int status =
        gated ? bvml_ffn_gated(x.data, K, w.data, K, b.data, nullptr, nullptr, m, c, k, x.type,
                               x.type, x.type, act, yp, N, nullptr, 0, sp, bytes, stream)
              : bvml_ffn_linear(x.data, K, w.data, K, b.data, nullptr, nullptr, r.data, N, m, c, k,
                                x.type, x.type, x.type, act, yp, N, nullptr, 0, sp, bytes, stream);
    if (status != BVML_FFN_OK) return refused(gated ? "gated" : "linear", status);
    Py_INCREF(y.o);
    return y.o;
}

// norm(x, residual, weight, eps, dtype): (y, stream), or None for an unusual call
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "norm takes five arguments");
        return nullptr;
    }
    Tensor x, r, w;
    if (!x.ask(args[0]) || !x.contiguous || x.dims < 1 || x.device < 0 ||
        !default_type(args[4], x.type))
        return unusual();
    if (!r.ask(args[1]) || r.type != x.type || !r.contiguous || r.device != x.device ||
        r.dims != x.dims)
        return unusual();
    for (int i = 0; i < x.dims; ++i)
        if (r.shape[i] != x.shape[i]) return unusual();
    const Py_ssize_t cols = x.shape[x.dims - 1], all = x.numel();
    if (!w.ask(args[2]) || w.type != x.type || !w.contiguous || w.device != x.device ||
        w.numel() != cols)
        return unusual();
    if (recorded(x.requires_grad || r.requires_grad || w.requires_grad)) return unusual();
    const double eps = PyFloat_AsDouble(args[3]);
    void* stream = nullptr;
    if (all < 1 || all / cols > (1 << 30) || cols > (1 << 30) || PyErr_Occurred() ||
        !stream_of(x.device, &stream))
        return unusual();
    const Held shape(PyObject_GetAttr(args[0], n_shape));
    if (!shape.o) return nullptr;
    const Held y(PyObject_CallMethodOneArg(args[0], n_empty, shape.o));
    const Held s(y.o ? PyObject_CallMethodOneArg(args[0], n_empty, shape.o) : nullptr);
    if (!s.o) return nullptr;
    void *const yp = data_of(y.o), *const sp = yp ? data_of(s.o) : nullptr;
    if (!sp) return nullptr;
    const int status = bvml_ffn_add_rms_norm(x.data, cols, r.data, cols, w.data, (int)(all / cols),
                                             (int)cols, eps, x.type, x.type, x.type, yp, cols, sp,
                                             cols, nullptr, nullptr, stream);
    if (status != BVML_FFN_OK) return refused("add_rms_norm", status);
    return PyTuple_Pack(2, y.o, s.o);
}

// setup(float16, bfloat16, float32, uint8, acts, current_device, raw_stream,
// is_grad_enabled)
PyObject* setup(PyObject*, PyObject* args) {
    PyObject* o[8];
    if (!PyArg_ParseTuple(args, "OOOOO!OOO", &o[0], &o[1], &o[2], &o[3], &PyDict_Type, &o[4], &o[5],
                          &o[6], &o[7]))
        return nullptr;
    PyObject** const to[8] = {&g_f16,  &g_bf16,   &g_f32,    &g_u8,
                              &g_acts, &g_device, &g_stream, &g_recording};
    for (int i = 0; i < 8; ++i) {
        Py_INCREF(o[i]);
        Py_XDECREF(*to[i]);
        *to[i] = o[i];
    }
    Py_RETURN_NONE;
}

// (METH_FASTCALL functions go through the table's one function type)
PyMethodDef g_methods[] = {
    {"product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product)), METH_FASTCALL,
     "product(x, w, bias, act, residual, gated, dtype): y, or None for an unusual call"},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm)), METH_FASTCALL,
     "norm(x, residual, weight, eps, dtype): (y, stream), or None for an unusual call"},
    {"setup", setup, METH_VARARGS,
     "setup(float16, bfloat16, float32, uint8, acts, current_device, raw_stream, is_grad_enabled)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ffn_call", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ffn_call(void) {
    struct {
        PyObject** to;
        const char* name;
    } const names[] = {{&n_dtype, "dtype"},       {&n_device, "get_device"},
                       {&n_contiguous, "is_contiguous"}, {&n_shape, "shape"},
                       {&n_ptr, "data_ptr"},      {&n_empty, "new_empty"},
                       {&n_grad, "requires_grad"}};
    for (const auto& n : names)
        if (!(*n.to = PyUnicode_InternFromString(n.name))) return nullptr;
    return PyModule_Create(&g_module);
}
