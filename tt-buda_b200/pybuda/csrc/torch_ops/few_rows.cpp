// pybuda._torch_ops: the few-row operators of include/buda_cuda.h on torch tensors.
//
// A decoding step calls these operators with a token or a few; the kernels take 2 to 20 us, and the same checks,
// allocations and C call written in Python and ctypes take 10 to 24.  Here a matvec takes 4.5 us of the host (3.5 into a tensor that
// is there; torch.add beside it takes 4.8), a layer with its three launches 13.  torch is used for what it is used for in cuda_ops.py:
// device memory, devices and streams.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>

#include "buda_cuda.h"

namespace {

struct Refused {};                       // a Python error has been set

PyObject *g_buda_error = nullptr;        // _cabi.BudaError

[[noreturn]] void refuse(const char *fmt, ...)
{
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    PyErr_SetString(PyExc_RuntimeError, msg);
    throw Refused();
}

void check(int rc)
{
    if (rc == BUDA_SUCCESS) return;
    char msg[512];
    buda_last_error(msg, sizeof msg);
    if (g_buda_error) {
        PyObject *args = Py_BuildValue("(is)", rc, msg);
        if (args) {
            PyErr_SetObject(g_buda_error, args);
            Py_DECREF(args);
        }
    } else {
        PyErr_Format(PyExc_RuntimeError, "status %d: %s", rc, msg);
    }
    throw Refused();
}

const at::Tensor &tensor(PyObject *o, const char *what, const char *name)
{
    if (!THPVariable_Check(o)) refuse("%s: %s must be a tensor", what, name);
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}

bool truth(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused();
    return v != 0;
}

bool dense_rows(const at::Tensor &t) { return t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1); }

void check_activations(const char *what, const at::Tensor &x)
{
    if (x.scalar_type() != at::kBFloat16 || !dense_rows(x)) refuse("%s: activations must be a bfloat16 matrix with dense rows", what);
}

void check_device(const char *what, const at::Tensor &x, const at::Tensor &other)
{
    if (!x.is_cuda() || other.device() != x.device()) refuse("%s: works on CUDA tensors of one device only (no CPU fallback)", what);
}

int64_t record_bytes(const char *what, int64_t df)
{
    if (df != BUDA_DF_Bfp8_b && df != BUDA_DF_Bfp4_b && df != BUDA_DF_Bfp2_b)
        refuse("%s: weights must be Bfp8_b, Bfp4_b or Bfp2_b, got data format %lld", what, (long long)df);
    return df == BUDA_DF_Bfp8_b ? 1088 : df == BUDA_DF_Bfp4_b ? 576 : 320;     // a tile record without header
}

int64_t tiles(int64_t n) { return (n + 31) / 32; }

void check_images(const char *what, const at::Tensor &x, const at::Tensor &images)
{
    check_device(what, x, images);
    if (images.scalar_type() != at::kByte || !images.is_contiguous()) refuse("%s: queue images are contiguous uint8 tensors", what);
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like)
{
    return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// `out` if it was given and fits, else a new tensor
at::Tensor output(const char *what, PyObject *out, const at::Tensor &x, int64_t rows, int64_t cols, at::ScalarType type)
{
    if (out == Py_None) return empty({rows, cols}, type, x);
    const at::Tensor &t = tensor(out, what, "out");
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || t.scalar_type() != type || t.device() != x.device() || !dense_rows(t))
        refuse("%s: out must be a %s [%lld, %lld] tensor with dense rows on the activations' device", what, c10::toString(type),
               (long long)rows, (long long)cols);
    return t;
}

PyObject *give(PyObject *out, at::Tensor &&t)
{
    if (out != Py_None) {
        Py_INCREF(out);
        return out;
    }
    return THPVariable_Wrap(std::move(t));
}

// Runs `call(stream)` on the current stream of x's device, with that device current and without the interpreter lock.
template <class F>
void launch(const at::Tensor &x, F call)
{
    const c10::cuda::CUDAGuard guard(x.device());
    void *stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call(stream);
    Py_END_ALLOW_THREADS
    check(rc);
}

template <class F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F body)
{
    try {
        if (got != want) refuse("takes %zd arguments", want);
        return body();
    } catch (const Refused &) {
    } catch (...) {                        // torch's own: memory that ran out is torch.OutOfMemoryError
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// a, w_image, n, w_df, out, out_dtype
PyObject *bfp_matvec(PyObject *, PyObject *const *p, Py_ssize_t np)
{
    return guarded(np, 6, [&]() {
        const char *what = "bfp_matvec";
        const int64_t df = integer(p[3]), n = integer(p[2]), record = record_bytes(what, df);
        const at::Tensor &a = tensor(p[0], what, "a"), &w = tensor(p[1], what, "w_image");
        check_activations(what, a);
        check_images(what, a, w);
        const int64_t m = a.size(0), k = a.size(1), need = tiles(k) * tiles(n) * record;
        if (n < 1) refuse("%s: %lld output columns", what, (long long)n);
        if (w.numel() < need) refuse("%s: the queue image holds %lld bytes, needs %lld", what, (long long)w.numel(), (long long)need);
        at::ScalarType type;
        if (p[4] != Py_None) {
            type = tensor(p[4], what, "out").scalar_type();
        } else {
            if (!THPDtype_Check(p[5])) refuse("%s: out_dtype must be a dtype", what);
            type = reinterpret_cast<THPDtype *>(p[5])->scalar_type;
        }
        if (type != at::kBFloat16 && type != at::kFloat) refuse("%s: the output is bfloat16 or float32", what);
        at::Tensor y = output(what, p[4], a, m, n, type);
        launch(a, [&](void *stream) {
            return buda_bfp_matvec(a.data_ptr(), m, k, a.stride(0), w.data_ptr(), n, (int)df, y.data_ptr(), y.stride(0),
                                   type == at::kFloat ? BUDA_DF_Float32 : BUDA_DF_Float16_b, stream);
        });
        return give(p[4], std::move(y));
    });
}

void check_router(const at::Tensor &x, const at::Tensor &w)
{
    check_activations("moe_route", x);
    check_device("moe_route", x, w);
    if ((w.scalar_type() != at::kBFloat16 && w.scalar_type() != at::kFloat) || !dense_rows(w) || w.size(1) != x.size(1))
        refuse("moe_route: router weights must be a bfloat16 or float32 [experts, %lld] matrix with dense rows", (long long)x.size(1));
}

int router_df(const at::Tensor &w) { return w.scalar_type() == at::kFloat ? BUDA_DF_Float32 : BUDA_DF_Float16_b; }

int64_t check_top(const char *what, int64_t top)
{
    if (top < 1 || top > BUDA_MAX_TOP) refuse("%s: %lld experts for a token, 1 to %d are supported", what, (long long)top, BUDA_MAX_TOP);
    return top;
}

// x, w_router, top, renormalize
PyObject *moe_route(PyObject *, PyObject *const *p, Py_ssize_t np)
{
    return guarded(np, 4, [&]() -> PyObject * {
        const at::Tensor &x = tensor(p[0], "moe_route", "x"), &w = tensor(p[1], "moe_route", "w_router");
        check_router(x, w);
        const int64_t t = x.size(0), top = check_top("moe_route", integer(p[2]));
        const bool renorm = truth(p[3]);
        at::Tensor weights = empty({t, top}, at::kFloat, x), ids = empty({t, top}, at::kInt, x);
        launch(x, [&](void *stream) {
            return buda_moe_route(x.data_ptr(), t, x.size(1), x.stride(0), w.data_ptr(), router_df(w), w.stride(0), w.size(0), (int)top, renorm,
                                  (float *)weights.data_ptr(), (int32_t *)ids.data_ptr(), stream);
        });
        PyObject *pair = PyTuple_New(2);
        if (!pair) throw Refused();
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(weights)));
        PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(ids)));
        return pair;
    });
}

struct Experts {
    at::Tensor gate, up, down;
    int64_t experts, inter, df;
    int act;
    const void *up_ptr() const { return up.defined() ? up.data_ptr() : nullptr; }
};

// p: gate, up, down, inter, w_df, activation
Experts experts_of(const at::Tensor &x, PyObject *const *p)
{
    const char *what = "moe_experts";
    Experts e;
    const char *act = PyUnicode_Check(p[5]) ? PyUnicode_AsUTF8(p[5]) : nullptr;
    if (act && !strcmp(act, "silu")) e.act = BUDA_ACT_SILU;
    else if (act && !strcmp(act, "gelu")) e.act = BUDA_ACT_GELU;
    else refuse("%s: activation must be 'gelu' or 'silu'", what);
    e.df = integer(p[4]);
    e.inter = integer(p[3]);
    const int64_t record = record_bytes(what, e.df);
    check_activations(what, x);
    const int64_t h = x.size(1);
    if (h < 1 || e.inter < 1) refuse("%s: hidden size %lld, intermediate size %lld", what, (long long)h, (long long)e.inter);
    const int64_t need = tiles(h) * tiles(e.inter) * record;
    e.gate = tensor(p[0], what, "gate");
    if (p[1] != Py_None) e.up = tensor(p[1], what, "up");
    e.down = tensor(p[2], what, "down");
    e.experts = e.gate.dim() ? e.gate.size(0) : 0;
    for (const at::Tensor *images : {&e.gate, &e.up, &e.down}) {
        if (!images->defined()) continue;
        check_images(what, x, *images);
        if (images->dim() != 2 || images->size(0) != e.experts || images->size(1) != need)
            refuse("%s: the experts' images of matrices of %lld and %lld rows and columns are one [experts, %lld] tensor for each of gate, up "
                   "and down", what, (long long)h, (long long)e.inter, (long long)need);
    }
    return e;
}

at::Tensor workspace(const at::Tensor &x, int64_t top, int64_t inter, int64_t more)
{
    const int64_t bytes = buda_moe_workspace_bytes(x.size(0), (int)top, x.size(1), inter);
    if (bytes < 0) check(BUDA_RUNTIME_ERROR);
    return empty({bytes + more}, at::kByte, x);
}

// x, weights, ids, gate, up, down, inter, w_df, activation, out
PyObject *moe_experts(PyObject *, PyObject *const *p, Py_ssize_t np)
{
    return guarded(np, 10, [&]() {
        const char *what = "moe_experts";
        const at::Tensor &x = tensor(p[0], what, "x"), &weights = tensor(p[1], what, "weights"), &ids = tensor(p[2], what, "ids");
        const Experts e = experts_of(x, p + 3);
        const int64_t t = x.size(0);
        if (ids.scalar_type() != at::kInt || weights.scalar_type() != at::kFloat || ids.dim() != 2 || ids.size(0) != t ||
            ids.sizes() != weights.sizes() || !ids.is_contiguous() || !weights.is_contiguous() || ids.device() != x.device() ||
            weights.device() != x.device())
            refuse("%s: ids (int32) and weights (float32) are contiguous [%lld, top] tensors on the activations' device", what, (long long)t);
        const int64_t top = check_top(what, ids.size(1));
        at::Tensor y = output(what, p[9], x, t, x.size(1), at::kBFloat16), ws = workspace(x, top, e.inter, 0);
        launch(x, [&](void *stream) {
            return buda_moe_experts(x.data_ptr(), t, x.size(1), x.stride(0), (const float *)weights.data_ptr(), (const int32_t *)ids.data_ptr(),
                                    (int)top, e.gate.data_ptr(), e.up_ptr(), e.down.data_ptr(), e.experts, e.inter, (int)e.df, e.act,
                                    y.data_ptr(), y.stride(0), ws.data_ptr(), (uint64_t)ws.numel(), stream);
        });
        return give(p[9], std::move(y));
    });
}

// x, w_router, top, gate, up, down, inter, w_df, activation, renormalize, out
PyObject *moe_layer(PyObject *, PyObject *const *p, Py_ssize_t np)
{
    return guarded(np, 11, [&]() {
        const char *what = "moe_layer";
        const at::Tensor &x = tensor(p[0], what, "x"), &w = tensor(p[1], what, "w_router");
        check_router(x, w);
        const Experts e = experts_of(x, p + 3);
        if (w.size(0) != e.experts) refuse("%s: the router has %lld rows for %lld experts", what, (long long)w.size(0), (long long)e.experts);
        const int64_t t = x.size(0), top = check_top(what, integer(p[2]));
        const bool renorm = truth(p[9]);
        at::Tensor y = output(what, p[10], x, t, x.size(1), at::kBFloat16), ws = workspace(x, top, e.inter, 8 * t * top);
        const int64_t bytes = ws.numel() - 8 * t * top;                  // behind it the choice: weights, ids
        uint8_t *choice = (uint8_t *)ws.data_ptr() + bytes;
        launch(x, [&](void *stream) {
            return buda_moe_layer(x.data_ptr(), t, x.size(1), x.stride(0), w.data_ptr(), router_df(w), w.stride(0), (int)top, renorm,
                                  e.gate.data_ptr(), e.up_ptr(), e.down.data_ptr(), e.experts, e.inter, (int)e.df, e.act, (float *)choice,
                                  (int32_t *)(choice + 4 * t * top), y.data_ptr(), y.stride(0), ws.data_ptr(), (uint64_t)bytes, stream);
        });
        return give(p[10], std::move(y));
    });
}

PyObject *set_error(PyObject *, PyObject *cls)
{
    Py_INCREF(cls);
    Py_XDECREF(g_buda_error);
    g_buda_error = cls;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(bfp_matvec), FAST(moe_route), FAST(moe_experts), FAST(moe_layer),
                           {"set_error", set_error, METH_O, "the exception class for refused C calls: error(code, text)"},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_ops", "few-row operators on torch tensors", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__torch_ops() { return PyModule_Create(&g_module); }
