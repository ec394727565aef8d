// The device operators for leaf-wise linear models on torch tensors: checks,
// outputs, workspaces and streams around the C ABI of include/gbm_b200.h, as
// the functions of the extension module _torch_ops (bsscl_gbm_b200.linear
// documents them).  In C++ because the calls are short: in Python the
// same checks and allocations took 8 us of a call whose kernel takes 5.
#include <ATen/ATen.h>
#include <Python.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <sstream>
#include <stdexcept>
#include <string>

#include "../../include/gbm_b200.h"

namespace {

using at::Tensor;

// what Python raises as ValueError
struct Value : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <class... A> [[noreturn]] void refuse(const A &...a) {
    std::ostringstream s;
    (s << ... << a);
    throw Value(s.str());
}

std::string shape_of(const Tensor &a) {
    std::ostringstream s;
    s << '(';
    for (int64_t i = 0; i < a.dim(); i++) s << (i ? ", " : "") << a.size(i);
    s << (a.dim() == 1 ? ",)" : ")");
    return s.str();
}

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(name, " must be a CUDA tensor");
    return THPVariable_Unpack(o);
}

bool in_place(const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

// A 2-D bf16/f16 CUDA tensor whose rows are contiguous.
struct Matrix {
    int64_t rows, cols, ld;
    void *p;
    Matrix(const Tensor &a, const char *name, const Tensor *like) {
        if (!a.is_cuda()) refuse(name, " must be a CUDA tensor");
        const auto t = a.scalar_type();
        if (t != at::kBFloat16 && t != at::kHalf) refuse(name, " must be bfloat16 or float16, got ", t);
        if (a.dim() != 2) refuse(name, " must be 2-D, got shape ", shape_of(a));
        if (like && (t != like->scalar_type() || a.device() != like->device()))
            refuse(name, " must have the type and device of the other operands (", like->scalar_type(), ", ", like->device(), "), got ", t, ", ", a.device());
        rows = a.size(0);
        cols = a.size(1);
        ld = a.stride(0);
        if (cols == 0) refuse(name, " has no columns");
        if (a.stride(1) != 1 && cols > 1) refuse(name, ": the elements of a row must be contiguous");
        if (rows <= 1) ld = cols;
        if (ld < cols) refuse(name, ": rows overlap (strides ", ld, ", ", a.stride(1), ")");
        p = a.data_ptr();
    }
    bool ready() const { return in_place(p, ld); }
};

// An output that the caller gave shares no memory with what the call reads: its
// kernels read on while they write.  Rows of one stride may lie beside one
// another, as columns of one matrix do; other areas are taken from end to end.
struct Area {
    uintptr_t at, row, step;      // bytes of a row, and from row to row
    int64_t rows;
    Area(const Matrix &m) : at(reinterpret_cast<uintptr_t>(m.p)), row(m.cols * 2), step(m.ld * 2), rows(m.rows) {}
    Area(const Tensor &a) : at(reinterpret_cast<uintptr_t>(a.data_ptr())), row(a.nbytes()), step(row), rows(row > 0) {}
    Area(const void *p, int64_t bytes) : at(reinterpret_cast<uintptr_t>(p)), row(bytes), step(row), rows(bytes > 0) {}
    uintptr_t end() const { return at + (rows - 1) * step + row; }
    bool meets(const Area &o) const {
        if (!rows || !o.rows || end() <= o.at || o.end() <= at) return false;
        if (step != o.step) return true;
        const uintptr_t off = o.at >= at ? (o.at - at) % step : (step - (at - o.at) % step) % step;
        return off < row || off + o.row > step;
    }
};

void apart(const Area &out, const char *name, std::initializer_list<Area> read) {
    for (const Area &a : read)
        if (out.meets(a)) refuse(name, " overlaps a tensor that the call reads");
}

int32_t code(const Tensor &a) { return a.scalar_type() == at::kBFloat16 ? GBM_TYPE_BF16 : GBM_TYPE_F16; }

// A contiguous vector of n elements.
template <class T> T *vector(PyObject *o, const char *name, at::ScalarType type, int64_t n, const Tensor &like) {
    const bool is = THPVariable_Check(o);
    if (is) {
        const Tensor &a = THPVariable_Unpack(o);
        if (a.scalar_type() == type && a.dim() == 1 && a.size(0) == n && a.device() == like.device()) {
            if (n > 1 && a.stride(0) != 1) refuse(name, " must be contiguous");
            return static_cast<T *>(a.data_ptr());
        }
    }
    refuse(name, " must be a ", type, " tensor of shape (", n, ",) on ", like.device());
}

// Uninitialised, of the current stream's pool.
Tensor fresh(at::IntArrayRef shape, const Tensor &like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }

// One library call on the tensors' device and its current stream, with the
// workspace it needs (of the stream's pool, so that calls on two streams, and two
// captured graphs, never share one).
struct Call {
    c10::cuda::OptionalCUDAGuard guard;
    Tensor room;
    void *ws = nullptr;
    int64_t bytes;
    void *stream;
    char err[256] = "";
    Call(const Tensor &on, int64_t bytes_) : bytes(bytes_) {
        if (bytes < 0) refuse("a size is out of range");
        if (on.get_device() != c10::cuda::current_device()) guard.set_device(on.device());
        if (bytes) {
            room = fresh({bytes}, on, at::kByte);
            ws = room.data_ptr();
        }
        stream = c10::cuda::getCurrentCUDAStream(on.get_device()).stream();
    }
    void done(int rc) const {
        if (rc == GBM_OK) return;
        if (rc == GBM_ERR_ARG || rc == GBM_ERR_UNSUPPORTED) throw Value(err);
        throw std::runtime_error(err);
    }
};

PyObject *wrap(const Tensor &a) {
    if (!a.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(a);
}

PyObject *pair(const Tensor &a, const Tensor &b) {
    PyObject *x = wrap(a), *y = x ? wrap(b) : nullptr, *t = y ? PyTuple_New(2) : nullptr;
    if (!t) {
        Py_XDECREF(x);
        Py_XDECREF(y);
        return nullptr;
    }
    PyTuple_SET_ITEM(t, 0, x);
    PyTuple_SET_ITEM(t, 1, y);
    return t;
}

bool truth(PyObject *o) {
    const int is = PyObject_IsTrue(o);
    if (is < 0) throw python_error();      // an array of several values: Python's own error
    return is == 1;
}

// C++ exceptions end here; torch's own become what torch makes of them.
template <class F> PyObject *guarded(Py_ssize_t have, Py_ssize_t want, F f) {
    HANDLE_TH_ERRORS
    if (have != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd needed", have, want);
        return nullptr;
    }
    try {
        return f();
    } catch (const Value &e) {
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

struct Head {
    const Tensor &x, &w;
    Matrix a, b;
    int64_t n, d, v;
    int64_t *y;
    Head(PyObject *const *args) : x(tensor(args[0], "x")), w(tensor(args[1], "w")), a(x, "x", nullptr), b(w, "w", &x) {
        n = a.rows, d = a.cols, v = b.rows;
        if (d != b.cols) refuse("x has ", d, " columns and w ", b.cols);
        y = vector<int64_t>(args[2], "target", at::kLong, n, x);
    }
    int64_t bytes(int grad) const { return gbm_softmax_xent_workspace(n, d, v, grad, a.ready() && b.ready()); }
};

PyObject *softmax_xent(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded(nargs, 3, [&] {
        Head h(args);
        Call c(h.x, h.bytes(0));
        Tensor loss = fresh({h.n}, h.x, at::kFloat), lse = fresh({h.n}, h.x, at::kFloat);
        c.done(gbm_softmax_xent(h.a.p, h.a.ld, h.b.p, h.b.ld, code(h.x), h.n, h.d, h.v, h.y, static_cast<float *>(loss.data_ptr()),
                                static_cast<float *>(lse.data_ptr()), c.ws, c.bytes, c.stream, c.err, sizeof c.err));
        return pair(loss, lse);
    });
}

// (x, w, target, lse, grad_loss, want_dx, want_dw, dw_out)
PyObject *softmax_xent_grad(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&] {
        Head h(args);
        const float *lse = vector<float>(args[3], "lse", at::kFloat, h.n, h.x), *g = vector<float>(args[4], "grad_loss", at::kFloat, h.n, h.x);
        const bool want_dx = truth(args[5]), want_dw = truth(args[6]);
        if (!want_dx && !want_dw) refuse("neither dx nor dw is wanted");
        Tensor dx, dw;
        int64_t lddw = h.d;
        if (want_dw && args[7] != Py_None) {
            dw = tensor(args[7], "dw_out");
            const Matrix m(dw, "dw_out", &h.x);
            if (m.rows != h.v || m.cols != h.d) refuse("dw_out must have shape (", h.v, ", ", h.d, "), got ", shape_of(dw));
            apart(m, "dw_out", {h.a, h.b, {h.y, h.n * 8}, {lse, h.n * 4}, {g, h.n * 4}});
            lddw = m.ld;
        }
        Call c(h.x, h.bytes(1));
        if (want_dx) dx = fresh({h.n, h.d}, h.x, h.x.scalar_type());
        if (want_dw && !dw.defined()) dw = fresh({h.v, h.d}, h.x, h.x.scalar_type());
        if (h.n || want_dw)
            c.done(gbm_softmax_xent_grad(h.a.p, h.a.ld, h.b.p, h.b.ld, code(h.x), h.n, h.d, h.v, h.y, lse, g, want_dx && h.n ? dx.data_ptr() : nullptr, h.d,
                                         want_dw ? dw.data_ptr() : nullptr, lddw, c.ws, c.bytes, c.stream, c.err, sizeof c.err));
        return pair(dx, dw);
    });
}

struct Leaf {
    const Tensor &x;
    Matrix a;
    const Tensor &w;
    int64_t n, e, dout, din;
    int32_t *off;
    Leaf(PyObject *const *args) : x(tensor(args[0], "x")), a(x, "x", nullptr), w(tensor(args[1], "w")) {
        if (w.dim() != 3 || !w.is_contiguous() || w.numel() == 0) refuse("w must be a contiguous tensor [leaves, dout, din]");
        if (w.scalar_type() != x.scalar_type() || w.device() != x.device())
            refuse("w must have x's type and device (", x.scalar_type(), ", ", x.device(), "), got ", w.scalar_type(), ", ", w.device());
        n = a.rows, e = w.size(0), dout = w.size(1), din = w.size(2);
        if (a.cols != din) refuse("x must have ", din, " columns, got ", a.cols);
        if (e >= 65536) refuse("more than 65535 leaves");
        off = vector<int32_t>(args[2], "offsets", at::kInt, e + 1, x);
    }
};

// (x, w, offsets, out)
PyObject *leaf_linear(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded(nargs, 4, [&] {
        Leaf l(args);
        Tensor y;
        int64_t ldy = l.dout;
        const bool own = args[3] == Py_None;
        if (!own) {
            y = tensor(args[3], "out");
            const Matrix m(y, "out", &l.x);
            if (m.rows != l.n || m.cols != l.dout) refuse("out must have shape (", l.n, ", ", l.dout, "), got ", shape_of(y));
            apart(m, "out", {l.a, l.w, {l.off, (l.e + 1) * 4}});
            ldy = m.ld;
        }
        Call c(l.x, gbm_leaf_linear_workspace(l.n, (int32_t)l.e, l.din, l.dout, 0, l.a.ready() && in_place(l.w.data_ptr(), l.din)));
        if (own) y = fresh({l.n, l.dout}, l.x, l.x.scalar_type());
        if (l.n)
            c.done(gbm_leaf_linear(l.a.p, l.a.ld, l.w.data_ptr(), l.off, code(l.x), l.n, (int32_t)l.e, l.din, l.dout, y.data_ptr(), ldy, own, c.ws, c.bytes,
                                   c.stream, c.err, sizeof c.err));
        return wrap(y);
    });
}

// (x, w, offsets, dy, want_dx, want_dw, dw_out)
PyObject *leaf_linear_grad(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded(nargs, 7, [&] {
        Leaf l(args);
        const Matrix g(tensor(args[3], "dy"), "dy", &l.x);
        if (g.rows != l.n || g.cols != l.dout) refuse("dy must have shape (", l.n, ", ", l.dout, "), got (", g.rows, ", ", g.cols, ")");
        const bool want_dx = truth(args[4]), want_dw = truth(args[5]);
        if (!want_dx && !want_dw) refuse("neither dx nor dw is wanted");
        Tensor dx, dw;
        if (want_dw && args[6] != Py_None) {
            dw = tensor(args[6], "dw_out");
            if (dw.sizes() != l.w.sizes() || dw.scalar_type() != l.w.scalar_type() || dw.device() != l.w.device() || !dw.is_contiguous())
                refuse("dw_out must be contiguous and have w's shape, type and device");
            apart(dw, "dw_out", {l.a, l.w, g, {l.off, (l.e + 1) * 4}});
        }
        const bool ready = g.ready() && (!want_dw || l.a.ready()) && (!want_dx || in_place(l.w.data_ptr(), l.din));
        Call c(l.x, gbm_leaf_linear_workspace(l.n, (int32_t)l.e, l.din, l.dout, 1, ready));
        if (want_dx) dx = fresh({l.n, l.din}, l.x, l.x.scalar_type());
        if (want_dw && !dw.defined()) dw = fresh({l.e, l.dout, l.din}, l.x, l.x.scalar_type());
        if (l.n || want_dw)
            c.done(gbm_leaf_linear_grad(l.a.p, l.a.ld, l.w.data_ptr(), l.off, g.p, g.ld, code(l.x), l.n, (int32_t)l.e, l.din, l.dout,
                                        want_dx && l.n ? dx.data_ptr() : nullptr, l.din, 1, want_dw ? dw.data_ptr() : nullptr, c.ws, c.bytes, c.stream, c.err,
                                        sizeof c.err));
        return pair(dx, dw);
    });
}

// (plan's address on the host, plan on the device, max_norm)
PyObject *grad_clip(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded(nargs, 3, [&]() -> PyObject * {
        void *plan = PyLong_AsVoidPtr(args[0]);
        const Tensor &dev = tensor(args[1], "plan");
        const double most = PyFloat_AsDouble(args[2]);
        if (PyErr_Occurred()) return nullptr;
        Call c(dev, gbm_grad_clip_workspace(plan));
        // the plan's owner may let go of it while this stream still reads it
        c10::cuda::CUDACachingAllocator::recordStream(dev.storage().data_ptr(), c10::cuda::getCurrentCUDAStream(dev.get_device()));
        Tensor norm = fresh({}, dev, at::kFloat);
        c.done(gbm_grad_clip(plan, dev.data_ptr(), most, static_cast<float *>(norm.data_ptr()), c.ws, c.bytes, c.stream, c.err, sizeof c.err));
        return wrap(norm);
    });
}

#define FAST(f) #f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{FAST(softmax_xent)}, {FAST(softmax_xent_grad)}, {FAST(leaf_linear)}, {FAST(leaf_linear_grad)}, {FAST(grad_clip)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
