// CPython module ksmm_amd._native: the host side of KSLinear(algo='kernel') as one call.
//
// A layer on a small batch is done on the GPU in 5 to 15 us; the same call through Python checks,
// ctypes structures and torch.empty() took 20 to 30 us of host time.  Here the checks, the
// descriptors, the output and workspace tensors and the launch cost about 3 us.  Nothing is
// remembered between calls: pointers, sizes and types are read from the tensors each time.
//
// Every entry returns None when it does not take a call (an unusual argument, an error of the
// library, no memory): the caller then goes through ksmm_amd/kernel.py, which raises what is wrong
// with it.  The GIL is released from the first allocation on: both that and a launch can wait.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/ksmm_hip.h"

namespace {

int code_of(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return KSMM_F32;
    case at::kHalf: return KSMM_F16;
    case at::kFloat8_e4m3fn: return KSMM_FP8_E4M3;
    default: return -1;
    }
}

// makes a device current for the life of the object
struct DeviceScope {
    c10::DeviceIndex before = -1;
    explicit DeviceScope(c10::DeviceIndex want)
    {
        const c10::DeviceIndex now = c10::hip::current_device();
        if (now != want) {
            before = now;
            c10::hip::set_device(want);
        }
    }
    ~DeviceScope()
    {
        if (before >= 0) c10::hip::set_device(before);
    }
};

struct WithoutGil {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

struct Layer {
    ksmm_factor_desc f[KSMM_MAX_FACTORS];
    int n = 0;
    int64_t in_size = 0, out_size = 0;
};

// factor tensors, patterns (4-tuples) and scales (floats), lists of them; scales may be null: 1 each
bool read_layer(PyObject *params, PyObject *patterns, PyObject *scales, const at::Device &dev, Layer *l)
{
    if (!PyList_Check(params) || !PyList_Check(patterns) || (scales && !PyList_Check(scales))) return false;
    const Py_ssize_t n = PyList_GET_SIZE(params);
    if (n < 1 || n > KSMM_MAX_FACTORS || PyList_GET_SIZE(patterns) != n || (scales && PyList_GET_SIZE(scales) != n)) return false;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *w = PyList_GET_ITEM(params, i), *p = PyList_GET_ITEM(patterns, i);
        if (!THPVariable_Check(w) || !PyTuple_Check(p) || PyTuple_GET_SIZE(p) != 4) return false;
        const at::Tensor &t = THPVariable_Unpack(w);
        int64_t v[4];
        for (int k = 0; k < 4; ++k) {
            v[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(p, k));
            if (v[k] < 1 || v[k] > 0x7fffffff) return false;
        }
        ksmm_factor_desc &f = l->f[i];
        f.a = (int)v[0];
        f.b = (int)v[1];
        f.c = (int)v[2];
        f.d = (int)v[3];
        f.w_dtype = code_of(t.scalar_type());
        const double s = scales ? PyFloat_AsDouble(PyList_GET_ITEM(scales, i)) : 1.0;
        if (s == -1.0 && PyErr_Occurred()) return false;
        f.scale = (float)s;
        if (f.w_dtype < 0 || t.device() != dev || !t.is_contiguous() || t.dim() != 2 || t.size(0) != v[0] * v[2] * v[3] ||
            t.size(1) != v[1])
            return false;
        f.w = t.const_data_ptr();
        if (i == 0) l->in_size = v[0] * v[2] * v[3];
        l->out_size = v[0] * v[1] * v[3];
    }
    l->n = (int)n;
    return true;
}

// Shape of the result of a layer on x (batch-size-last: features first): false when x does not fit.
bool result_shape(const at::Tensor &x, bool bs_last, const Layer &l, int64_t *batch, c10::SmallVector<int64_t, 6> *shape)
{
    if (x.dim() < 1 || !x.is_contiguous() || x.numel() == 0) return false;
    const int64_t axis = bs_last ? 0 : x.dim() - 1;
    if (x.size(axis) != l.in_size) return false;
    shape->assign(x.sizes().begin(), x.sizes().end());
    (*shape)[axis] = l.out_size;
    if (bs_last && x.dim() == 1) shape->resize(1);
    *batch = x.numel() / l.in_size;
    return true;
}

// bias (None or a tensor) and activation (None or "gelu"); false: leave the call to Python
bool read_epilogue(PyObject *bias, PyObject *act, const at::Device &dev, at::ScalarType out, int64_t out_size, ksmm_epilogue *ep)
{
    ep->bias = nullptr;
    ep->act = KSMM_ACT_NONE;
    if (bias != Py_None) {
        if (!THPVariable_Check(bias)) return false;
        const at::Tensor &t = THPVariable_Unpack(bias);
        if (t.device() != dev || t.scalar_type() != out || !t.is_contiguous() || t.numel() != out_size) return false;
        ep->bias = t.const_data_ptr();
    }
    if (act != Py_None) {
        if (!PyUnicode_Check(act) || PyUnicode_CompareWithASCIIString(act, "gelu") != 0) return false;
        ep->act = KSMM_ACT_GELU;
    }
    return true;
}

// The whole layer without gradients: y = act(scale K_n .. K_1 x + bias), or KSMM error < 0.  quantise:
// x goes through e4m3 codes and a scale that the call finds itself.
int forward(const at::Tensor &x, const Layer &l, int64_t batch, const c10::SmallVector<int64_t, 6> &shape, bool bs_last,
            bool fuse, bool quantise, const ksmm_epilogue &ep, at::ScalarType out_type, at::Tensor *y)
{
    const int xd = code_of(x.scalar_type()), yd = code_of(out_type);
    void *const stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    const ksmm_epilogue *const epilogue = ep.bias || ep.act ? &ep : nullptr;
    // chains of one launch need no workspace (1.7 us); they are of 16 x 16 blocks, or of two factors on small batches (asking
    // costs the others 0.4 us)
    if (fuse && !quantise && l.n > 1 && ((l.f[0].b == 16 && l.f[0].c == 16) || (l.n == 2 && l.f[0].d == 1 && batch <= 4096))) {
        at::Tensor out = at::empty(shape, x.options().dtype(out_type));
        const int rc = ksmm_chain_forward_fused(l.f, l.n, x.const_data_ptr(), out.mutable_data_ptr(), batch, xd, yd, bs_last, epilogue, stream);
        *y = std::move(out);
        if (rc != KSMM_ERR_BAD_ALGO) return rc;
    }
    const int64_t need = quantise ? ksmm_chain_quant_workspace(l.f, l.n, batch, xd, yd, bs_last)
                                  : ksmm_chain_workspace_layout(l.f, l.n, batch, xd, yd, bs_last);
    if (need < 0) return (int)need;
    if (!y->defined()) *y = at::empty(shape, x.options().dtype(out_type));
    at::Tensor ws;
    if (need > 0) ws = at::empty({need}, x.options().dtype(at::kByte));
    const auto run = quantise ? ksmm_chain_forward_quant : ksmm_chain_forward_ep;
    return run(l.f, l.n, x.const_data_ptr(), y->mutable_data_ptr(), need > 0 ? ws.mutable_data_ptr() : nullptr, need, batch, xd, yd,
               bs_last, fuse, epilogue, stream);
}

// infer(x, factors, patterns, bs_last, scales, fuse, bias, act, quantise) -> y or None
PyObject *py_infer(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "infer() takes 9 arguments");
        return nullptr;
    }
    try {
        if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
        const at::Tensor &x = THPVariable_Unpack(args[0]);
        if (!x.is_cuda()) Py_RETURN_NONE;
        const bool bs_last = PyObject_IsTrue(args[3]) == 1, fuse = PyObject_IsTrue(args[5]) == 1, quantise = PyObject_IsTrue(args[8]) == 1;
        Layer l;
        int64_t batch;
        c10::SmallVector<int64_t, 6> shape;
        ksmm_epilogue ep;
        const bool taken = read_layer(args[1], args[2], args[4], x.device(), &l) && result_shape(x, bs_last, l, &batch, &shape);
        if (taken && code_of(x.scalar_type()) >= 0) {
            bool fp8 = false;
            for (int i = 0; i < l.n; ++i) fp8 |= l.f[i].w_dtype == KSMM_FP8_E4M3;
            const at::ScalarType out = fp8 ? at::kHalf : x.scalar_type();
            if (read_epilogue(args[6], args[7], x.device(), out, l.out_size, &ep)) {
                at::Tensor y;
                int status;
                {
                    WithoutGil released;
                    DeviceScope scope(x.device().index());
                    status = forward(x, l, batch, shape, bs_last, fuse, quantise, ep, out, &y);
                }
                if (status == KSMM_OK) return THPVariable_Wrap(std::move(y));
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

bool trainable(at::ScalarType t) { return t == at::kFloat || t == at::kHalf; }

// every factor of type t and in line with its neighbours (a chain's own check comes too late for the intermediates' sizes)
bool of_type(const Layer &l, at::ScalarType t)
{
    for (int i = 0; i < l.n; ++i) {
        if (l.f[i].w_dtype != code_of(t)) return false;
        if (i > 0 && (int64_t)l.f[i].a * l.f[i].c * l.f[i].d != (int64_t)l.f[i - 1].a * l.f[i - 1].b * l.f[i - 1].d) return false;
    }
    return true;
}

PyObject *wrapped(const at::Tensor &t)
{
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// train_forward(x, factors, patterns, bs_last, bias, act) -> (y, what each factor but the first was applied to.., z) or
// None; z is what the activation was applied to (None without one).
PyObject *py_train_forward(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "train_forward() takes 6 arguments");
        return nullptr;
    }
    try {
        if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
        const at::Tensor &x = THPVariable_Unpack(args[0]);
        const bool bs_last = PyObject_IsTrue(args[3]) == 1;
        Layer l;
        int64_t batch;
        c10::SmallVector<int64_t, 6> shape;
        ksmm_epilogue ep;
        if (x.is_cuda() && x.dim() == 2 && trainable(x.scalar_type()) && read_layer(args[1], args[2], nullptr, x.device(), &l) &&
            of_type(l, x.scalar_type()) && result_shape(x, bs_last, l, &batch, &shape) &&
            read_epilogue(args[4], args[5], x.device(), x.scalar_type(), l.out_size, &ep)) {
            const int dt = code_of(x.scalar_type());
            at::Tensor out[KSMM_MAX_FACTORS], y;
            int status = KSMM_OK;
            {
                WithoutGil released;
                DeviceScope scope(x.device().index());
                void *const stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
                const ksmm_epilogue bias_only{ep.bias, KSMM_ACT_NONE};
                const void *in = x.const_data_ptr();
                for (int i = 0; i < l.n && status == KSMM_OK; ++i) {
                    const ksmm_factor_desc &f = l.f[i];
                    const int64_t size = (int64_t)f.a * f.b * f.d;
                    const int64_t need = ksmm_factor_workspace(batch, f.a, f.b, f.c, f.d, dt, dt, dt, bs_last);
                    if (need < 0) {
                        status = (int)need;
                        break;
                    }
                    out[i] = at::empty({bs_last ? size : batch, bs_last ? batch : size}, x.options());
                    at::Tensor ws;
                    if (need > 0) ws = at::empty({need}, x.options().dtype(at::kByte));
                    status = ksmm_factor_forward_ep(in, f.w, out[i].mutable_data_ptr(), batch, f.a, f.b, f.c, f.d, dt, dt, dt, bs_last, 1.f,
                                                    i + 1 == l.n && ep.bias ? &bias_only : nullptr,
                                                    need > 0 ? ws.mutable_data_ptr() : nullptr, need, stream);
                    in = out[i].const_data_ptr();
                }
                if (status == KSMM_OK) y = ep.act ? at::gelu(out[l.n - 1]) : out[l.n - 1];
            }
            if (status == KSMM_OK) {
                PyObject *r = PyTuple_New(l.n + 1);
                if (!r) return nullptr;
                PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(y));
                for (int i = 0; i + 1 < l.n; ++i) PyTuple_SET_ITEM(r, i + 1, THPVariable_Wrap(out[i]));
                PyTuple_SET_ITEM(r, l.n, wrapped(ep.act ? out[l.n - 1] : at::Tensor()));
                return r;
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// train_backward(grad, factors, patterns, inputs, z, bs_last, act, need_x, need_bias, need_factors) -> (grad_x, grad_bias, [grad_factors])
// or None; lists but for grad, z (None without an activation) and need_factors (a tuple).  What is not needed is None.
PyObject *py_train_backward(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 10) {
        PyErr_SetString(PyExc_TypeError, "train_backward() takes 10 arguments");
        return nullptr;
    }
    try {
        if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
        const at::Tensor &grad = THPVariable_Unpack(args[0]);
        const bool bs_last = PyObject_IsTrue(args[5]) == 1, need_x = PyObject_IsTrue(args[7]) == 1, need_bias = PyObject_IsTrue(args[8]) == 1;
        Layer l;
        ksmm_epilogue ep;
        bool taken = grad.is_cuda() && grad.dim() == 2 && grad.is_contiguous() && grad.numel() > 0 && trainable(grad.scalar_type()) &&
                     read_layer(args[1], args[2], nullptr, grad.device(), &l) && of_type(l, grad.scalar_type()) &&
                     read_epilogue(Py_None, args[6], grad.device(), grad.scalar_type(), l.out_size, &ep) &&
                     grad.size(bs_last ? 0 : 1) == l.out_size && PyList_Check(args[3]) && PyList_GET_SIZE(args[3]) == l.n &&
                     PyTuple_Check(args[9]) && PyTuple_GET_SIZE(args[9]) == l.n;
        const int64_t batch = taken ? grad.size(bs_last ? 1 : 0) : 0;
        const void *inputs[KSMM_MAX_FACTORS], *z = nullptr;
        bool need[KSMM_MAX_FACTORS];
        // a tensor of the pass: the gradient's type, as many features as factor i takes (i == n: as the layer gives)
        auto fits = [&](PyObject *o, int i, const void **p) {
            if (!THPVariable_Check(o)) return false;
            const at::Tensor &t = THPVariable_Unpack(o);
            const int64_t size = i == l.n ? l.out_size : (int64_t)l.f[i].a * l.f[i].c * l.f[i].d;
            *p = t.scalar_type() == grad.scalar_type() && t.device() == grad.device() && t.dim() == 2 && t.is_contiguous() &&
                         t.size(bs_last ? 0 : 1) == size && t.size(bs_last ? 1 : 0) == batch
                     ? t.const_data_ptr() : nullptr;
            return *p != nullptr;
        };
        for (int i = 0; taken && i < l.n; ++i) {
            need[i] = PyObject_IsTrue(PyTuple_GET_ITEM(args[9], i)) == 1;
            taken = fits(PyList_GET_ITEM(args[3], i), i, &inputs[i]);
        }
        if (taken && ep.act) taken = fits(args[4], l.n, &z);
        if (taken) {
            const int dt = code_of(grad.scalar_type());
            at::Tensor dx, dbias, dw[KSMM_MAX_FACTORS];
            int status;
            {
                WithoutGil released;
                DeviceScope scope(grad.device().index());
                const int64_t bytes = ksmm_layer_backward_workspace(l.f, l.n, batch, dt, bs_last, ep.act);
                status = bytes < 0 ? (int)bytes : KSMM_OK;
                if (status == KSMM_OK) {
                    const auto opts = grad.options();
                    void *to[KSMM_MAX_FACTORS];
                    if (need_x) dx = at::empty({bs_last ? l.in_size : batch, bs_last ? batch : l.in_size}, opts);
                    if (need_bias) dbias = bs_last ? at::empty({l.out_size, 1}, opts) : at::empty({l.out_size}, opts);
                    for (int i = 0; i < l.n; ++i) {
                        if (need[i]) dw[i] = at::empty({(int64_t)l.f[i].a * l.f[i].c * l.f[i].d, l.f[i].b}, opts);
                        to[i] = need[i] ? dw[i].mutable_data_ptr() : nullptr;
                    }
                    const at::Tensor ws = at::empty({bytes}, opts.dtype(at::kByte));
                    status = ksmm_layer_backward(l.f, l.n, inputs, z, grad.const_data_ptr(), need_x ? dx.mutable_data_ptr() : nullptr, to,
                                                 need_bias ? dbias.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), bytes, batch, dt,
                                                 bs_last, ep.act, c10::hip::getCurrentHIPStream(grad.device().index()).stream());
                }
            }
            if (status == KSMM_OK) {
                PyObject *ws = PyList_New(l.n);
                if (!ws) return nullptr;
                for (int i = 0; i < l.n; ++i) PyList_SET_ITEM(ws, i, wrapped(dw[i]));
                return Py_BuildValue("(NNN)", wrapped(dx), wrapped(dbias), ws);
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// ---- operators around a feed-forward block ------------------------------------------------------------------
// Their autograd nodes are C++ ones: a forward and a backward pass through Python ones took 175 us of host time, more
// than the kernels of 25088 rows.

namespace ag = torch::autograd;

// torch.jit.trace records what is called through the dispatcher: of these calls the allocations alone.  The Python functions are
// nodes of their own there.
bool traced() { return torch::jit::tracer::isTracing(); }
// a tensor argument, or none; false: neither
bool read_optional(PyObject *o, at::Tensor *t)
{
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    *t = THPVariable_Unpack(o);
    return t->defined();
}
bool like(const at::Tensor &t, const at::Tensor &of)
{
    return t.scalar_type() == of.scalar_type() && t.device() == of.device() && t.is_contiguous() && !t._fw_grad(0).defined();
}
const void *data_of(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out_of(const at::Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check_status(int status)
{
    TORCH_CHECK(status == KSMM_OK, "ksmm: ", ksmm_strerror(status), " (status ", status, ")");
}
// what a node returns, when its gradients are asked to be differentiated in their turn
ag::variable_list once(ag::variable_list &&grads, const char *name)
{
    if (!at::GradMode::is_enabled()) return std::move(grads);
    const auto error = std::make_shared<ag::DelayedError>(std::string(name) + ": its gradients cannot be differentiated again", (int64_t)grads.size());
    return (*error)(std::move(grads));
}

struct NormHow {
    double alpha, eps;
    int kind;
    bool bs_last;
    int64_t batch, features, groups;
};
ksmm_norm_desc norm_desc(const at::Tensor (&in)[6], const NormHow &how)
{
    return ksmm_norm_desc{data_of(in[0]), data_of(in[1]), data_of(in[2]), data_of(in[3]), data_of(in[4]), data_of(in[5]),
                          how.groups, (float)how.alpha, (float)how.eps, how.kind};
}

struct NormNode : ag::Node {
    ag::SavedVariable in[6], stats;  // x, residual, gate, post_weight, weight, bias
    NormHow how;
    int r_at, n_at;  // which of the node's outputs r and n are, -1: none
    std::string name() const override { return "ResidualNormBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);  // (another thread's pass may be reading them)
        for (auto &v : in) v.reset_data();
        stats.reset_data();
    }
    ag::variable_list apply(ag::variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        at::Tensor t[6], out[6];
        for (int i = 0; i < 6; ++i) t[i] = in[i].unpack();
        const at::Tensor s = stats.unpack();
        at::Tensor dr, dn;
        if (r_at >= 0 && grads[r_at].defined()) dr = grads[r_at].contiguous();
        if (n_at >= 0 && grads[n_at].defined()) dn = grads[n_at].contiguous();
        ag::variable_list result(6);
        if (!dr.defined() && !dn.defined()) return result;
        {
        at::NoGradGuard no_grad;
        DeviceScope scope(t[1].device().index());
        for (int i = 0; i < 6; ++i)
            if (t[i].defined() && task_should_compute_output(i)) out[i] = at::empty_like(t[i]);
        const int dt = code_of(t[1].scalar_type());
        const int64_t need = ksmm_residual_norm_backward_workspace(how.batch, how.features, how.groups, dt, how.bs_last);
        check_status(need < 0 ? (int)need : KSMM_OK);
        const at::Tensor ws = at::empty({need}, t[1].options().dtype(at::kByte));
        const ksmm_norm_desc d = norm_desc(t, how);
        check_status(ksmm_residual_norm_backward(&d, s.const_data_ptr<float>(), data_of(dr), data_of(dn), out_of(out[0]), out_of(out[1]), out_of(out[2]),
                                                 out_of(out[3]), out_of(out[4]), out_of(out[5]), ws.mutable_data_ptr(), need, how.batch, how.features, dt,
                                                 how.bs_last, stream_of(t[1])));
        }
        for (int i = 0; i < 6; ++i) result[i] = out[i];
        return once(std::move(result), "residual_norm");
    }
};

// residual_norm(x, residual, gate, post_weight, weight, bias, alpha, kind, eps, bs_last, need_norm) -> (r_out, n_out) or None
PyObject *py_residual_norm(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 11) {
        PyErr_SetString(PyExc_TypeError, "residual_norm() takes 11 arguments");
        return nullptr;
    }
    try {
        at::Tensor in[6];
        bool taken = !traced();
        for (int i = 0; i < 6 && taken; ++i) taken = read_optional(args[i], &in[i]);
        const at::Tensor &x = in[0], &res = in[1];
        NormHow how;
        how.alpha = PyFloat_AsDouble(args[6]);
        how.kind = PyUnicode_Check(args[7]) ? PyUnicode_CompareWithASCIIString(args[7], "rms") == 0     ? KSMM_NORM_RMS
                                              : PyUnicode_CompareWithASCIIString(args[7], "layer") == 0 ? KSMM_NORM_LAYER
                                                                                                         : -1
                                            : -1;
        how.eps = PyFloat_AsDouble(args[8]);
        how.bs_last = PyObject_IsTrue(args[9]) == 1;
        const bool need_norm = PyObject_IsTrue(args[10]) == 1;
        taken = taken && !PyErr_Occurred() && how.kind >= 0 && res.defined() && res.is_cuda() && trainable(res.scalar_type()) && res.dim() > 0 &&
                res.numel() > 0 && (x.defined() || (need_norm && !in[2].defined() && !in[3].defined()));
        if (taken) {
            how.features = res.size(how.bs_last ? 0 : res.dim() - 1);
            how.batch = res.numel() / how.features;
            how.groups = 1;
            for (int i = 0; i < 6 && taken; ++i) {
                if (!in[i].defined()) continue;
                taken = like(in[i], res);
                if (i == 0) taken = taken && x.sizes() == res.sizes();
                if (i >= 3) taken = taken && in[i].numel() == how.features;
                if (i == 2) {
                    how.groups = in[2].numel() / how.features;
                    taken = taken && in[2].dim() > 0 && in[2].size(in[2].dim() - 1) == how.features && how.groups > 0 && how.batch % how.groups == 0;
                }
            }
        }
        if (taken) {
            bool gradients = false;
            if (at::GradMode::is_enabled())
                for (const at::Tensor &t : in) gradients |= t.defined() && t.requires_grad();
            at::Tensor r, n, stats;
            int status;
            {
                WithoutGil released;
                DeviceScope scope(res.device().index());
                at::AutoDispatchBelowADInplaceOrView below;
                r = x.defined() ? at::empty_like(res) : res;
                if (need_norm) n = at::empty_like(res);
                if (gradients) stats = at::empty({4, how.batch}, res.options().dtype(at::kFloat));
                const ksmm_norm_desc d = norm_desc(in, how);
                const int dt = code_of(res.scalar_type());
                const int64_t need = ksmm_residual_norm_forward_workspace(how.batch, how.features, dt, how.bs_last);
                at::Tensor ws;
                if (need > 0) ws = at::empty({need}, res.options().dtype(at::kByte));
                status = need < 0 ? (int)need
                                  : ksmm_residual_norm_forward(&d, x.defined() ? out_of(r) : nullptr, out_of(n),
                                                               gradients ? stats.mutable_data_ptr<float>() : nullptr, out_of(ws), need, how.batch,
                                                               how.features, dt, how.bs_last, stream_of(res));
            }
            if (status == KSMM_OK) {
                if (gradients) {
                    std::shared_ptr<NormNode> node(new NormNode(), ag::deleteNode);
                    node->set_next_edges(ag::collect_next_edges(in[0], in[1], in[2], in[3], in[4], in[5]));
                    node->how = how;
                    for (int i = 0; i < 6; ++i) node->in[i] = ag::SavedVariable(in[i], false);
                    node->stats = ag::SavedVariable(stats, false);
                    node->r_at = x.defined() ? 0 : -1;
                    node->n_at = !need_norm ? -1 : x.defined() ? 1 : 0;
                    if (x.defined()) ag::set_history(r, node);
                    if (need_norm) ag::set_history(n, node);
                }
                return Py_BuildValue("(NN)", THPVariable_Wrap(r), wrapped(n));
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

struct GatedHow {
    int a, b, c, d, act;
    bool bs_last;
    int64_t batch;
};

struct GatedNode : ag::Node {
    ag::SavedVariable in[3];  // x, factor, bias
    GatedHow how;
    std::string name() const override { return "GatedLinearBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto &v : in) v.reset_data();
    }
    ag::variable_list apply(ag::variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        ag::variable_list result(3);
        if (!grads[0].defined()) return result;
        at::Tensor t[3], out[3];
        for (int i = 0; i < 3; ++i) t[i] = in[i].unpack();
        const at::Tensor dh = grads[0].contiguous();
        {
            at::NoGradGuard no_grad;
            DeviceScope scope(t[0].device().index());
            for (int i = 0; i < 3; ++i)
                if (t[i].defined() && task_should_compute_output(i)) out[i] = at::empty_like(t[i]);
            const int dt = code_of(t[0].scalar_type());
            const int64_t need = ksmm_gated_backward_workspace(how.batch, how.a, how.b, how.c, how.d, dt, how.bs_last);
            check_status(need < 0 ? (int)need : KSMM_OK);
            const at::Tensor ws = at::empty({need}, t[0].options().dtype(at::kByte));
            check_status(ksmm_gated_backward(data_of(dh), data_of(t[0]), data_of(t[1]), data_of(t[2]), out_of(out[0]), out_of(out[1]), out_of(out[2]),
                                             ws.mutable_data_ptr(), need, how.batch, how.a, how.b, how.c, how.d, dt, how.bs_last, how.act, stream_of(t[0])));
        }
        for (int i = 0; i < 3; ++i) result[i] = out[i];
        return once(std::move(result), "gated_linear");
    }
};

// gated_linear(x, factor, pattern, bias, act, bs_last) -> h or None
PyObject *py_gated_linear(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "gated_linear() takes 6 arguments");
        return nullptr;
    }
    try {
        at::Tensor x, w, bias;
        int64_t v[4] = {0, 0, 0, 0};
        bool taken = !traced() && THPVariable_Check(args[0]) && THPVariable_Check(args[1]) && read_optional(args[3], &bias) && PyTuple_Check(args[2]) && PyTuple_GET_SIZE(args[2]) == 4;
        GatedHow how;
        how.bs_last = PyObject_IsTrue(args[5]) == 1;
        how.act = args[4] == Py_None ? KSMM_ACT_NONE : -1;
        if (PyUnicode_Check(args[4]))
            how.act = PyUnicode_CompareWithASCIIString(args[4], "silu") == 0   ? KSMM_ACT_SILU
                      : PyUnicode_CompareWithASCIIString(args[4], "gelu") == 0 ? KSMM_ACT_GELU
                      : PyUnicode_CompareWithASCIIString(args[4], "none") == 0 ? KSMM_ACT_NONE
                                                                                : -1;
        for (int k = 0; k < 4 && taken; ++k) {
            v[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[2], k));
            taken = v[k] >= 1 && v[k] <= 0x3fffffff;
        }
        if (taken) {
            x = THPVariable_Unpack(args[0]);
            w = THPVariable_Unpack(args[1]);
            const int64_t in_size = v[0] * v[2] * v[3], out_size = v[0] * v[1] * v[3];
            taken = how.act >= 0 && x.is_cuda() && trainable(x.scalar_type()) && x.dim() > 0 && x.numel() > 0 && like(x, x) && like(w, x) && w.dim() == 2 &&
                    w.size(0) == in_size && w.size(1) == 2 * v[1] && x.size(how.bs_last ? 0 : x.dim() - 1) == in_size &&
                    (!bias.defined() || (like(bias, x) && bias.numel() == 2 * out_size));
            if (taken) {
                how.a = (int)v[0];
                how.b = (int)v[1];
                how.c = (int)v[2];
                how.d = (int)v[3];
                how.batch = x.numel() / in_size;
                c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
                shape[how.bs_last ? 0 : shape.size() - 1] = out_size;
                const bool gradients = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()));
                at::Tensor h;
                int status;
                {
                    WithoutGil released;
                    DeviceScope scope(x.device().index());
                    at::AutoDispatchBelowADInplaceOrView below;
                    h = at::empty(shape, x.options());
                    status = ksmm_gated_forward(data_of(x), data_of(w), data_of(bias), out_of(h), how.batch, how.a, how.b, how.c, how.d,
                                                code_of(x.scalar_type()), how.bs_last, how.act, stream_of(x));
                }
                if (status == KSMM_OK) {
                    if (gradients) {
                        std::shared_ptr<GatedNode> node(new GatedNode(), ag::deleteNode);
                        node->set_next_edges(ag::collect_next_edges(x, w, bias));
                        node->how = how;
                        node->in[0] = ag::SavedVariable(x, false);
                        node->in[1] = ag::SavedVariable(w, false);
                        node->in[2] = ag::SavedVariable(bias, false);
                        ag::set_history(h, node);
                    }
                    return THPVariable_Wrap(h);
                }
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"train_forward", (PyCFunction)(void (*)(void))py_train_forward, METH_FASTCALL, "one layer, its intermediates kept"},
    {"train_backward", (PyCFunction)(void (*)(void))py_train_backward, METH_FASTCALL, "gradients of one layer"},
    {"residual_norm", (PyCFunction)(void (*)(void))py_residual_norm, METH_FASTCALL, "gated residual addition between two norms"},
    {"gated_linear", (PyCFunction)(void (*)(void))py_gated_linear, METH_FASTCALL, "gated projection"},
    {"infer", (PyCFunction)(void (*)(void))py_infer, METH_FASTCALL, "one layer without gradients"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
