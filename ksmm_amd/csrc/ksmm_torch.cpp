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
#include <hip/hip_runtime_api.h>
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

// ---- microscaled 4-bit numbers --------------------------------------------------------------------------------

int64_t mx_blocks(int64_t c) { return (c + 31) / 32; }
// a tuple of n sizes from 1 on
bool read_sizes(PyObject *o, int n, int64_t *v)
{
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != n) return false;
    for (int k = 0; k < n; ++k) {
        v[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, k));
        if (v[k] < 1 || v[k] > 0x3fffffff) return false;
    }
    return true;
}
int read_act(PyObject *o)
{
    if (o == Py_None) return KSMM_ACT_NONE;
    if (!PyUnicode_Check(o)) return -1;
    return PyUnicode_CompareWithASCIIString(o, "silu") == 0   ? KSMM_ACT_SILU
           : PyUnicode_CompareWithASCIIString(o, "gelu") == 0 ? KSMM_ACT_GELU
           : PyUnicode_CompareWithASCIIString(o, "none") == 0 ? KSMM_ACT_NONE
                                                             : -1;
}
// codes and scales of `matrices` matrices of rows of c values; rows, or -1
int64_t operand_rows(const at::Tensor &codes, const at::Tensor &scales, int64_t matrices, int64_t c)
{
    const bool fits = codes.is_cuda() && codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.device() == scales.device() &&
                      codes.is_contiguous() && scales.is_contiguous() && codes.dim() == 3 && scales.dim() == 3 && codes.size(0) == matrices &&
                      scales.size(0) == matrices && codes.size(1) == scales.size(1) && codes.size(2) == 16 * mx_blocks(c) &&
                      scales.size(2) == mx_blocks(c) && ((uintptr_t)codes.const_data_ptr() & 15) == 0;
    return fits ? codes.size(1) : -1;
}

// mx_rows(codes, scales, matrices, c) -> rows of an operand, or None
PyObject *py_mx_rows(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args == 4 && THPVariable_Check(args[0]) && THPVariable_Check(args[1])) {
        const int64_t matrices = PyLong_AsLongLong(args[2]), c = PyLong_AsLongLong(args[3]);
        if (!PyErr_Occurred()) {
            const int64_t rows = operand_rows(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), matrices, c);
            if (rows >= 0) return PyLong_FromLongLong(rows);
        }
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

at::Tensor bytes_like(const at::Tensor &x, at::IntArrayRef shape) { return at::empty(shape, x.options().dtype(at::kByte)); }

// mx_quantize(x, (a, c, d), bs_last) -> (codes, scales) or None
PyObject *py_mx_quantize(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 3) {
        PyErr_SetString(PyExc_TypeError, "mx_quantize() takes 3 arguments");
        return nullptr;
    }
    try {
        int64_t v[3];
        if (!traced() && THPVariable_Check(args[0]) && read_sizes(args[1], 3, v)) {
            const at::Tensor &x = THPVariable_Unpack(args[0]);
            const bool bs_last = PyObject_IsTrue(args[2]) == 1;
            const int64_t features = v[0] * v[1] * v[2];
            if (x.is_cuda() && trainable(x.scalar_type()) && x.dim() > 0 && x.numel() > 0 && like(x, x) && x.size(bs_last ? 0 : x.dim() - 1) == features) {
                const int64_t rows = x.numel() / features;
                at::Tensor codes, scales;
                int status;
                {
                    WithoutGil released;
                    DeviceScope scope(x.device().index());
                    at::AutoDispatchBelowADInplaceOrView below;
                    codes = bytes_like(x, {v[0] * v[2], rows, 16 * mx_blocks(v[1])});
                    scales = bytes_like(x, {v[0] * v[2], rows, mx_blocks(v[1])});
                    status = ksmm_mx_quantize(data_of(x), out_of(codes), out_of(scales), rows, (int)v[0], (int)v[1], (int)v[2], code_of(x.scalar_type()),
                                              bs_last, stream_of(x));
                }
                if (status == KSMM_OK) return Py_BuildValue("(NN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales));
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// mx_dequantize(codes, scales, (a, c, d), shape, half, bs_last) -> values or None
PyObject *py_mx_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "mx_dequantize() takes 6 arguments");
        return nullptr;
    }
    try {
        int64_t v[3];
        if (!traced() && THPVariable_Check(args[0]) && THPVariable_Check(args[1]) && read_sizes(args[2], 3, v) && PyTuple_Check(args[3])) {
            const at::Tensor &codes = THPVariable_Unpack(args[0]), &scales = THPVariable_Unpack(args[1]);
            const bool half = PyObject_IsTrue(args[4]) == 1, bs_last = PyObject_IsTrue(args[5]) == 1;
            const int64_t rows = operand_rows(codes, scales, v[0] * v[2], v[1]);
            c10::SmallVector<int64_t, 6> shape;
            int64_t values = 1;
            for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[3]); ++i) {
                shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(args[3], i)));
                values *= shape.back();
            }
            if (rows > 0 && !PyErr_Occurred() && values == rows * v[0] * v[1] * v[2]) {
                at::Tensor x;
                int status;
                {
                    WithoutGil released;
                    DeviceScope scope(codes.device().index());
                    at::AutoDispatchBelowADInplaceOrView below;
                    x = at::empty(shape, codes.options().dtype(half ? at::kHalf : at::kFloat));
                    status = ksmm_mx_dequantize(data_of(codes), data_of(scales), out_of(x), rows, (int)v[0], (int)v[1], (int)v[2], half ? KSMM_F16 : KSMM_F32,
                                                bs_last, stream_of(codes));
                }
                if (status == KSMM_OK) return THPVariable_Wrap(x);
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

struct MxHow {
    int a, b, c, d, act, gated;
    bool bs_last, wide;  // wide: fp16 may not have the factor's values, gradients are computed in fp32
    int64_t batch;
    int rows() const { return gated ? 2 * b : b; }
};
int mx_forward(const void *x, const void *x_scales, const at::Tensor &w, const at::Tensor &w_scales, const at::Tensor &bias, at::Tensor &y, at::Tensor *codes,
               at::Tensor *scales, const MxHow &h, int act)
{
    const int dt = code_of(y.scalar_type());
    const int64_t need = x_scales ? 0 : ksmm_mx_forward_workspace(h.batch, h.a, h.b, h.c, h.d, dt, h.bs_last, h.gated);
    if (need < 0) return (int)need;
    at::Tensor ws;
    if (need > 0) ws = bytes_like(y, {need});
    return ksmm_mx_forward(x, x_scales, data_of(w), data_of(w_scales), data_of(bias), out_of(y), codes ? out_of(*codes) : nullptr,
                           scales ? out_of(*scales) : nullptr, out_of(ws), need, h.batch, h.a, h.b, h.c, h.d, dt, h.bs_last, act, h.gated, stream_of(y));
}

// A pass that is being captured is refused where it comes to a node of the default stream: a leaf that an eager graph outside still
// holds.  The engine would make the default stream wait for the captured one, which is an error where nothing catches it.
void refuse_outside(const ag::edge_list &edges, void *stream)
{
    for (const ag::Edge &e : edges) {
        const auto other = e.function ? e.function->stream() : c10::nullopt;
        if (!other || other->id() != 0 || !stream) continue;
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing((hipStream_t)stream, &status) != hipSuccess) status = hipStreamCaptureStatusNone;
        TORCH_CHECK(status == hipStreamCaptureStatusNone,
                    "mx_linear: a backward pass cannot be captured while a graph of the same leaves from outside the capture is alive; drop what holds it first");
    }
}

struct MxNode : ag::Node {
    ag::SavedVariable in[5];  // codes and scales of x and of the factor, bias
    MxHow how;
    c10::SmallVector<int64_t, 6> x_shape;
    std::string name() const override { return "MXLinearBackward"; }
    void layer_backward(const ksmm_factor_desc &f, const at::Tensor &x, const at::Tensor &z, const at::Tensor &dy, at::Tensor (&out)[3], int act, int dt, void *stream)
    {
        const int64_t need = ksmm_layer_backward_workspace(&f, 1, how.batch, dt, how.bs_last, act);
        check_status(need < 0 ? (int)need : KSMM_OK);
        const at::Tensor ws = bytes_like(dy, {need});
        const void *inputs[] = {data_of(x)};
        void *dw[] = {out_of(out[1])};
        check_status(ksmm_layer_backward(&f, 1, inputs, data_of(z), data_of(dy), out_of(out[0]), dw, out_of(out[2]), ws.mutable_data_ptr(), need, how.batch, dt,
                                         how.bs_last, act, stream));
    }
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
        at::Tensor t[5], out[3];
        for (int i = 0; i < 5; ++i) t[i] = in[i].unpack();
        const at::ScalarType type = grads[0].scalar_type(), held = how.wide ? at::kFloat : type;
        {
            at::NoGradGuard no_grad;
            DeviceScope scope(grads[0].device().index());
            void *const stream = stream_of(grads[0]);
            refuse_outside(next_edges(), stream);
            const at::Tensor dy = grads[0].to(held).contiguous();
            if (t[4].defined()) t[4] = t[4].to(held);
            const int dt = code_of(held);
            const int64_t features = (int64_t)how.a * how.c * how.d;
            at::Tensor x = at::empty(x_shape, dy.options()), w = at::empty({features, how.rows()}, dy.options());
            check_status(ksmm_mx_values(data_of(t[0]), data_of(t[1]), out_of(x), data_of(t[2]), data_of(t[3]), out_of(w), how.batch, how.rows(), how.a, how.c, how.d, dt,
                                        how.bs_last, stream));
            if (task_should_compute_output(0)) out[0] = at::empty(x_shape, dy.options());
            if (task_should_compute_output(1)) out[1] = at::empty_like(w);
            if (t[4].defined() && task_should_compute_output(2)) out[2] = at::empty_like(t[4]);
            // what the activation was applied to is computed again, with the gradients of it where there is a kernel for both
            const bool nothing = how.act == KSMM_ACT_NONE && !how.gated;
            auto slope = [&](void *dz) {
                return ksmm_mx_slope(data_of(t[0]), data_of(t[1]), data_of(t[2]), data_of(t[3]), data_of(t[4]), data_of(dy), dz, how.batch, how.a, how.b, how.c, how.d,
                                     dt, how.bs_last, how.act, how.gated, stream);
            };
            if (nothing || slope(nullptr) == KSMM_OK) {
                at::Tensor dz = dy;
                if (!nothing) {
                    dz = at::empty({how.batch * how.a * how.rows() * how.d}, dy.options());
                    check_status(slope(out_of(dz)));
                }
                const ksmm_factor_desc f{data_of(w), how.a, how.rows(), how.c, how.d, dt, 1.f};
                layer_backward(f, x, at::Tensor(), dz, out, KSMM_ACT_NONE, dt, stream);
            } else if (how.gated) {
                const int64_t need = ksmm_gated_backward_workspace(how.batch, how.a, how.b, how.c, how.d, dt, how.bs_last);
                check_status(need < 0 ? (int)need : KSMM_OK);
                const at::Tensor ws = bytes_like(dy, {need});
                check_status(ksmm_gated_backward(data_of(dy), data_of(x), data_of(w), data_of(t[4]), out_of(out[0]), out_of(out[1]), out_of(out[2]),
                                                 ws.mutable_data_ptr(), need, how.batch, how.a, how.b, how.c, how.d, dt, how.bs_last, how.act, stream));
            } else {
                at::Tensor z = at::empty_like(dy);
                // (in the tensors' type: z in 32 bits beside fp16 took a pass of (1,128,128,8), 25088 rows from 240 to 280 us, for gradients 2.93e-4
                // off instead of 2.99e-4)
                check_status(ksmm_mx_sums(data_of(t[0]), data_of(t[1]), data_of(t[2]), data_of(t[3]), data_of(t[4]), out_of(z), how.batch, how.a, how.b, how.c, how.d, dt,
                                          how.bs_last, stream));
                const ksmm_factor_desc f{data_of(w), how.a, how.b, how.c, how.d, dt, 1.f};
                layer_backward(f, x, z, dy, out, how.act, dt, stream);
            }
            for (int i = 0; i < 3; ++i)
                if (out[i].defined()) result[i] = out[i].to(type);
        }
        return once(std::move(result), "mx_linear");
    }
};

// mx_linear(x, factor, scales, pattern, gated, bias, act, bs_last, wide) -> y or None; scales None: a factor in kernel format, else its codes,
// with `wide` of values that fp16 may not have
PyObject *py_mx_linear(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 9) {
        PyErr_SetString(PyExc_TypeError, "mx_linear() takes 9 arguments");
        return nullptr;
    }
    try {
        at::Tensor w, w_scales, bias;
        int64_t v[4];
        MxHow h;
        h.gated = PyObject_IsTrue(args[4]) == 1;
        h.act = read_act(args[6]);
        h.bs_last = PyObject_IsTrue(args[7]) == 1;
        bool taken = !traced() && THPVariable_Check(args[0]) && read_optional(args[1], &w) && w.defined() && read_optional(args[2], &w_scales) &&
                     read_sizes(args[3], 4, v) && read_optional(args[5], &bias) && h.act >= 0 && (h.act != KSMM_ACT_SILU || h.gated);
        if (taken) {
            const at::Tensor &x = THPVariable_Unpack(args[0]);
            const int64_t features = v[0] * v[2] * v[3], rows = h.gated ? 2 * v[1] : v[1], out_features = v[0] * v[1] * v[3];
            const bool packed = w_scales.defined();
            taken = x.is_cuda() && trainable(x.scalar_type()) && x.dim() > 0 && x.numel() > 0 && like(x, x) && x.size(h.bs_last ? 0 : x.dim() - 1) == features &&
                    w.device() == x.device() && (!bias.defined() || (like(bias, x) && bias.numel() == v[0] * rows * v[3]));
            if (taken && packed) taken = operand_rows(w, w_scales, v[0] * v[3], v[2]) == rows;
            if (taken && !packed) taken = like(w, x) && w.dim() == 2 && w.size(0) == features && w.size(1) == rows;
            const bool gradients =
                taken && at::GradMode::is_enabled() && (x.requires_grad() || (!packed && w.requires_grad()) || (bias.defined() && bias.requires_grad()));
            if (taken) {
                h.a = (int)v[0];
                h.b = (int)v[1];
                h.c = (int)v[2];
                h.d = (int)v[3];
                h.batch = x.numel() / features;
                h.wide = PyObject_IsTrue(args[8]) == 1 && x.scalar_type() == at::kHalf;
                c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
                shape[h.bs_last ? 0 : shape.size() - 1] = out_features;
                at::Tensor y, codes, scales, x_codes, x_scales;
                int status = KSMM_OK;
                {
                    WithoutGil released;
                    DeviceScope scope(x.device().index());
                    at::AutoDispatchBelowADInplaceOrView below;
                    y = at::empty(shape, x.options());
                    const int64_t blocks = mx_blocks(v[2]);
                    if (packed) {
                        codes = w;
                        scales = w_scales;
                    } else {
                        codes = bytes_like(x, {v[0] * v[3], rows, 16 * blocks});
                        scales = bytes_like(x, {v[0] * v[3], rows, blocks});
                        status = ksmm_mx_quantize(data_of(w), out_of(codes), out_of(scales), rows, (int)(v[0] * v[3]), h.c, 1, code_of(x.scalar_type()), 1,
                                                  stream_of(x));
                    }
                    if (gradients) {
                        x_codes = bytes_like(x, {v[0] * v[3], h.batch, 16 * blocks});
                        x_scales = bytes_like(x, {v[0] * v[3], h.batch, blocks});
                    }
                    if (status == KSMM_OK)
                        status = mx_forward(data_of(x), nullptr, codes, scales, bias, y, gradients ? &x_codes : nullptr, gradients ? &x_scales : nullptr, h, h.act);
                }
                if (status == KSMM_OK) {
                    if (gradients) {
                        std::shared_ptr<MxNode> node(new MxNode(), ag::deleteNode);
                        node->set_next_edges(ag::collect_next_edges(x, packed ? at::Tensor() : w, bias));
                        node->how = h;
                        node->x_shape.assign(x.sizes().begin(), x.sizes().end());
                        const at::Tensor *const kept[] = {&x_codes, &x_scales, &codes, &scales, &bias};
                        for (int i = 0; i < 5; ++i) node->in[i] = ag::SavedVariable(*kept[i], false);
                        ag::set_history(y, node);
                    }
                    return THPVariable_Wrap(y);
                }
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// ---- AdamW ----------------------------------------------------------------------------------------------------

// tensors of a list or tuple; false: something else is among them
bool read_tensors(PyObject *o, Py_ssize_t n, std::vector<at::Tensor> *t)
{
    if (!(PyList_Check(o) || PyTuple_Check(o)) || PySequence_Fast_GET_SIZE(o) != n) return false;
    t->reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *item = PySequence_Fast_GET_ITEM(o, i);
        if (!THPVariable_Check(item)) return false;
        t->push_back(THPVariable_Unpack(item));
    }
    return true;
}
bool holds(const at::Tensor &t, int64_t n, at::ScalarType type, const at::Device &device)
{
    return t.scalar_type() == type && t.device() == device && t.numel() == n && t.is_contiguous() && !t._fw_grad(0).defined();
}
int64_t moment_scales(int64_t n) { return 2 * ((n + 31) / 32); }

// adamw_update(params, grads, exp_avgs, exp_avg_sqs, scales, masters, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed, follow)
// -> True, None, or the status of a launch that failed: tensors may have been updated by then, and the call is not to be made again
PyObject *py_adamw_update(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 15) {
        PyErr_SetString(PyExc_TypeError, "adamw_update() takes 15 arguments");
        return nullptr;
    }
    try {
        const bool small = args[4] != Py_None, master = args[5] != Py_None;
        std::vector<at::Tensor> p, g, m, v, s, w;
        const Py_ssize_t n = PyList_Check(args[0]) || PyTuple_Check(args[0]) ? PySequence_Fast_GET_SIZE(args[0]) : 0;
        bool taken = !traced() && n > 0 && read_tensors(args[0], n, &p) && read_tensors(args[1], n, &g) && read_tensors(args[2], n, &m) &&
                     read_tensors(args[3], n, &v) && (!small || read_tensors(args[4], n, &s)) && (!master || read_tensors(args[5], n, &w));
        ksmm_adamw_desc d{};
        at::Tensor step;
        if (taken) {
            if (THPVariable_Check(args[6])) {
                step = THPVariable_Unpack(args[6]);
                d.step = 1;
                taken = holds(step, 1, at::kLong, p[0].device());
                if (taken) d.device_step = step.const_data_ptr<int64_t>();
            } else {
                d.step = PyLong_AsLongLong(args[6]);
            }
            d.lr = PyFloat_AsDouble(args[7]);
            d.beta1 = PyFloat_AsDouble(args[8]);
            d.beta2 = PyFloat_AsDouble(args[9]);
            d.eps = PyFloat_AsDouble(args[10]);
            d.weight_decay = PyFloat_AsDouble(args[11]);
            d.grad_scale = PyFloat_AsDouble(args[12]);
            d.seed = (uint32_t)PyLong_AsUnsignedLongLongMask(args[13]);
            d.follow = PyObject_IsTrue(args[14]) == 1;
            d.bits = small ? 8 : 32;
            taken = taken && !PyErr_Occurred();
        }
        std::vector<ksmm_adamw_tensor> table(taken ? n : 0);
        if (taken) {
            const at::ScalarType type = p[0].scalar_type(), state = small ? at::kByte : at::kFloat;
            const at::Device device = p[0].device();
            taken = p[0].is_cuda() && trainable(type);
            for (Py_ssize_t i = 0; i < n && taken; ++i) {
                const int64_t k = p[i].numel();
                taken = holds(p[i], k, type, device) && holds(g[i], k, type, device) && holds(m[i], k, state, device) && holds(v[i], k, state, device) &&
                        (!small || holds(s[i], moment_scales(k), at::kByte, device)) && (!master || holds(w[i], k, at::kFloat, device));
                if (taken)
                    table[i] = ksmm_adamw_tensor{p[i].mutable_data_ptr(), g[i].const_data_ptr(), master ? (float *)w[i].mutable_data_ptr() : nullptr,
                                                 m[i].mutable_data_ptr(), v[i].mutable_data_ptr(), small ? s[i].mutable_data_ptr() : nullptr, k};
            }
        }
        if (taken) {
            int status;
            {
                WithoutGil released;
                DeviceScope scope(p[0].device().index());
                status = ksmm_adamw_update(&d, table.data(), (int)n, code_of(p[0].scalar_type()), stream_of(p[0]));
            }
            if (status == KSMM_OK || status == KSMM_ERR_LAUNCH) {
                for (const auto *list : {&p, &m, &v, &s, &w})
                    for (const at::Tensor &t : *list)
                        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
                if (status == KSMM_OK) Py_RETURN_TRUE;
                return PyLong_FromLong(status);
            }
        }
    } catch (const std::exception &) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// adamw_moments(exp_avgs, exp_avg_sqs, scales) -> (list, list) or None
PyObject *py_adamw_moments(PyObject *, PyObject *const *args, Py_ssize_t n_args)
{
    if (n_args != 3) {
        PyErr_SetString(PyExc_TypeError, "adamw_moments() takes 3 arguments");
        return nullptr;
    }
    try {
        std::vector<at::Tensor> m, v, s, out_m, out_v;
        const Py_ssize_t n = PyList_Check(args[0]) || PyTuple_Check(args[0]) ? PySequence_Fast_GET_SIZE(args[0]) : 0;
        bool taken = !traced() && n > 0 && read_tensors(args[0], n, &m) && read_tensors(args[1], n, &v) && read_tensors(args[2], n, &s) && m[0].is_cuda();
        for (Py_ssize_t i = 0; i < n && taken; ++i) {
            const int64_t k = m[i].numel();
            taken = holds(m[i], k, at::kByte, m[0].device()) && holds(v[i], k, at::kByte, m[0].device()) && holds(s[i], moment_scales(k), at::kByte, m[0].device());
        }
        if (taken) {
            int status;
            {
                WithoutGil released;
                DeviceScope scope(m[0].device().index());
                at::AutoDispatchBelowADInplaceOrView below;
                std::vector<ksmm_adamw_moment> table(n);
                // (one memory for all of them, each from 256 bytes on: an allocation each took 1 us)
                int64_t all = 0;
                for (const at::Tensor &t : m) all += 2 * ((t.numel() + 63) / 64 * 64);
                const at::Tensor memory = at::empty({all}, m[0].options().dtype(at::kFloat));
                int64_t at = 0;
                auto part = [&](const at::Tensor &shape) {
                    at::Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(memory.storage()), memory.key_set(), memory.dtype());
                    t.unsafeGetTensorImpl()->set_storage_offset(at);
                    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape.sizes());
                    at += (shape.numel() + 63) / 64 * 64;
                    return t;
                };
                for (Py_ssize_t i = 0; i < n; ++i) {
                    out_m.push_back(part(m[i]));
                    out_v.push_back(part(m[i]));
                    table[i] = ksmm_adamw_moment{m[i].const_data_ptr(), v[i].const_data_ptr(), s[i].const_data_ptr(), out_m[i].mutable_data_ptr<float>(),
                                                 out_v[i].mutable_data_ptr<float>(), m[i].numel()};
                }
                status = ksmm_adamw_moments(table.data(), (int)n, stream_of(m[0]));
            }
            if (status == KSMM_OK) {
                PyObject *lists[] = {PyList_New(n), PyList_New(n)};
                if (!lists[0] || !lists[1]) return nullptr;
                for (Py_ssize_t i = 0; i < n; ++i) {
                    PyList_SET_ITEM(lists[0], i, THPVariable_Wrap(out_m[i]));
                    PyList_SET_ITEM(lists[1], i, THPVariable_Wrap(out_v[i]));
                }
                return Py_BuildValue("(NN)", lists[0], lists[1]);
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
    {"mx_rows", (PyCFunction)(void (*)(void))py_mx_rows, METH_FASTCALL, "rows of a 4-bit operand"},
    {"mx_quantize", (PyCFunction)(void (*)(void))py_mx_quantize, METH_FASTCALL, "values as 4-bit numbers"},
    {"mx_dequantize", (PyCFunction)(void (*)(void))py_mx_dequantize, METH_FASTCALL, "what 4-bit numbers stand for"},
    {"mx_linear", (PyCFunction)(void (*)(void))py_mx_linear, METH_FASTCALL, "product of 4-bit numbers"},
    {"adamw_update", (PyCFunction)(void (*)(void))py_adamw_update, METH_FASTCALL, "AdamW over many tensors"},
    {"adamw_moments", (PyCFunction)(void (*)(void))py_adamw_moments, METH_FASTCALL, "what 8-bit moments stand for"},
    {"infer", (PyCFunction)(void (*)(void))py_infer, METH_FASTCALL, "one layer without gradients"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
