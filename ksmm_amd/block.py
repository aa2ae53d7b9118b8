"""What a feed-forward block of Kronecker-sparse layers needs around its products: the gated projection (two factors of
one pattern, the activation of one and the product in one kernel) and the norms around its residual connection, each
with its backward pass.  fp32 and fp16, both layouts, on the hand-written kernels of libksmm_hip.so.

    n1 = residual_norm(None, r, weight=w1)[1]               # the norm before the block
    h  = gated_linear(n1, factor, (a, b, c, d), act="silu") # act(G n1) * (U n1)
    y  = down(h)                                            # a KSLinear
    r, n2 = residual_norm(y, r, gate=g, weight=w2)          # the gated addition and the norm before the next block

``KSGatedLinear``, ``ResidualNorm`` and ``KSFeedForward`` are the modules.
"""
import ctypes
import math

import torch
from torch import nn

from . import _lib
from .kernel import _check_input, _stream_ptr, dtype_code
from .layer import KSLinear, generate_factor

GATED_ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}
NORMS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _written(*tensors):
    """Tells autograd that these were written: a kernel does not, and a graph that holds one of them must not run on."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _trainable_type(t, name):
    if t.dtype not in (torch.float32, torch.float16):
        raise AssertionError("Unsupported data type %s of %s: float32 and float16 are" % (t.dtype, name))


def _same(t, like, name):
    _check_input(t, name)
    if t.dtype != like.dtype or t.device != like.device:
        raise RuntimeError("%s must be %s on %s" % (name, like.dtype, like.device))


# -- gated projection --------------------------------------------------------------------------------


def _check_gated(x, factor, pattern, bias, act, bs_last):
    if act not in GATED_ACTS:
        raise ValueError("act must be one of %s" % sorted(k for k in GATED_ACTS if k))
    a, b, c, d = (int(v) for v in pattern)
    if min(a, b, c, d) < 1:
        raise ValueError("pattern must hold four sizes of one and more, not %s" % (pattern,))
    _check_input(x, "input")
    _trainable_type(x, "input")
    _same(factor, x, "factor")
    axis = 0 if bs_last else -1
    if x.dim() < 1 or x.size(axis) != a * c * d:
        raise ValueError("input must have %d features, not %s" % (a * c * d, tuple(x.shape)))
    if tuple(factor.shape) != (a * d * c, 2 * b):
        raise ValueError("factor must be %s (gate columns, then up columns), not %s" % ((a * d * c, 2 * b), tuple(factor.shape)))
    if bias is not None:
        _same(bias, x, "bias")
        if bias.numel() != 2 * a * b * d:
            raise ValueError("bias must hold %d values (gate, then up, of each a), not %d" % (2 * a * b * d, bias.numel()))
    return a, b, c, d


class GatedKernel:
    """Both directions of the gated projection as single calls on tensors, without autograd."""

    @staticmethod
    def forward(x, factor, pattern, bias=None, act="silu", bs_last=False, out=None):
        lib = _lib.load()
        bs_last = bool(bs_last)
        a, b, c, d = _check_gated(x, factor, pattern, bias, act, bs_last)
        batch = x.numel() // (a * c * d)
        shape = (a * b * d, *x.shape[1:]) if bs_last else (*x.shape[:-1], a * b * d)
        given = out is not None
        if not given:
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        elif tuple(out.shape) != tuple(shape) or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous %s of shape %s" % (x.dtype, tuple(shape)))
        if batch == 0:
            return out
        with torch.cuda.device(x.device):
            _lib.check(lib.ksmm_gated_forward(x.data_ptr(), factor.data_ptr(), _ptr(bias), out.data_ptr(), batch, a, b, c, d,
                                              dtype_code(x.dtype), int(bs_last), GATED_ACTS[act], _stream_ptr(x)))
        if given:
            _written(out)
        return out

    @staticmethod
    def backward(grad_output, x, factor, pattern, bias=None, act="silu", bs_last=False, need_input=True, need_weight=True,
                 need_bias=True, workspace=None):
        """(grad_input, grad_factor, grad_bias); None for what is not needed."""
        lib = _lib.load()
        bs_last = bool(bs_last)
        a, b, c, d = _check_gated(x, factor, pattern, bias, act, bs_last)
        _same(grad_output, x, "grad_output")
        batch = x.numel() // (a * c * d)
        if grad_output.numel() != batch * a * b * d or grad_output.size(0 if bs_last else -1) != a * b * d:
            raise ValueError("grad_output must have the result's shape, not %s" % (tuple(grad_output.shape),))
        dx = torch.empty_like(x) if need_input else None
        dw = torch.empty_like(factor) if need_weight else None
        dbias = torch.empty_like(bias) if need_bias and bias is not None else None
        if batch == 0:
            return dx, None if dw is None else dw.zero_(), None if dbias is None else dbias.zero_()
        dt = dtype_code(x.dtype)
        need = lib.ksmm_gated_backward_workspace(batch, a, b, c, d, dt, int(bs_last))
        if need < 0:
            _lib.check(int(need))
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.check(lib.ksmm_gated_backward(grad_output.data_ptr(), x.data_ptr(), factor.data_ptr(), _ptr(bias), _ptr(dx), _ptr(dw),
                                               _ptr(dbias), workspace.data_ptr(), workspace.numel() * workspace.element_size(), batch,
                                               a, b, c, d, dt, int(bs_last), GATED_ACTS[act], _stream_ptr(x)))
        return dx, dw, dbias


class KSGatedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, factor, bias, pattern, act, bs_last):
        ctx.save_for_backward(x, factor, bias)
        ctx.pattern, ctx.act, ctx.bs_last = pattern, act, bs_last
        return GatedKernel.forward(x, factor, pattern, bias, act, bs_last)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, factor, bias = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, dbias = GatedKernel.backward(grad.contiguous(), x, factor, ctx.pattern, bias, ctx.act, ctx.bs_last, need_x, need_w,
                                             need_b)
        return dx, dw, dbias, None, None, None


def gated_linear(x, factor, pattern, bias=None, act="silu", bs_last=False):
    """``act(G x + bias_g) * (U x + bias_u)`` in one kernel; G and U are factors of ``pattern`` (a, b, c, d).

    ``factor`` (a*d*c, 2*b) holds the kernel-format weights of both side by side, gate columns first
    (``pack_gated``); ``bias`` 2*a*b*d values, for each of the ``a`` groups those of the gate, then those of up.
    ``x`` has a*c*d features, in the last axis, or with ``bs_last`` in the first, like the result's a*b*d.
    ``act``: "silu", "gelu" (erf form) or None.  Gradients of all three go through one call that computes
    the projections again instead of keeping them; they cannot be differentiated a second time.  The gradients of the
    projections, which those three are sums of, are held in the tensors' type: in fp16 they are rounded once before the sums, and are
    infinities beyond 65504, as between two fp16 layers.  Who needs more than that passes fp32 tensors."""
    out = _lib.native().gated_linear(x, factor, pattern, bias, act, bs_last)
    if out is not None:
        return out
    if torch.jit.is_tracing() or (torch.is_grad_enabled() and (
            x.requires_grad or factor.requires_grad or (bias is not None and bias.requires_grad))):
        return KSGatedFunction.apply(x, factor, bias, tuple(pattern), act, bs_last)
    return GatedKernel.forward(x, factor, pattern, bias, act, bs_last)


def pack_gated(gate, up, dtype=torch.float16, device="cpu"):
    """(a*d*c, 2*b): the kernel-format weights of two (a, b, c, d) tensors side by side."""
    assert gate.shape == up.shape and gate.dim() == 4
    return torch.cat([generate_factor(*gate.shape, "kernel", w, dtype, device) for w in (gate, up)], dim=1).contiguous()


class KSGatedLinear(nn.Module):
    """``act(G x + bias) * (U x + bias)``: the gated counterpart of a one-factor ``KSLinear(algo='kernel')``.
    ``weights``: two (a, b, c, d) tensors, of the gate and of the other projection; drawn like KSLinear's if None."""

    def __init__(self, pattern, weights=None, bias=True, dtype=torch.float16, bs_last=False, device="cuda", act="silu"):
        super().__init__()
        if act not in GATED_ACTS:
            raise ValueError("act must be one of %s" % sorted(k for k in GATED_ACTS if k))
        if dtype not in (torch.float32, torch.float16):
            raise AssertionError("Unsupported data type %s" % (dtype,))
        self.pattern = a, b, c, d = tuple(int(v) for v in pattern)
        self.in_size, self.out_size = a * c * d, a * b * d
        self.act, self.bs_last, self.dtype = act, bs_last, dtype
        if weights is None:
            s = 1.0 / math.sqrt(c)
            weights = [torch.empty(a, b, c, d).uniform_(-s, s) for _ in range(2)]
        assert len(weights) == 2 and all(tuple(w.shape) == self.pattern for w in weights)
        self.factor = nn.Parameter(pack_gated(*weights, dtype, device))
        if bias:
            bound = 1 / math.sqrt(self.in_size)
            self.bias = nn.Parameter(torch.empty(2 * self.out_size, device=device).uniform_(-bound, bound).to(dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        return gated_linear(x, self.factor, self.pattern, self.bias, self.act, self.bs_last)

    def extra_repr(self):
        return "pattern={}, act={}, bias={}, bs_last={}".format(self.pattern, self.act, self.bias is not None, self.bs_last)


# -- norms around a residual connection ----------------------------------------------------------------


def _check_norm(x, residual, gate, post_weight, weight, bias, norm, bs_last):
    """(batch, features, groups)"""
    if norm not in NORMS:
        raise ValueError("norm must be one of %s" % sorted(NORMS))
    _check_input(residual, "residual")
    _trainable_type(residual, "residual")
    if residual.dim() < 1:
        raise ValueError("residual must have features")
    features = residual.size(0 if bs_last else -1)
    if features < 1:
        raise ValueError("residual must have features, not %s" % (tuple(residual.shape),))
    batch = residual.numel() // features
    if x is not None:
        _same(x, residual, "x")
        if x.shape != residual.shape:
            raise ValueError("x and residual must have one shape, not %s and %s" % (tuple(x.shape), tuple(residual.shape)))
    elif gate is not None or post_weight is not None:
        raise ValueError("gate and post_weight go with x")
    for t, name in ((post_weight, "post_weight"), (weight, "weight"), (bias, "bias")):
        if t is not None:
            _same(t, residual, name)
            if t.numel() != features:
                raise ValueError("%s must hold %d values, not %d" % (name, features, t.numel()))
    groups = 1
    if gate is not None:
        _same(gate, residual, "gate")
        groups = gate.numel() // features
        if gate.size(-1) != features or groups < 1 or batch % groups:
            raise ValueError("gate must hold rows of %d values, as many as divide the batch of %d, not %s" % (features, batch, tuple(gate.shape)))
    return batch, features, groups


class NormKernel:
    """Both directions of the residual norm as single calls on tensors, without autograd."""

    @staticmethod
    def _desc(x, residual, gate, post_weight, weight, bias, alpha, norm, eps, groups):
        d = _lib.KsmmNormDesc(_ptr(x), residual.data_ptr(), _ptr(gate), _ptr(post_weight), _ptr(weight), _ptr(bias))
        d.groups, d.alpha, d.eps, d.kind = groups, alpha, eps, NORMS[norm]
        return d

    @staticmethod
    def forward(x, residual, gate=None, post_weight=None, weight=None, bias=None, alpha=1.0, norm="rms", eps=1e-6, bs_last=False,
                need_norm=True, need_stats=False):
        """(r_out, n_out, stats); r_out is ``residual`` itself where ``x`` is None, what is not needed is None."""
        lib = _lib.load()
        bs_last = bool(bs_last)
        batch, features, groups = _check_norm(x, residual, gate, post_weight, weight, bias, norm, bs_last)
        if x is None and not need_norm:
            raise ValueError("without x there is only the norm to compute")
        r = residual if x is None else torch.empty_like(residual)
        n = torch.empty_like(residual) if need_norm else None
        stats = torch.empty(4, batch, dtype=torch.float32, device=residual.device) if need_stats else None
        if batch > 0:
            desc = NormKernel._desc(x, residual, gate, post_weight, weight, bias, alpha, norm, eps, groups)
            dt = dtype_code(residual.dtype)
            need = lib.ksmm_residual_norm_forward_workspace(batch, features, dt, int(bs_last))
            if need < 0:
                _lib.check(int(need))
            workspace = torch.empty(need, dtype=torch.uint8, device=residual.device) if need else None
            with torch.cuda.device(residual.device):
                _lib.check(lib.ksmm_residual_norm_forward(ctypes.byref(desc), None if x is None else r.data_ptr(), _ptr(n), _ptr(stats),
                                                          _ptr(workspace), need, batch, features, dt, int(bs_last), _stream_ptr(residual)))
        return r, n, stats

    @staticmethod
    def backward(grad_r, grad_n, stats, x, residual, gate=None, post_weight=None, weight=None, bias=None, alpha=1.0, norm="rms",
                 eps=1e-6, bs_last=False, needs=(True,) * 6):
        """Gradients of (x, residual, gate, post_weight, weight, bias); None for what is not needed or not there."""
        lib = _lib.load()
        bs_last = bool(bs_last)
        batch, features, groups = _check_norm(x, residual, gate, post_weight, weight, bias, norm, bs_last)
        for g, name in ((grad_r, "grad_r"), (grad_n, "grad_n")):
            if g is not None:
                _same(g, residual, name)
                if g.shape != residual.shape:
                    raise ValueError("%s must have the residual's shape" % name)
        out = [torch.empty_like(t) if t is not None and need else None
               for t, need in zip((x, residual, gate, post_weight, weight, bias), needs)]
        if batch == 0 or (grad_r is None and grad_n is None):
            return [None if t is None else t.zero_() for t in out]
        dt = dtype_code(residual.dtype)
        need = lib.ksmm_residual_norm_backward_workspace(batch, features, groups, dt, int(bs_last))
        if need < 0:
            _lib.check(int(need))
        workspace = torch.empty(need, dtype=torch.uint8, device=residual.device)
        desc = NormKernel._desc(x, residual, gate, post_weight, weight, bias, alpha, norm, eps, groups)
        with torch.cuda.device(residual.device):
            _lib.check(lib.ksmm_residual_norm_backward(ctypes.byref(desc), stats.data_ptr(), _ptr(grad_r), _ptr(grad_n),
                                                       *(_ptr(t) for t in out), workspace.data_ptr(), need, batch, features, dt,
                                                       int(bs_last), _stream_ptr(residual)))
        return out


class ResidualNormFunction(torch.autograd.Function):
    """``apply(x, residual, gate, post_weight, weight, bias, alpha, norm, eps, bs_last, need_norm)`` -> (r_out, n_out), without
    ``x`` n_out alone, without ``need_norm`` r_out alone."""

    @staticmethod
    def forward(ctx, x, residual, gate, post_weight, weight, bias, alpha, norm, eps, bs_last, need_norm):
        r, n, stats = NormKernel.forward(x, residual, gate, post_weight, weight, bias, alpha, norm, eps, bs_last, need_norm, True)
        ctx.save_for_backward(x, residual, gate, post_weight, weight, bias, stats)
        ctx.how = alpha, norm, eps, bs_last
        ctx.results = x is not None, need_norm
        ctx.set_materialize_grads(False)
        return n if x is None else (r, n) if need_norm else r

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        *inputs, stats = ctx.saved_tensors
        has_x, need_norm = ctx.results
        grads = [None if g is None else g.contiguous() for g in grads]
        grad_r = grads[0] if has_x else None
        grad_n = grads[-1] if need_norm else None
        out = NormKernel.backward(grad_r, grad_n, stats, *inputs, *ctx.how, needs=ctx.needs_input_grad[:6])
        return (*out, None, None, None, None, None)


def residual_norm(x, residual, gate=None, post_weight=None, weight=None, bias=None, alpha=1.0, norm="rms", eps=1e-6, bs_last=False,
                  need_norm=True):
    """(r_out, n_out): the residual connection around a block and the norm before the next one, in one kernel.

        r_out = residual + alpha * gate * P(x)    P(x) = x, or norm(x) * post_weight where that is given
        n_out = norm(r_out) * weight + bias       ``norm``: "rms" or "layer", over the features of a row

    Tensors have their features in the last axis, or with ``bs_last`` in the first.  ``gate``: one value a feature, or
    rows of them ((groups, features): one for every batch / groups consecutive rows, as for the tokens of an image).
    ``x`` None: the norm before the first block, r_out is ``residual`` itself.  ``need_norm`` False: the
    addition alone, n_out is None.  Missing gates and weights count as ones.  Everything has a gradient but ``alpha``;
    gradients cannot be differentiated a second time."""
    inputs = x, residual, gate, post_weight, weight, bias
    out = _lib.native().residual_norm(*inputs, alpha, norm, eps, bs_last, need_norm)
    if out is not None:
        return out
    if torch.jit.is_tracing() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)):
        out = ResidualNormFunction.apply(*inputs, float(alpha), norm, float(eps), bs_last, need_norm)
        return (residual, out) if x is None else out if need_norm else (out, None)
    r, n, _ = NormKernel.forward(*inputs, alpha, norm, eps, bs_last, need_norm)
    return r, n


class ResidualNorm(nn.Module):
    """``residual_norm`` with its parameters: ``post`` a norm (with weights) of the block's result, ``gate`` a learned
    value a feature that starts at ``gate_init`` (False: none, or one handed to ``forward``)."""

    def __init__(self, features, norm="rms", post=False, gate=False, gate_init=1.0, alpha=1.0, bias=None, eps=1e-6,
                 dtype=torch.float16, bs_last=False, device="cuda", need_norm=True):
        super().__init__()
        if norm not in NORMS:
            raise ValueError("norm must be one of %s" % sorted(NORMS))
        self.norm, self.alpha, self.eps, self.bs_last, self.need_norm = norm, alpha, eps, bs_last, need_norm
        bias = norm == "layer" if bias is None else bias

        def vector(wanted, value):
            return nn.Parameter(torch.full((features,), value, dtype=dtype, device=device)) if wanted else None

        self.gate, self.post_weight = vector(gate, float(gate_init)), vector(post, 1.0)
        self.weight, self.bias = vector(need_norm, 1.0), vector(need_norm and bias, 0.0)

    def forward(self, x, residual, gate=None):
        if x is None:
            return residual_norm(None, residual, weight=self.weight, bias=self.bias, norm=self.norm, eps=self.eps, bs_last=self.bs_last)
        return residual_norm(x, residual, self.gate if gate is None else gate, self.post_weight, self.weight, self.bias, self.alpha,
                             self.norm, self.eps, self.bs_last, self.need_norm)


class KSFeedForward(nn.Module):
    """Gated feed-forward block of Kronecker-sparse layers between two norms:

        h = act(G n) * (U n),  y = K_m .. K_1 h,  (r, n) <- residual_norm(y, r)

    ``gated``: pattern of G and U; ``down``: patterns of the KSLinear behind them.  ``forward(n, r)`` takes the
    normed input and the residual stream and returns both for the next block; ``begin(r)`` norms the first one's."""

    def __init__(self, gated, down, norm="rms", post=True, gate=True, gate_init=1.0, alpha=1.0, act="silu", bias=False,
                 dtype=torch.float16, bs_last=False, device="cuda"):
        super().__init__()
        self.gated = KSGatedLinear(gated, bias=bias, dtype=dtype, bs_last=bs_last, device=device, act=act)
        self.down = KSLinear(down, bias=bias, algo="kernel", dtype=dtype, bs_last=bs_last, device=device)
        if self.gated.out_size != self.down.in_size or self.down.out_size != self.gated.in_size:
            raise ValueError("%d -> %d and %d -> %d features do not make a block" % (
                self.gated.in_size, self.gated.out_size, self.down.in_size, self.down.out_size))
        self.norm = ResidualNorm(self.gated.in_size, norm, post, gate, gate_init, alpha, dtype=dtype, bs_last=bs_last, device=device)

    def begin(self, residual):
        """The norm before the first block (without weights: the first products have their own)."""
        return residual_norm(None, residual, norm=self.norm.norm, eps=self.norm.eps, bs_last=self.norm.bs_last)[1]

    def forward(self, normed, residual):
        residual, normed = self.norm(self.down(self.gated(normed)), residual)
        return normed, residual
