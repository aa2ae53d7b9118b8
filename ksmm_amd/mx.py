"""Kronecker-sparse products of microscaled 4-bit numbers, on the hand-written kernels of libksmm_hip.so.

A number is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (e2m1); 32 of them along c have a power of two in common (E8M0).
17 bytes hold 32 weights or activations where fp16 takes 64.

    w = pack_mx(factor, (a, b, c, d))            # a factor in kernel format, once
    y = mx_linear(x, w, bias=bias, act="gelu")   # x is made such numbers in the call
    y = mx_linear(x, factor, (a, b, c, d))       # training: the factor too, gradients go straight through the roundings

``KSLinearMX`` and ``KSGatedLinearMX`` are the modules that train so; their ``packed()`` are ``MXLinear``, which hold codes.
"""
import copy
import math

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib
from .block import GATED_ACTS, GatedKernel, KSFeedForward, KSGatedLinear, _ptr, _trainable_type, _written
from .kernel import Kernel, _check_input, _stream_ptr, dtype_code
from .layer import KSLinear

BLOCK = 32


def _sizes(sizes, count, name):
    sizes = tuple(int(v) for v in sizes)
    if len(sizes) != count or min(sizes) < 1:
        raise ValueError("%s must hold %d sizes of one and more, not %s" % (name, count, sizes))
    return sizes


def _blocks(c):
    return (c + BLOCK - 1) // BLOCK


def _check_codes(codes, scales, matrices, c):
    """rows of an operand"""
    rows = _lib.native().mx_rows(codes, scales, matrices, c)
    if rows is not None:
        return rows
    for t, name in ((codes, "codes"), (scales, "scales")):
        _check_input(t, name)
        if t.dtype != torch.uint8 or t.device != codes.device:
            raise ValueError("codes and scales must be uint8 on one device")
    if codes.dim() != 3 or codes.size(0) != matrices or codes.size(2) != 16 * _blocks(c):
        raise ValueError("codes must be (%d, rows, %d), not %s" % (matrices, 16 * _blocks(c), tuple(codes.shape)))
    if tuple(scales.shape) != (matrices, codes.size(1), _blocks(c)):
        raise ValueError("scales must be %s, not %s" % ((matrices, codes.size(1), _blocks(c)), tuple(scales.shape)))
    if codes.data_ptr() % 16:
        raise ValueError("codes must start on a 16-byte boundary")
    return codes.size(1)


def _quantize(x, rows, a, c, d, bs_last):
    done = _lib.native().mx_quantize(x, (a, c, d), bs_last)
    if done is not None:
        return done
    codes = torch.empty(a * d, rows, 16 * _blocks(c), dtype=torch.uint8, device=x.device)
    scales = torch.empty(a * d, rows, _blocks(c), dtype=torch.uint8, device=x.device)
    if rows > 0:
        with torch.cuda.device(x.device):
            _lib.check(_lib.load().ksmm_mx_quantize(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, a, c, d, dtype_code(x.dtype),
                                                    int(bs_last), _stream_ptr(x)))
    return codes, scales


def _dequantize(codes, scales, shape, dtype, rows, a, c, d, bs_last):
    if dtype in (torch.float32, torch.float16):
        x = _lib.native().mx_dequantize(codes, scales, (a, c, d), tuple(shape), dtype == torch.float16, bs_last)
        if x is not None:
            return x
    x = torch.empty(shape, dtype=dtype, device=codes.device)
    if rows > 0:
        with torch.cuda.device(codes.device):
            _lib.check(_lib.load().ksmm_mx_dequantize(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), rows, a, c, d, dtype_code(dtype),
                                                      int(bs_last), _stream_ptr(codes)))
    return x


class MXTensor:
    """Activations as microscaled 4-bit numbers: ``codes`` (a*d, rows, 16 * ceil(c / 32)) and ``scales`` (a*d, rows, ceil(c / 32)),
    both uint8.  A block that held an infinity or a NaN has the scale 255 and stands for NaNs."""

    def __init__(self, codes, scales, sizes, shape, dtype, bs_last=False):
        self.sizes = a, c, d = _sizes(sizes, 3, "sizes")
        rows = _check_codes(codes, scales, a * d, c)
        self.codes, self.scales, self.shape, self.dtype, self.bs_last = codes, scales, tuple(shape), dtype, bool(bs_last)
        if math.prod(self.shape) != rows * a * c * d or not self.shape or self.shape[0 if self.bs_last else -1] != a * c * d:
            raise ValueError("%d rows of %d features do not make a tensor of shape %s" % (rows, a * c * d, self.shape))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=None):
        """The values that the numbers stand for, a tensor like the one that was quantised."""
        dtype = self.dtype if dtype is None else dtype
        a, c, d = self.sizes
        return _dequantize(self.codes, self.scales, self.shape, dtype, self.codes.size(1), a, c, d, self.bs_last)


def quantize_mx(x, sizes, bs_last=False):
    """``x`` as an ``MXTensor``: ``sizes`` (a, c, d) are those of the pattern that it is to be multiplied with, whose a*c*d
    features lie in the last axis, or with ``bs_last`` in the first.  Blocks of 32 along c have the scale 2^e, e = floor(log2 of
    their largest magnitude) - 2 and at least -120; what is larger than 6 of it counts as 6.  fp32 and fp16; no gradients."""
    a, c, d = _sizes(sizes, 3, "sizes")
    _check_input(x, "input")
    _trainable_type(x, "input")
    if x.dim() < 1 or x.size(0 if bs_last else -1) != a * c * d:
        raise ValueError("input must have %d features, not %s" % (a * c * d, tuple(x.shape)))
    codes, scales = _quantize(x.detach(), x.numel() // (a * c * d), a, c, d, bool(bs_last))
    return MXTensor(codes, scales, (a, c, d), x.shape, x.dtype, bs_last)


class MXFactor:
    """A factor of ``pattern`` (a, b, c, d) as microscaled 4-bit numbers: ``codes`` (a*d, b, 16 * ceil(c / 32)) and ``scales``
    (a*d, b, ceil(c / 32)), uint8; with ``gated`` two of them side by side, 2*b rows, the gate's first.  ``dtype``: what they were made
    from.  Numbers of float16 are all float16 values; of float32, or of what is not said, gradients of fp16 inputs are computed in 32 bits."""

    def __init__(self, codes, scales, pattern, gated=False, dtype=None):
        self.pattern = a, b, c, d = _sizes(pattern, 4, "pattern")
        self.codes, self.scales, self.gated, self.dtype = codes, scales, bool(gated), dtype
        rows = _check_codes(codes, scales, a * d, c)
        if rows != (2 * b if gated else b):
            raise ValueError("codes must have %d rows, not %d" % (2 * b if gated else b, rows))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float16):
        """The factor in kernel format, (a*d*c, rows)."""
        a, _, c, d = self.pattern
        rows = self.codes.size(1)
        return _dequantize(self.codes, self.scales, (a * d * c, rows), dtype, rows, a * d, c, 1, True)


def _check_factor(factor, pattern, gated):
    a, b, c, d = _sizes(pattern, 4, "pattern")
    _check_input(factor, "factor")
    _trainable_type(factor, "factor")
    rows = 2 * b if gated else b
    if tuple(factor.shape) != (a * d * c, rows):
        raise ValueError("factor must be %s, not %s" % ((a * d * c, rows), tuple(factor.shape)))
    return a, b, c, d


def pack_mx(factor, pattern, gated=False):
    """A factor in kernel format, (a*d*c, b) or with ``gated`` (a*d*c, 2*b), as an ``MXFactor``."""
    a, b, c, d = _check_factor(factor, pattern, gated)
    codes, scales = _quantize(factor.detach(), factor.size(1), a * d, c, 1, True)
    return MXFactor(codes, scales, (a, b, c, d), gated, factor.dtype)


def _check_product(x, device, pattern, bias, act, gated, bs_last):
    """(rows of the batch, dtype, shape of the result)"""
    if act not in GATED_ACTS or (act == "silu" and not gated):
        raise ValueError("act must be one of %s" % ([k for k in GATED_ACTS if k and (gated or k != "silu")],))
    a, b, c, d = pattern
    if isinstance(x, MXTensor):
        if x.sizes != (a, c, d) or x.bs_last != bool(bs_last):
            raise ValueError("input is quantised for sizes %s, bs_last=%s" % (x.sizes, x.bs_last))
        shape = x.shape
    else:
        _check_input(x, "input")
        shape = tuple(x.shape)
        if x.dim() < 1 or x.size(0 if bs_last else -1) != a * c * d:
            raise ValueError("input must have %d features, not %s" % (a * c * d, shape))
    if x.dtype not in (torch.float32, torch.float16):
        raise AssertionError("Unsupported data type %s of input: float32 and float16 are" % (x.dtype,))
    if x.device != device:
        raise RuntimeError("factor must be on %s" % (x.device,))
    if bias is not None:
        _check_input(bias, "bias")
        if bias.dtype != x.dtype or bias.device != x.device:
            raise RuntimeError("bias must be %s on %s" % (x.dtype, x.device))
        if bias.numel() != (2 * a * b * d if gated else a * b * d):
            raise ValueError("bias must hold %d values, not %d" % (2 * a * b * d if gated else a * b * d, bias.numel()))
    return math.prod(shape) // (a * c * d), x.dtype, ((a * b * d, *shape[1:]) if bs_last else (*shape[:-1], a * b * d))


class MXKernel:
    """The product as a single call on tensors, without autograd."""

    @staticmethod
    def forward(x, factor, bias=None, act=None, bs_last=False, out=None, workspace=None, need_codes=False):
        """The result, or with ``need_codes`` (the result, codes, scales) of x as it was multiplied."""
        lib = _lib.load()
        bs_last = bool(bs_last)
        a, b, c, d = factor.pattern
        batch, dtype, shape = _check_product(x, factor.device, factor.pattern, bias, act, factor.gated, bs_last)
        given = out is not None
        if not given:
            out = torch.empty(shape, dtype=dtype, device=x.device)
        elif tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != x.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous %s of shape %s" % (dtype, tuple(shape)))
        quantised = isinstance(x, MXTensor)
        codes = scales = None
        if need_codes:
            codes = x.codes if quantised else torch.empty(a * d, batch, 16 * _blocks(c), dtype=torch.uint8, device=x.device)
            scales = x.scales if quantised else torch.empty(a * d, batch, _blocks(c), dtype=torch.uint8, device=x.device)
        if batch == 0:
            return (out, codes, scales) if need_codes else out
        dt = dtype_code(dtype)
        need = 0
        if not quantised:
            need = lib.ksmm_mx_forward_workspace(batch, a, b, c, d, dt, int(bs_last), int(factor.gated))
            if need < 0:
                _lib.check(int(need))
            if workspace is not None and (workspace.device != x.device or not workspace.is_contiguous()):
                raise ValueError("workspace must be contiguous on %s" % (x.device,))
            if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
                workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.check(lib.ksmm_mx_forward(
                (x.codes if quantised else x).data_ptr(), x.scales.data_ptr() if quantised else None, factor.codes.data_ptr(),
                factor.scales.data_ptr(), _ptr(bias), out.data_ptr(), None if quantised else _ptr(codes), None if quantised else _ptr(scales),
                workspace.data_ptr() if need > 0 else None,
                workspace.numel() * workspace.element_size() if need > 0 else 0, batch, a, b, c, d, dt, int(bs_last), GATED_ACTS[act],
                int(factor.gated), _stream_ptr(out)))
        if given:
            _written(out)
        return (out, codes, scales) if need_codes else out


class MXFunction(torch.autograd.Function):
    """``apply(x, factor, bias, pattern, act, gated, bs_last)``: both operands are quantised, and kept so (17 bytes for 32 values)
    for the gradients, which are those of the product of what the codes stand for.  ``factor``: in kernel format, or an
    ``MXFactor``, which takes no gradient; where fp16 may not have its values, those of fp16 tensors are computed in fp32."""

    @staticmethod
    def forward(ctx, x, factor, bias, pattern, act, gated, bs_last):
        packed = factor if isinstance(factor, MXFactor) else pack_mx(factor, pattern, gated)
        out, codes, scales = MXKernel.forward(x, packed, bias, act, bs_last, need_codes=True)
        ctx.save_for_backward(codes, scales, packed.codes, packed.scales, bias)
        ctx.how = tuple(pattern), act, bool(gated), bool(bs_last), tuple(x.shape), torch.float32 if packed.dtype != torch.float16 else x.dtype
        ctx.dtype, ctx.factor_dtype = x.dtype, None if packed is factor else factor.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x_codes, x_scales, w_codes, w_scales, bias = ctx.saved_tensors
        pattern, act, gated, bs_last, shape, dtype = ctx.how
        a, b, c, d = pattern
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need_w = need_w and ctx.factor_dtype is not None
        q = MXTensor(x_codes, x_scales, (a, c, d), shape, dtype, bs_last)
        packed = MXFactor(w_codes, w_scales, pattern, gated)
        w = packed.dequantize(dtype)
        grad, bias = grad.to(dtype).contiguous(), None if bias is None else bias.to(dtype)
        dz = _slope(grad, q, packed, bias, act, bs_last) if grad.numel() > 0 and (gated or act not in (None, "none")) else None
        if dz is not None:  # those of a layer without an activation, of the gate's and the other projection's outputs side by side
            packed = MXFactor(w_codes, w_scales, (a, packed.codes.size(1), c, d))
            dx, dw, dbias = _backward(dz, q, packed, w, bias, None, bs_last, need_x, need_w, need_b)
        elif gated:
            dx, dw, dbias = GatedKernel.backward(grad, q.dequantize(), w, pattern, bias, act, bs_last, need_x, need_w, need_b)
        else:
            dx, dw, dbias = _backward(grad, q, packed, w, bias, act, bs_last, need_x, need_w, need_b)
        dx, dbias = (None if t is None else t.to(ctx.dtype) for t in (dx, dbias))
        return dx, None if dw is None else dw.to(ctx.factor_dtype), dbias, None, None, None, None


def _slope(grad, q, packed, bias, act, bs_last):
    """The gradient of what the activation was applied to, or None where no kernel computes both."""
    lib = _lib.load()
    a, b, c, d = packed.pattern
    rows, batch = packed.codes.size(1), q.codes.size(1)

    def call(out):
        return lib.ksmm_mx_slope(q.codes.data_ptr(), q.scales.data_ptr(), packed.codes.data_ptr(), packed.scales.data_ptr(), _ptr(bias), grad.data_ptr(),
                                 _ptr(out), batch, a, b, c, d, dtype_code(grad.dtype), int(bs_last), GATED_ACTS[act], int(packed.gated), _stream_ptr(grad))

    if call(None) != 0:
        return None
    out = torch.empty((a * rows * d, batch) if bs_last else (batch, a * rows * d), dtype=grad.dtype, device=grad.device)
    with torch.cuda.device(grad.device):
        _lib.check(call(out))
    return out


def _backward(grad, q, packed, w, bias, act, bs_last, need_x, need_w, need_b):
    a, b, c, d = packed.pattern
    if grad.numel() == 0:
        shape = q.shape
        return (grad.new_empty(shape) if need_x else None, torch.zeros_like(w) if need_w else None,
                torch.zeros_like(bias) if need_b and bias is not None else None)
    out = a * b * d
    flat = grad.view(out, -1) if bs_last else grad.view(-1, out)
    act = None if act == "none" else act
    z = None
    if act is not None:  # what the activation was applied to, computed again
        z = torch.empty_like(flat)
        with torch.cuda.device(grad.device):
            _lib.check(_lib.load().ksmm_mx_sums(q.codes.data_ptr(), q.scales.data_ptr(), packed.codes.data_ptr(), packed.scales.data_ptr(), _ptr(bias), z.data_ptr(),
                                                q.codes.size(1), a, b, c, d, dtype_code(q.dtype), int(bs_last), _stream_ptr(grad)))
    need_b = need_b and bias is not None
    x = q.dequantize()
    x = x.view(a * c * d, -1) if bs_last else x.view(-1, a * c * d)
    done = _lib.native().train_backward(flat, [w], [(a, b, c, d)], [x], z, bs_last, act, need_x, need_b, (need_w,))
    if done is not None:
        dx, dbias, (dw,) = done
    else:
        dbias = None
        if act is not None or need_b:
            flat, dbias = Kernel.epilogue_backward(flat, z, bs_last, act, need_b)
        dx, dw = Kernel.backward(flat, x, w, bs_last, a, b, c, d, need_input=need_x, need_weight=need_w) if need_x or need_w else (None, None)
    return None if dx is None else dx.view(q.shape), dw, None if dbias is None else dbias.reshape(bias.shape)


def mx_linear(x, factor, pattern=None, bias=None, act=None, gated=False, bs_last=False):
    """``act(W x + bias)``, or with ``gated`` ``act(G x + bias_g) * (U x + bias_u)``, of microscaled 4-bit numbers with fp32 sums.

    ``x``: fp32 or fp16, with a*c*d features in the last axis (``bs_last``: the first), quantised in the call, or an ``MXTensor``.
    ``factor``: an ``MXFactor`` (``pattern`` and ``gated`` are its own then), or a factor in kernel format, which is quantised in
    the call.  ``bias`` has x's type.  ``act``: None, "gelu" (erf form), and with ``gated`` "silu".  The result has x's type.
    Gradients of x, of a factor in kernel format and of the bias are those of the product of the quantised values, handed
    straight through the roundings; they cannot be differentiated a second time, nor in forward mode.  In fp16 the gradients of the
    projections are held in fp16 between the steps, as ``gated_linear`` holds them; and where no kernel has both, what GELU is applied to is too
    (at most 65504): of one factor batch-size-first d of 5 and more, or c that registers do not hold.  Through an ``MXFactor`` that was not made
    from fp16 values the gradients of fp16 tensors are computed in fp32, and rounded at the end."""
    if isinstance(factor, MXFactor):
        if pattern is not None and tuple(pattern) != factor.pattern:
            raise ValueError("factor has the pattern %s, not %s" % (factor.pattern, tuple(pattern)))
        if gated and not factor.gated:
            raise ValueError("factor is not a gated one")
        pattern, gated = factor.pattern, factor.gated
        out = _lib.native().mx_linear(x, factor.codes, factor.scales, pattern, gated, bias, act, bs_last, factor.dtype != torch.float16)
        if out is not None:
            return out
    elif pattern is None:
        raise ValueError("a factor in kernel format needs its pattern")
    else:
        out = _lib.native().mx_linear(x, factor, None, pattern, gated, bias, act, bs_last, False)
        if out is not None:
            return out
        pattern = _check_factor(factor, pattern, gated)[:4]
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in (x, factor, bias)):
        raise RuntimeError("mx_linear has no forward-mode derivative: a tangent would be lost")
    if torch.jit.is_tracing() or (torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, factor, bias))):
        if isinstance(x, MXTensor):
            raise RuntimeError("a quantised input has no gradient: pass the tensor, or call without gradients")
        return MXFunction.apply(x, factor, bias, pattern, act, bool(gated), bool(bs_last))
    if not isinstance(factor, MXFactor):
        factor = pack_mx(factor, pattern, gated)
    return MXKernel.forward(x, factor, bias, act, bs_last)


class KSLinearMX(KSLinear):
    """``KSLinear(algo='kernel')`` whose products are of microscaled 4-bit numbers: every factor and what it is applied to are
    quantised in each pass, between factors the result has the layer's type.  Trains (gradients go straight through the
    roundings); ``packed()`` is the layer to serve."""

    def __init__(self, patterns, weights=None, bias=True, dtype=torch.float16, bs_last=False, device="cuda", act=None):
        if dtype not in (torch.float32, torch.float16):
            raise AssertionError("Unsupported data type %s" % (dtype,))
        super().__init__(patterns, weights, bias, algo="kernel", dtype=dtype, bs_last=bs_last, device=device, act=act)

    def forward(self, x):
        return _chain(x, list(self.factors), self.patterns, self.bias, self.act, self.bs_last)

    def packed(self):
        return MXLinear([pack_mx(f, p) for f, p in zip(self.factors, self.patterns)], self.bias, self.act, self.bs_last)


class KSGatedLinearMX(KSGatedLinear):
    """``KSGatedLinear`` whose products are of microscaled 4-bit numbers, as ``KSLinearMX``'s."""

    def forward(self, x):
        return mx_linear(x, self.factor, self.pattern, self.bias, self.act, True, self.bs_last)

    def packed(self):
        return MXLinear([pack_mx(self.factor, self.pattern, True)], self.bias, self.act, self.bs_last)


def _chain(x, factors, patterns, bias, act, bs_last):
    last = len(factors) - 1
    for i, (f, p) in enumerate(zip(factors, patterns)):
        gated = isinstance(f, MXFactor) and f.gated
        x = mx_linear(x, f, p, bias if i == last else None, act if i == last else None, gated, bs_last)
    return x


def _type_of(scales):
    """float16 where all of a factor's numbers are float16 values, else float32.  6 * 2^13 and 0.5 * 2^-23 are; of 2^-77 and less (and of zeros)
    nothing is left in a float16 gradient."""
    fine = ((scales >= 104) & (scales <= 140)) | (scales <= 50) | (scales == 255)
    return torch.float16 if bool(fine.all()) else torch.float32


class MXLinear(nn.Module):
    """A layer of packed factors, the first one applied first: what ``KSLinearMX.packed()`` gives, or of any
    ``KSLinear(algo='kernel')`` or ``KSGatedLinear`` ``MXLinear.of``.  Codes and scales are buffers, a copy of the factors as they
    were; the bias is a buffer too.  Gradients of the input go straight through."""

    def __init__(self, factors, bias=None, act=None, bs_last=False):
        super().__init__()
        if not factors:
            raise ValueError("no factors")
        self.patterns, self.gated, self.dtypes = [f.pattern for f in factors], [f.gated for f in factors], [f.dtype for f in factors]
        if any(self.gated[:-1]):
            raise ValueError("only the last factor may be gated")
        for p, q in zip(self.patterns, self.patterns[1:]):
            if p[0] * p[1] * p[3] != q[0] * q[2] * q[3]:
                raise ValueError("%s and %s do not make a chain" % (p, q))
        if act not in GATED_ACTS or (act == "silu" and not self.gated[-1]):
            raise ValueError("act must be one of %s" % ([k for k in GATED_ACTS if k and (self.gated[-1] or k != "silu")],))
        self.act, self.bs_last = act, bool(bs_last)
        first, last = self.patterns[0], self.patterns[-1]
        self.in_size, self.out_size = first[0] * first[2] * first[3], last[0] * last[1] * last[3]
        for i, f in enumerate(factors):
            self.register_buffer("codes%d" % i, f.codes)
            self.register_buffer("scales%d" % i, f.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def of(cls, layer):
        if isinstance(layer, KSGatedLinear):
            return cls([pack_mx(layer.factor, layer.pattern, True)], layer.bias, layer.act, layer.bs_last)
        if not isinstance(layer, KSLinear) or layer.algo != "kernel" or layer.dtype not in (torch.float32, torch.float16):
            raise ValueError("a KSGatedLinear, or a KSLinear(algo='kernel') in fp32 or fp16, can be packed")
        return cls([pack_mx(f, p) for f, p in zip(layer.factors, layer.patterns)], layer.bias, layer.act, layer.bs_last)

    def factors(self):
        return [MXFactor(getattr(self, "codes%d" % i), getattr(self, "scales%d" % i), p, g, t)
                for i, (p, g, t) in enumerate(zip(self.patterns, self.gated, self.dtypes))]

    def _load_from_state_dict(self, state_dict, prefix, *how):
        super()._load_from_state_dict(state_dict, prefix, *how)
        for i in range(len(self.dtypes)):
            scales = state_dict.get("%sscales%d" % (prefix, i))
            if scales is not None:
                self.dtypes[i] = None if scales.is_meta else _type_of(scales)

    def forward(self, x):
        return _chain(x, self.factors(), self.patterns, self.bias, self.act, self.bs_last)

    def extra_repr(self):
        return "patterns={}, gated={}, act={}, bias={}, bs_last={}".format(self.patterns, self.gated[-1], self.act, self.bias is not None,
                                                                           self.bs_last)


class KSFeedForwardMX(KSFeedForward):
    """``KSFeedForward`` whose products are of microscaled 4-bit numbers.  ``packed()``: a copy that serves, its factors as codes."""

    def __init__(self, gated, down, *args, bias=False, dtype=torch.float16, bs_last=False, device="cuda", act="silu", **how):
        super().__init__(gated, down, *args, bias=bias, dtype=dtype, bs_last=bs_last, device=device, act=act, **how)
        self.gated = KSGatedLinearMX(gated, bias=bias, dtype=dtype, bs_last=bs_last, device=device, act=act)
        self.down = KSLinearMX(down, bias=bias, dtype=dtype, bs_last=bs_last, device=device)

    def packed(self):
        return pack_block(self)


def _shell(module):
    """A copy of a module with what it has, whose modules, parameters, buffers and hooks are registered for itself."""
    new = copy.copy(module)
    new.__dict__.update({k: v.copy() for k, v in module.__dict__.items() if isinstance(v, (dict, set))})
    return new


def pack_block(block):
    """A copy of a ``KSFeedForward`` whose factors are packed; its norm is copied too."""
    new = _shell(block)
    new.gated, new.down, new.norm = MXLinear.of(block.gated), MXLinear.of(block.down), copy.deepcopy(block.norm)
    return new
