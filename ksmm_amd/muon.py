"""Updates of Kronecker-sparse factors that are made orthogonal block by block (Newton-Schulz), and the optimiser
that takes them, on the hand-written kernels of libksmm_hip.so.

A factor in kernel format is its a*d dense blocks (c x b) one after the other, so that each of them is orthogonalised as a
matrix of its own; a gated projection's factor holds two side by side (``parts=2``).
"""
import ctypes
import math

import torch

from . import _lib
from .block import KSGatedLinear, _ptr, _same, _trainable_type, _written
from .kernel import _check_input, _stream_ptr, dtype_code
from .layer import KSLinear

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _check(update, pattern, parts, steps, coefficients, name):
    a, b, c, d = (int(v) for v in pattern)
    if min(a, b, c, d) < 1 or parts < 1:
        raise ValueError("pattern must hold four sizes of one and more, and parts be one or more: %s, %s" % (pattern, parts))
    if steps < 1:
        raise ValueError("steps must be one or more")
    if len(coefficients) != 3:
        raise ValueError("coefficients must be three")
    _check_input(update, name)
    _trainable_type(update, name)
    if tuple(update.shape) != (a * d * c, parts * b):
        raise ValueError("%s must be %s, not %s" % (name, (a * d * c, parts * b), tuple(update.shape)))
    return a, b, c, d


def _launch(grad, shape, parts, steps, coefficients, eps, out, momentum=None, momentum_out=None, weight=None, master=None,
            master_out=None, beta=0.0, keep=1.0, rate=1.0, nesterov=True, follow=False):
    lib = _lib.load()
    a, b, c, d = shape
    need = lib.ksmm_muon_workspace(a * d, c, b, parts)
    if need < 0:
        _lib.check(int(need))
    workspace = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
    desc = _lib.KsmmMuonDesc((ctypes.c_float * 3)(*coefficients), eps, beta, keep, rate, steps, int(nesterov), int(follow))
    with torch.cuda.device(grad.device):
        _lib.check(lib.ksmm_muon_update(ctypes.byref(desc), grad.data_ptr(), _ptr(momentum), _ptr(momentum_out), _ptr(weight),
                                        _ptr(master), _ptr(master_out), out.data_ptr(), _ptr(workspace), need, a * d, c, b, parts,
                                        dtype_code(grad.dtype), _stream_ptr(grad)))


def orthogonalize(update, pattern, parts=1, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The blocks of ``update``, a factor of ``pattern`` in kernel format (a*d*c, parts*b), made orthogonal: each
    c x b matrix X is divided by its Frobenius norm + ``eps`` and goes through ``steps`` steps of
    X <- p0 X + (p1 A + p2 A A) X, A = X X^T.  X is held in 22 bits (and to 1.5e-11), sums are fp32; the result is rounded once to the
    update's type.  Coefficients whose steps could take a matrix of singular values up to 1 beyond 60000 are refused."""
    shape = _check(update, pattern, parts, steps, coefficients, "update")
    out = torch.empty_like(update)
    _launch(update.detach(), shape, parts, steps, coefficients, eps, out)
    return out


def muon_update(weight, grad, momentum, pattern, parts=1, lr=0.02, beta=0.95, weight_decay=0.0, nesterov=True, steps=5,
                coefficients=COEFFICIENTS, eps=1e-7, master=None, inplace=False, follow=False):
    """(new weight, new momentum) of one step:

        m = beta * momentum + grad,  u = grad + beta * m (``nesterov``) or m
        w = (1 - lr * weight_decay) * weight - lr * sqrt(max(1, b / c)) * orthogonalize(u)

    ``weight`` and ``grad`` are kernel-format tensors of one type, ``momentum`` is fp32 and of their shape.  ``master``: fp32
    weights that ``weight`` is rounded from; they are read instead of it and updated in place.  ``follow``: where ``weight`` is not
    what ``master`` rounds to, it was written since, and counts instead.  ``inplace`` writes the results over ``weight`` and
    ``momentum``."""
    shape = _check(grad, pattern, parts, steps, coefficients, "grad")
    _same(weight, grad, "weight")
    for t, name in ((momentum, "momentum"), (master, "master")):
        if t is None and name == "master":
            continue
        _check_input(t, name)
        if t.dtype != torch.float32 or t.device != grad.device or t.shape != grad.shape:
            raise ValueError("%s must be float32 of the gradient's shape" % name)
    if weight.shape != grad.shape:
        raise ValueError("weight and grad must have one shape")
    weight, grad = weight.detach(), grad.detach()
    out, m = (weight, momentum) if inplace else (torch.empty_like(weight), torch.empty_like(momentum))
    _, b, c, _ = shape
    _launch(grad, shape, parts, steps, coefficients, eps, out, momentum, m, weight, master, master, beta, 1 - lr * weight_decay,
            lr * math.sqrt(max(1.0, b / c)), nesterov, follow)
    _written(*((weight, momentum) if inplace else ()), *(() if master is None else (master,)))
    return out, m


class KSMuon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for the factors of ``KSLinear(algo='kernel')`` and ``KSGatedLinear`` modules.

        opt = KSMuon(model)            # every such factor of a module, or a list of (parameter, pattern, parts)

    The other parameters (biases, norms, gates) belong to another optimiser; ``others(model)`` lists them.  fp16
    factors are rounded from fp32 weights that the optimiser keeps (``master=False``: updated as they are); values that were
    written into a factor since, a checkpoint's say, replace them."""

    def __init__(self, factors, lr=0.02, beta=0.95, weight_decay=0.0, nesterov=True, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                 master=True):
        if isinstance(factors, torch.nn.Module):
            factors = self.factors_of(factors)
        factors = list(factors)
        if not factors:
            raise ValueError("no Kronecker-sparse factors")
        defaults = dict(lr=lr, beta=beta, weight_decay=weight_decay, nesterov=nesterov, steps=steps, coefficients=tuple(coefficients),
                        eps=eps, master=master)
        for p, pattern, parts in factors:
            _check(p.detach(), pattern, parts, steps, coefficients, "factor")
        super().__init__([{"params": [p], "pattern": tuple(pattern), "parts": parts} for p, pattern, parts in factors], defaults)

    @staticmethod
    def factors_of(module):
        """(parameter, pattern, parts) of every factor that takes gradients; one that several modules share is one."""
        found = []
        for m in module.modules():
            if isinstance(m, KSGatedLinear):
                found.append((m.factor, m.pattern, 2))
            elif isinstance(m, KSLinear) and m.algo == "kernel":
                found += [(f, p, 1) for f, p in zip(m.factors, m.patterns)]
        once = {}
        for f in found:
            if f[0].requires_grad:
                once.setdefault(id(f[0]), f)
        return list(once.values())

    @classmethod
    def others(cls, module):
        """The parameters of a module that are none of its factors."""
        mine = {id(p) for p, _, _ in cls.factors_of(module)}
        return [p for p in module.parameters() if id(p) not in mine]

    def load_state_dict(self, state_dict):
        """As any optimiser's, but that the fp32 momentum and weights of fp16 factors stay fp32 (the base class rounds what it
        loads to the parameters' type), and are copies."""
        given = []

        def seen(_, loaded):
            given.append(loaded)

        def widen(_):
            of = [i for g in given[-1]["param_groups"] for i in g["params"]]
            for i, p in zip(of, (p for g in self.param_groups for p in g["params"])):
                for name in ("momentum", "master"):
                    t = given[-1]["state"].get(i, {}).get(name)
                    if t is not None:
                        self.state[p][name] = t.to(device=p.device, dtype=torch.float32, copy=True).contiguous()

        # (what the user's own hooks make of the state is what is loaded, and they see it as it will be)
        hooks = self.register_load_state_dict_pre_hook(seen), self.register_load_state_dict_post_hook(widen, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for g in self.param_groups:
            for p in g["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                    state["master"] = p.detach().float() if g["master"] and p.dtype == torch.float16 else None
                muon_update(p, p.grad.contiguous(), state["momentum"], g["pattern"], g["parts"], g["lr"], g["beta"], g["weight_decay"],
                            g["nesterov"], g["steps"], g["coefficients"], g["eps"], state["master"], inplace=True, follow=True)
        return loss
