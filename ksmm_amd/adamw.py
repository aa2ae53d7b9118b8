"""AdamW over many tensors in one launch, its moments in 32 or in 8 bits, on the hand-written kernels of libksmm_hip.so: for all
parameters of a model, or for those that ``KSMuon`` leaves (``KSMuon.others``).
"""
import ctypes
import math

import torch

from . import _lib
from .block import _ptr, _written
from .kernel import _check_input, _stream_ptr, dtype_code

BLOCK = 32


def _check_lists(params, **lists):
    for name, tensors in lists.items():
        if tensors is not None and len(tensors) != len(params):
            raise ValueError("%d %s for %d parameters" % (len(tensors), name, len(params)))


def _check_one(t, name, n, dtype, device):
    _check_input(t, name)
    if t.dtype != dtype or t.device != device or t.numel() != n:
        raise ValueError("%s must hold %d values in %s on %s" % (name, n, dtype, device))


def _scales_of(n):
    return 2, (n + BLOCK - 1) // BLOCK


def adamw_update(params, grads, exp_avgs, exp_avg_sqs, scales=None, masters=None, step=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.01, grad_scale=1.0, seed=0, follow=False):
    """One step of AdamW over all of ``params``, in their place:

        g = grad_scale * grad,  m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        w = (1 - lr * weight_decay) w - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)

    Lists of contiguous tensors, parameters and gradients of one type (float32 or float16) on one device.  ``exp_avgs`` and
    ``exp_avg_sqs``: float32; or uint8 with ``scales`` (uint8, (2, ceil(n / 32)) each), blocks of 32 values with a power of two in common,
    e4m3 and unsigned e5m3, rounded up or down by a hash of ``seed``, the tensor's number, step and place, so that
    their mean is kept.  Zeros everywhere are a state to start from.
    ``masters``: fp32 weights that the parameters are rounded from; they are read instead of them and written too.
    ``follow``: a parameter that is not what its master rounds to was written since, and counts instead.
    ``eps``: 0, or 2^-126 and more.  ``step``: from 1 on, or an int64 tensor of one value on the device, which a captured graph reads anew on every replay.
    What a NaN or an infinity among the gradients reaches is its own element alone."""
    if len(betas) != 2:
        raise ValueError("betas must be two values from 0 on and below 1, not %s" % (betas,))
    done = _lib.native().adamw_update(params, grads, exp_avgs, exp_avg_sqs, scales, masters, step, lr, betas[0], betas[1], eps, weight_decay,
                                      grad_scale, seed, follow)
    if done is not None:
        if done is not True:  # a launch failed: others may have been made, and a second call would update their tensors twice
            _lib.check(done)
        return
    lib = _lib.load()
    params, grads = [p.detach() for p in params], [g.detach() for g in grads]
    _check_lists(params, grads=grads, exp_avgs=exp_avgs, exp_avg_sqs=exp_avg_sqs, scales=scales, masters=masters)
    if not params:
        return
    like = params[0]
    small = scales is not None
    if like.dtype not in (torch.float32, torch.float16):
        raise AssertionError("Unsupported data type %s of parameters: float32 and float16 are" % (like.dtype,))
    if not all(0.0 <= b < 1.0 for b in betas):
        raise ValueError("betas must be two values from 0 on and below 1, not %s" % (betas,))
    if not all(math.isfinite(v) for v in (lr, eps, weight_decay, grad_scale)):
        raise ValueError("lr, eps, weight_decay and grad_scale must be finite")
    on_device = isinstance(step, torch.Tensor)
    if on_device:
        _check_one(step, "step", 1, torch.int64, like.device)
    elif step < 1:
        raise ValueError("step counts from 1 on, not %s" % (step,))
    table = (_lib.KsmmAdamwTensor * len(params))()
    state = torch.uint8 if small else torch.float32
    for i, p in enumerate(params):
        n = p.numel()
        _check_one(p, "params[%d]" % i, n, like.dtype, like.device)
        _check_one(grads[i], "grads[%d]" % i, n, like.dtype, like.device)
        _check_one(exp_avgs[i], "exp_avgs[%d]" % i, n, state, like.device)
        _check_one(exp_avg_sqs[i], "exp_avg_sqs[%d]" % i, n, state, like.device)
        if small:
            _check_one(scales[i], "scales[%d]" % i, math.prod(_scales_of(n)), torch.uint8, like.device)
        if masters is not None:
            _check_one(masters[i], "masters[%d]" % i, n, torch.float32, like.device)
        table[i] = _lib.KsmmAdamwTensor(p.data_ptr(), grads[i].data_ptr(), None if masters is None else masters[i].data_ptr(),
                                        exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(), scales[i].data_ptr() if small else None, n)
    desc = _lib.KsmmAdamwDesc(lr, betas[0], betas[1], eps, weight_decay, grad_scale, 1 if on_device else int(step),
                              step.data_ptr() if on_device else None, seed & 0xffffffff, 8 if small else 32, int(follow))
    with torch.cuda.device(like.device):
        status = lib.ksmm_adamw_update(ctypes.byref(desc), table, len(params), dtype_code(like.dtype), _stream_ptr(like))
    if status in (0, _lib.ERR_LAUNCH):  # (of several launches some may have been made)
        _written(*params, *exp_avgs, *exp_avg_sqs, *(scales or ()), *(masters or ()))
    _lib.check(status)


def adamw_moments(exp_avgs, exp_avg_sqs, scales):
    """What moments in 8 bits stand for: two lists of float32 tensors, of the shapes of ``exp_avgs``."""
    done = _lib.native().adamw_moments(exp_avgs, exp_avg_sqs, scales)
    if done is not None:
        return done
    lib = _lib.load()
    _check_lists(exp_avgs, exp_avg_sqs=exp_avg_sqs, scales=scales)
    if not exp_avgs:
        return [], []
    device = exp_avgs[0].device
    table = (_lib.KsmmAdamwMoment * len(exp_avgs))()
    m, v = [], []
    for i, (x, y, s) in enumerate(zip(exp_avgs, exp_avg_sqs, scales)):
        n = x.numel()
        for t, name, k in ((x, "exp_avgs[%d]", n), (y, "exp_avg_sqs[%d]", n), (s, "scales[%d]", math.prod(_scales_of(n)))):
            _check_one(t, name % i, k, torch.uint8, device)
        m.append(torch.empty(x.shape, dtype=torch.float32, device=device))
        v.append(torch.empty(x.shape, dtype=torch.float32, device=device))
        table[i] = _lib.KsmmAdamwMoment(x.data_ptr(), y.data_ptr(), s.data_ptr(), m[i].data_ptr(), v[i].data_ptr(), n)
    with torch.cuda.device(device):
        _lib.check(lib.ksmm_adamw_moments(table, len(m), _stream_ptr(exp_avgs[0])))
    return m, v


class KSAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over all parameters of a group, type and device in one launch.

        opt = KSAdamW(model.parameters(), lr=1e-3)                  # of everything
        muon, rest = KSMuon(model), KSAdamW(KSMuon.others(model))   # beside the factors' own updates

    ``bits``: 32, or 8 for moments that take 2.06 bytes a weight instead of 8 (``adamw_update`` says how; the tensors' numbers go on over
    all groups).  fp16 parameters are
    rounded from fp32 weights that the optimiser keeps (``master=False``: updated as they are); values that were written into
    a parameter since replace them.  ``grad_scale`` multiplies the gradients: one over a loss's scale.  ``capturable``: the count of steps is
    a tensor of the group's on its one device, so that a captured step counts on with every replay (a step before the capture sets the
    state up; without either a capture is refused)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, bits=32, master=True, grad_scale=1.0, seed=0,
                 capturable=False):
        if bits not in (8, 32):
            raise ValueError("bits must be 8 or 32, not %s" % (bits,))
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas must be two values from 0 on and below 1, not %s" % (betas,))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, bits=bits, master=master,
                                      grad_scale=grad_scale, seed=seed, capturable=capturable))
        for g in self.param_groups:
            for p in g["params"]:
                self._check_parameter(p)
            if capturable and len({p.device for p in g["params"]}) > 1:
                raise ValueError("capturable parameters of a group must be on one device")

    @staticmethod
    def _check_parameter(p):
        if p.dtype not in (torch.float32, torch.float16):
            raise AssertionError("Unsupported data type %s of a parameter: float32 and float16 are" % (p.dtype,))
        if not p.is_contiguous():
            raise ValueError("parameters must be contiguous")

    def _state_of(self, p, g):
        state = self.state[p]
        if not state:
            n = p.numel()
            if g["bits"] == 8:
                state["exp_avg"] = torch.zeros(n, dtype=torch.uint8, device=p.device)
                state["exp_avg_sq"] = torch.zeros(n, dtype=torch.uint8, device=p.device)
                state["scales"] = torch.zeros(_scales_of(n), dtype=torch.uint8, device=p.device)
            else:
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if g["master"] and p.dtype == torch.float16:
                state["master"] = p.detach().float()
            state["step"] = 0
        return state

    def load_state_dict(self, state_dict):
        """As any optimiser's, but that the state keeps its types (the base class rounds what it loads to the parameters'
        type), and is a copy."""
        given = []

        def seen(_, loaded):
            given.append(loaded)

        def widen(_):
            of = [i for g in given[-1]["param_groups"] for i in g["params"]]
            for i, p in zip(of, (p for g in self.param_groups for p in g["params"])):
                for name, t in given[-1]["state"].get(i, {}).items():
                    if isinstance(t, torch.Tensor):
                        self.state[p][name] = t.to(device=p.device, copy=True).contiguous()
            for g in self.param_groups:
                if isinstance(g.get("step"), torch.Tensor):
                    g["step"] = g["step"].to(device=g["params"][0].device, copy=True)

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
        capturing = torch.cuda.is_current_stream_capturing()
        number = 0  # of tensors whose step was made: those of all groups and types are rounded by numbers of their own
        for g in self.param_groups:
            sets = {}
            if capturing and not (g["capturable"] and g.get("step") is not None and all(self.state[p] for p in g["params"] if p.grad is not None)):
                raise RuntimeError("a captured step needs capturable=True and a step before the capture: it would not count, or begin anew on every replay")
            if g["capturable"]:
                if g.get("step") is None:
                    g["step"] = torch.zeros(1, dtype=torch.int64, device=g["params"][0].device)
                g["step"] += 1
            for p in g["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("KSAdamW does not take sparse gradients")
                self._check_parameter(p)
                state = self._state_of(p, g)
                state["step"] += 1  # (one that was left out of some steps counts its own, but for capturable ones)
                key = p.dtype, p.device, "scales" in state, "master" in state, None if g["capturable"] else state["step"]
                sets.setdefault(key, []).append((p, state))
            for (_, _, small, master, count), found in sets.items():
                ps, states = zip(*found)
                adamw_update(ps, [p.grad.contiguous() for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                             [s["scales"] for s in states] if small else None, [s["master"] for s in states] if master else None,
                             g["step"] if count is None else count, g["lr"], g["betas"], g["eps"], g["weight_decay"], g["grad_scale"],
                             g["seed"] + number, follow=True)
                number += len(ps)
        return loss
