"""Residual norm: gradients of gates that belong to groups of rows, each group with its own.

Tolerances as in test_gpu_norm.py: fp16 results are rounded once, from fp32: 4.9e-4 relative Frobenius, and 2^-25 a value where they
are subnormal; fp32 5e-6.  Gradients of gates also value by value: half a step of the type, and 4e-6 of the sum of the terms' sizes
(a dozen fp32 roundings of each, and those of the sum)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
TOL = {"fp32": 5e-6, "fp16": 4.9e-4}


def oracle(x, residual, gate, post, weight, bias, alpha, norm, eps):
    """On float64 rows, differentiable: (r_out, n_out)."""
    def normed(v):
        if norm == "layer":
            v = v - v.mean(1, keepdim=True)
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)

    p = normed(x) * post if post is not None else x
    r = residual + alpha * p * gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)
    return r, normed(r) * weight + bias


def rel(x, y):
    assert bool(x.isfinite().all())
    n = float(torch.linalg.vector_norm(y))
    e = float(torch.linalg.vector_norm(x.double().cpu() - y))
    if x.dtype == torch.float16:
        e = max(0.0, e - 2 ** -25 * math.sqrt(y.numel()))
    return e / n if n else e


def operands(features, batch, groups, dtype, post, seed=0, x_scale=1.0, dr_scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def make(*s, scale=1.0, mean=0.0):
        return (torch.randn(s, generator=g) * scale + mean).to(dtype)

    t = {"x": make(batch, features, scale=x_scale), "residual": make(batch, features, mean=-0.2), "gate": make(groups, features, scale=0.3, mean=0.5),
         "post": make(features, scale=0.1, mean=1.0) if post else None, "weight": make(features, scale=0.1, mean=1.0), "bias": make(features, scale=0.1)}
    return t, make(batch, features, scale=dr_scale), make(batch, features)


def check(t, dr, dn, prec, norm, bs_last, wanted, use_dr=True):
    from ksmm_amd import residual_norm

    leaves = {k: v.double().requires_grad_(k in wanted) for k, v in t.items() if v is not None}
    args = [leaves.get(k) for k in ("x", "residual", "gate", "post", "weight", "bias")]

    def laid(v, k):
        return v.t().contiguous() if bs_last and k in ("x", "residual") else v

    with torch.enable_grad():
        r, n = oracle(*args, 0.7, norm, 1e-5)
        outs, grads = ([r, n], [dr.double(), dn.double()]) if use_dr else ([n], [dn.double()])
        want = torch.autograd.grad(outs, [leaves[k] for k in wanted], grads)
        dev = {k: laid(v, k).cuda().requires_grad_(k in wanted) if v is not None else None for k, v in t.items()}
        outs = residual_norm(dev["x"], dev["residual"], dev["gate"], dev["post"], dev["weight"], dev["bias"], 0.7, norm, 1e-5, bs_last)
        up = [laid(v, "x").cuda() for v in (dr, dn)]
        got = torch.autograd.grad(outs if use_dr else outs[1:], [dev[k] for k in wanted], up if use_dr else up[1:])
    for k, g, w in zip(wanted, got, want):
        w = laid(w, k)
        assert rel(g, w) <= TOL[prec], (k, rel(g, w))
        if k == "gate":
            off = gate_error(g, w, leaves, r, (dr if use_dr else dr * 0, dn), norm)
            assert off <= 1.0, off


def gate_error(g, want, t, r, outs_grads, norm):
    """The largest error of a gate's gradient, of what it may be.  It is a sum of 0.7 D p, both of which are sums and differences
    themselves: p = (x - mean) rho post, D = dr + rho (dv - mean(dv) - v mean(dv v)), v = (r - mean) rho; what is rounded
    are their terms, and a value's size here is that of its terms together."""
    def mean(v):
        return v.mean(1, keepdim=True)

    def normed(v, size):
        m, m_size = (mean(v), mean(size)) if norm == "layer" else (0.0, 0.0)
        rho = (mean((v - m) ** 2) + 1e-5) ** -0.5
        return (v - m) * rho, (size + m_size) * rho, rho

    t = {k: v.detach() for k, v in t.items()}
    dr, dn = (v.double() for v in outs_grads)
    p, p_size = t["x"], t["x"].abs()
    if "post" in t:
        p, p_size, _ = normed(p, p_size)
        p, p_size = p * t["post"], p_size * t["post"].abs()
    gate = t["gate"].repeat_interleave(len(p) // len(t["gate"]), 0)
    v, v_size, rho = normed(r.detach(), t["residual"].abs() + 0.7 * gate.abs() * p_size)
    dv = dn * t["weight"]
    D = dr + rho * (dv - v * mean(dv * v) - (mean(dv) if norm == "layer" else 0))
    D_size = dr.abs() + rho * (dv.abs() + v_size * mean(dv.abs() * v_size) + (mean(dv.abs()) if norm == "layer" else 0))

    def summed(v):
        return 0.7 * v.reshape(want.shape[0], -1, want.shape[1]).sum(1)

    sizes = summed(D_size * p_size)
    assert torch.allclose(summed(D * p), want, rtol=1e-9, atol=1e-9 * float(sizes.max()))
    half = 2.0 ** (torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -14))) - 11) if g.dtype == torch.float16 else 0.0
    return float(((g.double().cpu() - want).abs() / (half + 4e-6 * sizes)).max())


@pytest.mark.parametrize("bs_last", [True, False])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("features,batch,groups", [(96, 60, 60), (97, 60, 4), (384, 5 * 197, 5), (41, 2000, 1000), (768, 1600, 2), (64, 7000, 7),
                                                   (1300, 66, 6), (1299, 2048, 2), (6, 130, 1)])
def test_each_group_has_its_own_gate(features, batch, groups, prec, bs_last):
    for post, norm in ((True, "layer"), (False, "rms")):
        t, dr, dn = operands(features, batch, max(groups, 1), DT[prec], post)
        names = [k for k in ("x", "residual", "gate", "post", "weight", "bias") if t[k] is not None]
        check(t, dr, dn, prec, norm, bs_last, names)


@pytest.mark.parametrize("bs_last", [True, False])
@pytest.mark.parametrize("features", [64, 1200])
def test_gate_alone(features, bs_last):
    """Nobody asks for the gradient of the residual; with and without one of r_out."""
    for use_dr in (True, False):
        t, dr, dn = operands(features, 120, 4, torch.float16, True, seed=1)
        check(t, dr, dn, "fp16", "layer", bs_last, ["gate"], use_dr)


@pytest.mark.parametrize("bs_last", [True, False])
@pytest.mark.parametrize("features", [64, 1200])
def test_gradients_of_the_sum_beyond_the_type(features, bs_last):
    """Gradients of r_out near the largest fp16 number: with what the norm adds they leave fp16, their sums over small x do not."""
    t, dr, dn = operands(features, 240, 3, torch.float16, False, seed=2, x_scale=1e-3, dr_scale=10.0)
    dr = dr.clamp(-1, 1) * 60000
    t["residual"] = t["residual"] * 0.01
    t["x"], dn = t["x"].abs() * dr.sign(), (dr.sign() * 300).half()
    check(t, dr.half(), dn, "fp16", "rms", bs_last, ["gate"])
