"""Gated projection, value by value: activations far from zero, where the result is small and the other projection is large.

One column of weights and one of x are chosen so that every gate and every `up` is an fp16 number that the sums give exactly.
fp16 results are rounded once, from fp32 values good to 1e-5 (the activation's own error; half a step is at least 2.4e-4 of a
value): every value is the nearest fp16 number or its neighbour, one step off at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def fp16_steps(x, want):
    """How far x is from want, in steps between neighbouring fp16 numbers there."""
    power = torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -14)))
    return (x.double() - want).abs() / 2 ** (power - 10)


def operands(n, b, bs_last):
    """z0[row, :] = gates[row], z1[:, col] = ups[col]."""
    gates = torch.linspace(-8, 0.5, n).half()
    ups = torch.logspace(-1, 4.5, b).half()
    x, w = torch.zeros(n, 64), torch.zeros(64, 2 * b)
    x[:, 0], x[:, 1] = gates.float(), 1.0
    w[0, :b], w[1, b:] = 1.0, ups.float()
    return gates, ups, (x.t() if bs_last else x).contiguous().half().cuda(), w.half().cuda()


def act64(name, z):
    return z / (1 + torch.exp(-z)) if name == "silu" else z * torch.special.erfc(-z / 2 ** 0.5) / 2


def slope64(name, z):
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.special.erfc(-z / 2 ** 0.5) / 2 + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5


# few rows; tiles that go through registers (rows or outputs that no vector divides); the ring of slabs
SHAPES = [(30, 64, False), (30, 64, True), (2049, 72, True), (2048, 75, False), (2048, 64, False), (2048, 64, True), (12544, 768, False)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n,b,bs_last", SHAPES)
def test_every_value_is_the_nearest_or_its_neighbour(n, b, bs_last, act):
    from ksmm_amd import gated_linear

    gates, ups, x, w = operands(n, b, bs_last)
    h = gated_linear(x, w, (1, b, 64, 1), act=act, bs_last=bs_last)
    want = act64(act, gates.double())[:, None] * ups.double()[None, :]
    off = fp16_steps((h.t() if bs_last else h).cpu(), want)
    worst = int(off.argmax())
    assert off.max() <= 1, (float(off.max()), float(gates[worst // b]), float(ups[worst % b]))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n,b,bs_last", SHAPES)
def test_every_gradient_of_the_gate(n, b, bs_last, act):
    """dh in one output only: dx of the gate's input is that output's dz, dh * up * act'.  Around the slope's zero the two terms
    of act' cancel: 2^-22 of the terms, which are below one, on top."""
    from ksmm_amd import gated_linear

    gates, ups, x, w = operands(n, b, bs_last)
    dh = torch.zeros(n, b)
    dh[:, b // 2] = 0.5
    x.requires_grad_()
    with torch.enable_grad():
        h = gated_linear(x, w, (1, b, 64, 1), act=act, bs_last=bs_last)
        g, = torch.autograd.grad(h, x, (dh.t() if bs_last else dh).contiguous().half().cuda())
    scale = 0.5 * float(ups[b // 2])
    want = scale * slope64(act, gates.double())
    got = (g[0] if bs_last else g[:, 0]).cpu()
    off = (got.double() - want).abs() - 2 ** -22 * scale
    assert (fp16_steps(want + off.clamp_min(0), want) <= 1).all()


@pytest.mark.parametrize("n,b,bs_last", SHAPES[:6])
def test_gradients_of_the_projections_beyond_the_type_are_seen(n, b, bs_last):
    """The gradients of both projections are held in the tensors' type on their way to the sums: one beyond the largest fp16 number is
    an infinity, in every gradient that it goes into and in no other.  (Mixed-precision training scales the loss by that.)"""
    from ksmm_amd import gated_linear

    x, w, dh = torch.zeros(n, 64), torch.zeros(64, 2 * b), torch.zeros(n, b)
    x[:, 0], x[:, 1] = 4.0, 1.0
    w[0, :b], w[1, b:] = 1.0, 1000.0
    dh[:, 3], dh[n // 2, 3] = 1.0, 100.0  # dz of the gate: 1.05e3, and 1.05e5
    x, dh = ((t.t() if bs_last else t).contiguous().half().cuda() for t in (x, dh))
    leaves = [x.requires_grad_(), w.half().cuda().requires_grad_()]
    with torch.enable_grad():
        dx, dw = torch.autograd.grad(gated_linear(*leaves, (1, b, 64, 1), bs_last=bs_last), leaves, dh)
    dx = dx.t() if bs_last else dx
    assert not dx[n // 2, 0].isfinite() and dx[:n // 2].isfinite().all() and dx[n // 2 + 1:].isfinite().all()
    assert not dw[0, 3].isfinite() and dw[:, :3].isfinite().all() and dw[:, 4:].isfinite().all()
