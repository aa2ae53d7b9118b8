"""Gated projection (gated_linear, KSGatedLinear): results and gradients against the definition in float64.

Tolerances, relative Frobenius.  fp32: sums of up to 400 products (up to 3000 rows for the weights' gradients) in fp32, 2^-24 a
rounding, random signs: below 1e-6 each; 5e-6.  fp16: rounding the result costs at most 2^-11 of a value (4.9e-4); gradients of
input and parameters are sums over dz, which is rounded before (another 2.1e-4 in the 2-norm): 1e-3."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
TOL = {"fp32": (5e-6, 5e-6), "fp16": (4.9e-4, 1e-3)}


def act64(name, z):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z


def oracle(x, factor, bias, pattern, act, bs_last):
    """On float64 CPU tensors, differentiable."""
    a, b, c, d = pattern
    x = x.t() if bs_last else x
    xs = x.reshape(-1, a, c, d)
    w = factor.reshape(a, d, c, 2, b)
    z = torch.einsum("nacd,adcpb->napbd", xs, w)
    if bias is not None:
        z = z + bias.reshape(a, 2, b, d)
    h = (act64(act, z[:, :, 0]) * z[:, :, 1]).reshape(-1, a * b * d)
    return h.t() if bs_last else h


def inputs(pattern, batch, dtype, bias, bs_last, seed=0):
    a, b, c, d = pattern
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((a * c * d, batch) if bs_last else (batch, a * c * d), generator=g)
    w = torch.randn(a * d * c, 2 * b, generator=g) / math.sqrt(c)
    v = torch.randn(2 * a * b * d, generator=g) * 0.2 if bias else None
    dh = torch.randn((a * b * d, batch) if bs_last else (batch, a * b * d), generator=g)
    return [None if t is None else t.to(dtype) for t in (x, w, v, dh)]


def rel(x, y):
    n = float(torch.linalg.vector_norm(y))
    e = float(torch.linalg.vector_norm(x.double().cpu() - y))
    return e / n if n else e


def check(pattern, batch, prec, act, bias, bs_last):
    from ksmm_amd import gated_linear

    x, w, v, dh = inputs(pattern, batch, DT[prec], bias, bs_last)
    leaves = [t.double().requires_grad_() for t in (x, w, v) if t is not None]
    with torch.enable_grad():
        z = oracle(leaves[0], leaves[1], leaves[2] if bias else None, pattern, act, bs_last)
        want = torch.autograd.grad(z, leaves, dh.double())
    dev = [t.cuda() for t in (x, w, v) if t is not None]
    quiet = gated_linear(dev[0], dev[1], pattern, dev[2] if bias else None, act, bs_last)
    assert rel(quiet, z.detach()) <= TOL[prec][0]
    dev = [t.requires_grad_() for t in dev]
    with torch.enable_grad():
        h = gated_linear(dev[0], dev[1], pattern, dev[2] if bias else None, act, bs_last)
        got = torch.autograd.grad(h, dev, dh.cuda())
    assert torch.equal(h.detach(), quiet)
    for g, t in zip(got, want):
        assert g.dtype == DT[prec] and rel(g, t) <= TOL[prec][1]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", [(1, 64, 48, 2), (2, 32, 64, 1), (1, 40, 96, 3), (1, 48, 32, 4), (1, 17, 19, 2), (2, 33, 50, 6),
                                     (1, 16, 16, 16), (3, 5, 7, 5), (1, 130, 384, 1), (1, 1, 1, 1), (4, 100, 3, 8)])
@pytest.mark.parametrize("batch", [1, 3, 130, 197])
def test_results_and_gradients(pattern, batch, prec, bs_last):
    check(pattern, batch, prec, "silu" if batch % 2 else "gelu", batch != 3, bs_last)


@pytest.mark.parametrize("act", ["silu", "gelu", None])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern,batch,bs_last", [((1, 192, 96, 2), 1500, False), ((2, 128, 64, 1), 2100, False), ((1, 128, 128, 3), 1031, False),
                                                   ((1, 64, 96, 4), 999, False), ((2, 96, 64, 1), 2049, True), ((1, 200, 120, 2), 1777, True)])
def test_larger_batches(pattern, batch, bs_last, prec, act):
    check(pattern, batch, prec, act, True, bs_last)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("pattern,batch,bs_last", [
    ((1, 64, 64, 2), 129, False), ((1, 72, 80, 2), 300, False), ((3, 136, 96, 2), 2000, False), ((1, 8, 64, 2), 9000, False),
    ((1, 128, 64, 1), 1300, False), ((3, 72, 80, 1), 517, False), ((1, 264, 176, 1), 3001, False), ((2, 640, 128, 1), 4500, False),
    ((1, 128, 64, 1), 1304, True), ((3, 72, 80, 2), 520, True), ((1, 264, 176, 1), 3008, True), ((2, 640, 128, 3), 1504, True),
    ((1, 8, 64, 2), 136, True)])
def test_aligned_fp16(pattern, batch, bs_last, bias):
    """The ring of slabs: few and many tiles a workgroup, outputs and rows that end inside a tile, few and many slabs."""
    check(pattern, batch, "fp16", "silu" if bias else "gelu", bias, bs_last)


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern,batch", [((8, 100, 19, 1), 1201), ((4, 100, 21, 2), 1201), ((3, 99, 20, 3), 1201), ((2, 101, 18, 4), 1201),
                                           ((2, 100, 17, 5), 1201), ((2, 72, 20, 6), 1201), ((1, 104, 33, 8), 1201), ((8, 9, 10, 8), 1201),
                                           ((8, 8, 3, 8), 1201), ((2, 104, 64, 4), 1208), ((16, 100, 16, 7), 77), ((24, 200, 64, 4), 40),
                                           ((24, 200, 65, 4), 33), ((40, 128, 64, 2), 48), ((40, 128, 64, 3), 48), ((40, 100, 40, 2), 47)])
def test_work_for_tiles(pattern, batch, prec, bs_last):
    """Enough work for the tiles of every d, at sizes that end inside them; few rows of large factors."""
    check(pattern, batch, prec, "silu", True, bs_last)


@pytest.mark.parametrize("pattern,batch,bs_last", [((40, 65, 6, 5), 300, True), ((60, 65, 6, 2), 1201, False), ((110, 65, 5, 1), 1201, False)])
def test_many_tiles_fp32(pattern, batch, bs_last):
    check(pattern, batch, "fp32", "gelu", True, bs_last)


@pytest.mark.parametrize("bs_last", [False, True])
def test_no_rows_and_more_axes(bs_last):
    from ksmm_amd import GatedKernel, KSGatedLinear

    layer = KSGatedLinear((2, 24, 8, 2), bs_last=bs_last)
    x = torch.randn((32, 0) if bs_last else (0, 32), device="cuda").half().requires_grad_()
    with torch.enable_grad():
        h = layer(x)
        assert tuple(h.shape) == ((96, 0) if bs_last else (0, 96))
        h.sum().backward()
    assert x.grad.shape == x.shape and not layer.factor.grad.any() and not layer.bias.grad.any()
    x = torch.randn((32, 3, 5) if bs_last else (3, 5, 32), device="cuda").half()
    h = layer(x)
    flat = GatedKernel.forward(x.reshape(32, 15) if bs_last else x.reshape(15, 32), layer.factor, layer.pattern, layer.bias, "silu", bs_last)
    assert tuple(h.shape) == ((96, 3, 5) if bs_last else (3, 5, 96)) and torch.equal(h.reshape(flat.shape), flat)


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("batch", [5, 300])
def test_tensors_off_the_vector_and_other_streams(batch, bs_last):
    """Operands that start one element behind a boundary give the bits of those that do not; so does another stream."""
    from ksmm_amd import GatedKernel

    pattern = (2, 48, 40, 2)
    x, w, v, dh = (t.cuda() for t in inputs(pattern, batch, torch.float16, True, bs_last))

    def moved(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)

    h = GatedKernel.forward(x, w, pattern, v, "silu", bs_last)
    out = torch.empty(h.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(h.shape)
    assert torch.equal(GatedKernel.forward(moved(x), moved(w), pattern, moved(v), "silu", bs_last, out=out), h)
    grads = GatedKernel.backward(dh, x, w, pattern, v, "silu", bs_last)
    again = GatedKernel.backward(moved(dh), moved(x), moved(w), pattern, moved(v), "silu", bs_last)
    assert all(rel(a, g.double().cpu()) <= 1e-3 for a, g in zip(again, grads))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = GatedKernel.forward(x, w, pattern, v, "silu", bs_last)
        g2 = GatedKernel.backward(dh, x, w, pattern, v, "silu", bs_last)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(there, h) and all(torch.equal(a, b) for a, b in zip(g2, grads))


def test_infinities_and_nan_stay_in_their_rows():
    from ksmm_amd import GatedKernel

    pattern = (1, 96, 64, 2)
    for bs_last in (False, True):
        x, w, v, _ = (t.cuda() for t in inputs(pattern, 300, torch.float16, True, bs_last))
        clean = GatedKernel.forward(x, w, pattern, v, "silu", bs_last)
        rows = x if not bs_last else x.t()
        rows[7, 3], rows[299, 0] = float("nan"), float("inf")
        h = GatedKernel.forward(x, w, pattern, v, "silu", bs_last)
        bad = ~torch.isfinite(h if not bs_last else h.t()).all(1)
        assert bad.nonzero().flatten().tolist() == [7, 299]
        same = (h == clean) if not bs_last else (h == clean).t()
        assert same[~bad].all()


def test_gradient_against_differences():
    """<dL, v> of the kernel's gradients against (L(p + e v) - L(p - e v)) / 2e of its results, fp32.  The quotient's own error:
    e^2 of the third derivative (about 1e-4 of the value), and fp32 rounding of L's terms, 1e-7 sqrt(terms) / e."""
    from ksmm_amd import gated_linear

    pattern, e = (2, 24, 32, 3), 1e-2
    x, w, v, dh = (t.cuda() for t in inputs(pattern, 64, torch.float32, True, False, seed=3))
    for act in ("silu", "gelu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, v)]
        with torch.enable_grad():
            grads = torch.autograd.grad(gated_linear(leaves[0], leaves[1], pattern, leaves[2], act), leaves, dh)
        g = torch.Generator(device="cuda").manual_seed(1)
        for i, t in enumerate((x, w, v)):
            step = torch.randn(t.shape, generator=g, device="cuda") * t.std()
            sides = []
            for sign in (1, -1):
                p = [x, w, v]
                p[i] = t + sign * e * step
                sides.append((gated_linear(p[0], p[1], pattern, p[2], act).double() * dh.double()).sum())
            slope, want = float((grads[i].double() * step.double()).sum()), float(sides[0] - sides[1]) / (2 * e)
            scale = float(torch.linalg.vector_norm(grads[i].double()) * torch.linalg.vector_norm(step.double()) / math.sqrt(t.numel()))
            assert abs(slope - want) <= 2e-3 * scale, (act, i, slope, want)


def test_captured_calls_replay():
    from ksmm_amd import GatedKernel

    pattern = (1, 96, 64, 2)
    x, w, v, dh = (t.cuda() for t in inputs(pattern, 260, torch.float16, True, False))

    def both():
        return [GatedKernel.forward(x, w, pattern, v), *GatedKernel.backward(dh, x, w, pattern, v)]

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(3):
        x.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both())), i


def test_refusals():
    from ksmm_amd import GatedKernel, KSGatedLinear, gated_linear

    pattern = (2, 8, 4, 2)
    x, w, v, dh = (t.cuda() for t in inputs(pattern, 6, torch.float16, True, False))
    for error, call in [
        (RuntimeError, lambda: gated_linear(x.cpu(), w, pattern)),
        (RuntimeError, lambda: gated_linear(x, w.cpu(), pattern)),
        (RuntimeError, lambda: gated_linear(x.t().contiguous().t(), w, pattern)),
        (RuntimeError, lambda: gated_linear(x, w.float(), pattern)),
        (RuntimeError, lambda: gated_linear(x, w, pattern, bias=v.float())),
        (ValueError, lambda: gated_linear(x, w, pattern, bias=v[:-1].contiguous())),
        (ValueError, lambda: gated_linear(x, w[:, :-1].contiguous(), pattern)),
        (ValueError, lambda: gated_linear(x[:, :-1].contiguous(), w, pattern)),
        (ValueError, lambda: gated_linear(x, w, pattern, act="relu")),
        (ValueError, lambda: gated_linear(x, w, (2, 0, 4, 2))),
        (AssertionError, lambda: gated_linear(x.bfloat16(), w.bfloat16(), pattern)),
        (ValueError, lambda: GatedKernel.forward(x, w, pattern, out=x)),
        (ValueError, lambda: GatedKernel.backward(dh[:-1], x, w, pattern)),
        (AssertionError, lambda: KSGatedLinear(pattern, dtype=torch.float8_e4m3fn)),
    ]:
        with pytest.raises(error):
            call()
