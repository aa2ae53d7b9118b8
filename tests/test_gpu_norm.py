"""Residual norm (residual_norm, ResidualNorm): results and gradients against the definition in float64.

Tolerances, relative Frobenius.  fp32: a row's sums and a dozen roundings of 2^-24: below 1e-6; sums over rows with random signs
too: 5e-6.  fp16: every result is rounded once, from fp32: at most 2^-11 of a value, 4.9e-4, and at most 2^-25 of it
where it is subnormal (the gradient of a row of one feature is 1e-7)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
TOL = {"fp32": 5e-6, "fp16": 4.9e-4}
NAMES = ("x", "residual", "gate", "post_weight", "weight", "bias")


def oracle(t, alpha, norm, eps, bs_last):
    """On float64 CPU tensors, differentiable: (r_out, n_out)."""
    rows = {k: (v.t() if bs_last and k in ("x", "residual") else v) for k, v in t.items()}

    def normed(v):
        if norm == "layer":
            v = v - v.mean(1, keepdim=True)
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)

    r = rows["residual"]
    if rows.get("x") is not None:
        p = rows["x"]
        if rows.get("post_weight") is not None:
            p = normed(p) * rows["post_weight"]
        if rows.get("gate") is not None:
            g = rows["gate"].reshape(-1, r.shape[1])
            p = p * g.repeat_interleave(r.shape[0] // g.shape[0], 0)
        r = r + alpha * p
    n = normed(r)
    if rows.get("weight") is not None:
        n = n * rows["weight"]
    if rows.get("bias") is not None:
        n = n + rows["bias"]
    return (r.t(), n.t()) if bs_last else (r, n)


def tensors(features, batch, dtype, bs_last, groups=1, post=True, gate=True, affine=True, x=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (features, batch) if bs_last else (batch, features)

    def make(*s, scale=1.0, mean=0.0):
        return (torch.randn(s, generator=g) * scale + mean).to(dtype)

    t = {"x": make(*shape, mean=0.3) if x else None, "residual": make(*shape, mean=-0.2),
         "gate": make(*((groups, features) if groups > 1 else (features,)), scale=0.3, mean=0.5) if gate and x else None,
         "post_weight": make(features, scale=0.1, mean=1.0) if post and x else None,
         "weight": make(features, scale=0.1, mean=1.0) if affine else None, "bias": make(features, scale=0.1) if affine else None}
    return t, make(*shape), make(*shape)


def rel(x, y):
    n = float(torch.linalg.vector_norm(y))
    e = float(torch.linalg.vector_norm(x.double().cpu() - y))
    if x.dtype == torch.float16:
        e = max(0.0, e - 2 ** -25 * math.sqrt(y.numel()))
    return e / n if n else e


def check(prec, bs_last, t, dr, dn, norm="rms", alpha=0.7, eps=1e-5, grads="both"):
    from ksmm_amd import residual_norm

    tol = TOL[prec]
    want_leaves = {k: v.double().requires_grad_() for k, v in t.items() if v is not None}
    with torch.enable_grad():
        want_r, want_n = oracle(want_leaves, alpha, norm, eps, bs_last)
        outs, gs = [], []
        if grads != "n" and t["x"] is not None:
            outs.append(want_r)
            gs.append(dr.double())
        if grads != "r":
            outs.append(want_n)
            gs.append(dn.double())
        want = torch.autograd.grad(outs, list(want_leaves.values()), gs, allow_unused=True)
    dev = {k: v.cuda() if v is not None else None for k, v in t.items()}
    r, n = residual_norm(*dev.values(), alpha, norm, eps, bs_last)
    assert rel(r, want_r.detach()) <= tol and rel(n, want_n.detach()) <= tol
    leaves = {k: v.requires_grad_() for k, v in dev.items() if v is not None}
    with torch.enable_grad():
        r2, n2 = residual_norm(*dev.values(), alpha, norm, eps, bs_last)
        outs = ([r2] if grads != "n" and t["x"] is not None else []) + ([n2] if grads != "r" else [])
        got = torch.autograd.grad(outs, list(leaves.values()), [g.cuda().to(r.dtype) for g in gs], allow_unused=True)
    assert torch.equal(r2, r) and torch.equal(n2, n)
    for name, g, w in zip(leaves, got, want):
        if w is None:  # (not reached: nothing, or zeros)
            assert g is None or not g.any(), name
        else:
            assert rel(g, w) <= tol, (name, rel(g, w))


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("features", [1, 7, 64, 100, 513, 768, 1030, 2500, 5000])
@pytest.mark.parametrize("batch", [1, 5, 67])
def test_results_and_gradients(features, batch, prec, bs_last):
    t, dr, dn = tensors(features, batch, DT[prec], bs_last)
    check(prec, bs_last, t, dr, dn, norm="layer" if features > 1 and batch != 5 else "rms")


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("features,batch,groups", [(96, 60, 60), (96, 60, 4), (384, 5 * 197, 5), (40, 2000, 1000), (768, 1600, 2)])
def test_gates_of_groups(features, batch, groups, bs_last):
    for prec in ("fp32", "fp16"):
        for post in (False, True):
            t, dr, dn = tensors(features, batch, DT[prec], bs_last, groups=groups, post=post)
            if prec == "fp16" and bs_last:
                # gates of groups are summed over dr as it is stored: its rounding counts once more
                t["gate"] = t["gate"][:1].expand(groups, features).contiguous()
            check(prec, bs_last, t, dr, dn, norm="layer") if not (prec == "fp16" and bs_last) else check_group_fp16(t, dr, dn)


def check_group_fp16(t, dr, dn):
    from ksmm_amd import residual_norm

    want_leaves = {k: v.double().requires_grad_() for k, v in t.items() if v is not None}
    with torch.enable_grad():
        outs = oracle(want_leaves, 0.7, "layer", 1e-5, True)
        want = torch.autograd.grad(outs, list(want_leaves.values()), [dr.double(), dn.double()])
        leaves = {k: v.cuda().requires_grad_() if v is not None else None for k, v in t.items()}
        out = residual_norm(*leaves.values(), 0.7, "layer", 1e-5, True)
        got = torch.autograd.grad(out, [v for v in leaves.values() if v is not None], [dr.cuda(), dn.cuda()])
    for name, g, w in zip(want_leaves, got, want):
        assert rel(g, w) <= (1e-3 if name == "gate" else TOL["fp16"]), name


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
def test_each_form(prec, bs_last):
    for kwargs in ({"x": False}, {"x": False, "affine": False}, {"gate": False}, {"post": False, "gate": False}, {"affine": False}):
        for grads in ("both", "r", "n"):
            if kwargs.get("x") is False and grads == "r":
                continue
            t, dr, dn = tensors(200, 37, DT[prec], bs_last, **kwargs)
            check(prec, bs_last, t, dr, dn, grads=grads)


@pytest.mark.parametrize("bs_last", [False, True])
def test_many_rows(bs_last):
    for features, batch in ((384, 6501), (32, 9001), (1536, 2000)):
        t, dr, dn = tensors(features, batch, torch.float16, bs_last)
        check("fp16", bs_last, t, dr, dn, norm="layer")


def test_the_addition_alone_no_rows_and_the_module():
    from ksmm_amd import ResidualNorm, residual_norm

    t, _, _ = tensors(48, 9, torch.float32, False, affine=False)
    dev = {k: v.cuda() if v is not None else None for k, v in t.items()}
    r, n = residual_norm(dev["x"], dev["residual"], dev["gate"], dev["post_weight"], need_norm=False)
    want = oracle({k: v.double() for k, v in t.items() if v is not None}, 1.0, "rms", 1e-6, False)[0]
    assert n is None and rel(r, want) <= TOL["fp32"]
    layer = ResidualNorm(48, "layer", post=True, gate=True, dtype=torch.float32)
    x = torch.randn(0, 48, device="cuda", requires_grad=True)
    with torch.enable_grad():
        r, n = layer(x, torch.randn(0, 48, device="cuda"))
        assert tuple(r.shape) == tuple(n.shape) == (0, 48)
        (r.sum() + n.sum()).backward()
    assert x.grad.shape == x.shape and all(not p.grad.any() for p in layer.parameters())
    out = layer(torch.randn(2, 3, 48, device="cuda"), torch.randn(2, 3, 48, device="cuda"))
    assert tuple(out[0].shape) == tuple(out[1].shape) == (2, 3, 48)


@pytest.mark.parametrize("bs_last", [False, True])
def test_rows_of_zeros_of_one_value_and_of_huge_ones(bs_last):
    """A row of zeros is normed to zeros, one of equal values too where a mean is taken; 60000 in fp16 does not overflow; a row
    with NaN spoils itself alone."""
    from ksmm_amd import residual_norm

    h = 300
    r = torch.randn(40, h, device="cuda").half()
    r[3], r[4], r[5], r[6, 17] = 0.0, 2.5, 60000.0, float("nan")
    r = r.t().contiguous() if bs_last else r
    for norm in ("rms", "layer"):
        n = residual_norm(None, r, norm=norm, bs_last=bs_last)[1]
        n = n.t() if bs_last else n
        assert not n[3].any() and n[6].isnan().all() and n[7:].isfinite().all() and n[:6].isfinite().all()
        if norm == "layer":
            assert n[4].abs().max() < 1e-3 and n[5].abs().max() < 1e-3
        else:
            assert (n[4].float() - 1).abs().max() < 1e-3 and (n[5].float() - 1).abs().max() < 1e-3


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("features", [96, 101])
def test_tensors_off_the_vector_other_streams_and_graphs(features, bs_last):
    from ksmm_amd import NormKernel

    t, dr, dn = tensors(features, 77, torch.float16, bs_last)
    dev = [v.cuda() for v in t.values()]

    def moved(v):
        room = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
        room[1:] = v.reshape(-1)
        return room[1:].view(v.shape)

    def both(args, dr, dn):
        r, n, stats = NormKernel.forward(*args, bs_last=bs_last, need_stats=True)
        return [r, n, *NormKernel.backward(dr, dn, stats, *args, bs_last=bs_last)]

    dr, dn = dr.cuda(), dn.cuda()
    here = both(dev, dr, dn)
    assert all(torch.equal(a, b) for a, b in zip(both([moved(v) for v in dev], moved(dr), moved(dn)), here))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = both(dev, dr, dn)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(there, here))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(dev, dr, dn)
    for i in range(3):
        dev[0].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both(dev, dr, dn))), i


def test_gradient_against_differences():
    """<dL, v> against (L(p + e v) - L(p - e v)) / 2e of the kernel's fp32 results; the quotient itself is good to about 1e-3."""
    from ksmm_amd import residual_norm

    e = 1e-2
    for norm in ("rms", "layer"):
        t, dr, dn = tensors(130, 44, torch.float32, False, groups=4, seed=2)
        dev = [v.cuda() for v in t.values()]
        dr, dn = dr.cuda(), dn.cuda()
        leaves = [v.clone().requires_grad_() for v in dev]
        with torch.enable_grad():
            grads = torch.autograd.grad(residual_norm(*leaves, 0.7, norm), leaves, [dr, dn])
        g = torch.Generator(device="cuda").manual_seed(1)
        for i, v in enumerate(dev):
            step, sides = torch.randn(v.shape, generator=g, device="cuda"), []
            for sign in (1, -1):
                p = list(dev)
                p[i] = v + sign * e * step
                r, n = residual_norm(*p, 0.7, norm)
                sides.append((r.double() * dr.double()).sum() + (n.double() * dn.double()).sum())
            slope, want = float((grads[i].double() * step.double()).sum()), float(sides[0] - sides[1]) / (2 * e)
            scale = float(torch.linalg.vector_norm(grads[i].double()) * torch.linalg.vector_norm(step.double()) / math.sqrt(v.numel()))
            assert abs(slope - want) <= 2e-3 * scale, (norm, NAMES[i], slope, want)


def test_refusals():
    from ksmm_amd import KSFeedForward, ResidualNorm, residual_norm

    x, r, w = torch.randn(6, 32, device="cuda"), torch.randn(6, 32, device="cuda"), torch.ones(32, device="cuda")
    for error, call in [
        (RuntimeError, lambda: residual_norm(x.cpu(), r)),
        (RuntimeError, lambda: residual_norm(x, r.cpu())),
        (RuntimeError, lambda: residual_norm(x.half(), r)),
        (RuntimeError, lambda: residual_norm(x, r.t().contiguous().t())),
        (ValueError, lambda: residual_norm(x[:5], r)),
        (ValueError, lambda: residual_norm(None, r, gate=w)),
        (ValueError, lambda: residual_norm(None, r, post_weight=w)),
        (ValueError, lambda: residual_norm(x, r, gate=torch.ones(4, 32, device="cuda"))),
        (ValueError, lambda: residual_norm(x, r, weight=w[:31].contiguous())),
        (ValueError, lambda: residual_norm(x, r, norm="batch")),
        (ValueError, lambda: residual_norm(None, r, need_norm=False)),
        (AssertionError, lambda: residual_norm(None, r.bfloat16())),
        (RuntimeError, lambda: residual_norm(None, torch.ones(2, 17000, device="cuda"))),
        (ValueError, lambda: ResidualNorm(32, "batch")),
        (ValueError, lambda: KSFeedForward((1, 64, 32, 1), [(1, 32, 32, 1)])),
    ]:
        with pytest.raises(error):
            call()


def test_second_derivatives_are_refused_and_saved_tensors_guarded():
    from ksmm_amd import gated_linear, residual_norm

    with torch.enable_grad():
        r = torch.randn(5, 32, device="cuda", requires_grad=True)
        n = residual_norm(None, r)[1]
        g, = torch.autograd.grad(n.sum(), r, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
        x = torch.randn(5, 32, device="cuda", requires_grad=True)
        w = torch.randn(32, 16, device="cuda", requires_grad=True)
        h = gated_linear(x, w, (1, 8, 32, 1))
        g, = torch.autograd.grad(h.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
        h = gated_linear(x, w, (1, 8, 32, 1))
        with torch.no_grad():
            w.add_(1.0)
        with pytest.raises(RuntimeError):  # changed in between
            h.sum().backward()


def test_through_ctypes_gives_the_same(monkeypatch):
    """Where the CPython module is not there, the same kernels run through ctypes and Python autograd nodes."""
    from ksmm_amd import _lib, gated_linear, residual_norm

    t, dr, dn = tensors(96, 50, torch.float16, False, groups=5)
    dev = [v.cuda().requires_grad_() for v in t.values()]
    w = torch.randn(96, 2 * 48, device="cuda").half().requires_grad_()

    def all_of():
        with torch.enable_grad():
            r, n = residual_norm(*dev, 0.7)
            h = gated_linear(n, w, (1, 48, 96, 1), act="gelu")
            return [r, n, h, *torch.autograd.grad([r, h], [*dev, w], [dr.cuda(), h.detach()])]

    native = all_of()
    assert native[1].grad_fn.name() == "ResidualNormBackward" and native[2].grad_fn.name() == "GatedLinearBackward"
    monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    python = all_of()
    assert "ResidualNormFunction" in python[1].grad_fn.name()
    # (gradients of 96 x 96 weights of size one overflow now and then: NaN in both)
    assert all(torch.allclose(a, b, rtol=0, atol=0, equal_nan=True) for a, b in zip(native, python))


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("features,batch,groups,post", [(1025, 130, 1, True), (1300, 66, 6, True), (1300, 66, 66, False), (2049, 2048, 1, False),
                                                        (1300, 2100, 1, True), (1300, 2100, 4, False)])
def test_many_features_of_few_and_of_many_columns(features, batch, groups, post, prec):
    t, dr, dn = tensors(features, batch, DT[prec], True, groups, post=post)
    check(prec, True, t, dr, dn, norm="layer" if post else "rms")


@pytest.mark.parametrize("grads", ["n", "r"])
def test_many_features_one_gradient(grads):
    t, dr, dn = tensors(1200, 70, torch.float32, True)
    check("fp32", True, t, dr, dn, norm="layer", grads=grads)


def test_many_features_without_a_branch():
    t, dr, dn = tensors(1200, 70, torch.float32, True, x=False)
    check("fp32", True, t, dr, dn)


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("features", [8193, 12000, 16384])
def test_widest_rows(features, prec):
    t, dr, dn = tensors(features, 13, DT[prec], False)
    check(prec, False, t, dr, dn, norm="layer")


@pytest.mark.parametrize("bs_last", [False, True])
def test_offsets_beyond_31_bits(bs_last):
    """The last rows of 2.2e9 values are those of a call on them alone."""
    from ksmm_amd import residual_norm

    features, batch, last = 1100, 2_000_001, 8195
    shape = (features, batch) if bs_last else (batch, features)
    x, r, dn = (torch.empty(shape, dtype=torch.float16, device="cuda").normal_() for _ in range(3))
    w = torch.ones(features, dtype=torch.float16, device="cuda")
    tail = [(t[:, -last:] if bs_last else t[-last:]).contiguous() for t in (x, r, dn)]

    def results(x, r, dn):
        x, r = x.requires_grad_(), r.requires_grad_()
        with torch.enable_grad():
            out = residual_norm(x, r, None, w, w, None, 0.5, bs_last=bs_last)
            return [t.detach() for t in out] + list(torch.autograd.grad(out[1], (x, r), dn))

    for a, b in zip(results(x, r, dn), results(*tail)):
        assert torch.equal(a[:, -last:] if bs_last else a[-last:], b)
