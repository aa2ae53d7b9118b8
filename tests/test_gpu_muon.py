"""Orthogonalised updates (orthogonalize, muon_update, KSMuon) against the steps in float64.

Tolerances, relative Frobenius.  The polynomial's slope at zero is 3.4445 and at most that in size between there and one, so that
rounding errors of a step grow at most 3.4445 times in each that follows; in the 2-norm the largest singular values, which hardly grow them,
dominate: fp32 products of up to 600 terms, five steps: 1e-5.  fp16: one rounding of the result: 4.9e-4."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
TOL = {"fp32": 1e-5, "fp16": 4.9e-4}
P = (3.4445, -4.7750, 2.0315)


def orthogonal64(u, pattern, parts, steps=5, eps=1e-7, coefficients=P):
    a, b, c, d = pattern
    x = u.double().reshape(a * d, c, parts, b).transpose(1, 2)
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    p0, p1, p2 = coefficients
    for _ in range(steps):
        g = x @ x.mT
        x = p0 * x + (p1 * g + p2 * g @ g) @ x
    return x.transpose(1, 2).reshape(u.shape)


def rel(x, y):
    n = float(torch.linalg.vector_norm(y))
    e = float(torch.linalg.vector_norm(x.double().cpu() - y))
    return e / n if n else e


def random_factor(pattern, parts, dtype=torch.float32, scale=1.0, seed=0):
    a, b, c, d = pattern
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(a * d * c, parts * b, generator=g) * scale).to(dtype)


PATTERNS = [(1, 1, 1, 1), (3, 1, 5, 2), (2, 16, 16, 3), (5, 9, 4, 2), (1, 40, 24, 3), (6, 64, 64, 1), (2, 17, 100, 1), (1, 300, 20, 2),
            (1, 128, 128, 2), (1, 96, 192, 1), (1, 160, 130, 2), (1, 33, 600, 1), (1, 260, 140, 1), (1, 512, 64, 1), (40, 16, 16, 3)]


@pytest.mark.parametrize("parts", [1, 2, 3])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", PATTERNS)
def test_blocks_become_orthogonal(pattern, prec, parts):
    from ksmm_amd import orthogonalize

    u = random_factor(pattern, parts, DT[prec], 0.01)
    assert rel(orthogonalize(u.cuda(), pattern, parts), orthogonal64(u, pattern, parts)) <= TOL[prec]


@pytest.mark.parametrize("steps", [1, 2, 8])
@pytest.mark.parametrize("pattern", [(2, 48, 32, 1), (1, 200, 150, 1)])
def test_steps_and_coefficients(pattern, steps):
    """Eight steps of the cubic (1.5, -0.5) converge: X X^T is the identity up to fp32."""
    from ksmm_amd import orthogonalize

    u = random_factor(pattern, 1)
    for p in (P, (1.5, -0.5, 0.0)):
        got = orthogonalize(u.cuda(), pattern, steps=steps, coefficients=p)
        # (errors grow with the steps: 3.4445 a step at most)
        assert rel(got, orthogonal64(u, pattern, 1, steps, coefficients=p)) <= TOL["fp32"] * max(1.0, 3.4445 ** (steps - 5))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern,parts", [((2, 48, 32, 1), 1), ((1, 20, 50, 2), 2), ((1, 200, 150, 1), 2)])
def test_update(pattern, parts, prec, nesterov):
    from ksmm_amd import muon_update

    a, b, c, d = pattern
    g, m, w = random_factor(pattern, parts, DT[prec], 0.01, 1), random_factor(pattern, parts, scale=0.03, seed=2), random_factor(pattern, parts, DT[prec], 0.2, 3)
    beta, lr, decay = 0.9, 0.05, 0.1
    m64 = beta * m.double() + g.double()
    u = g.double() + beta * m64 if nesterov else m64
    step = lr * math.sqrt(max(1, b / c)) * orthogonal64(u, pattern, parts)
    dev = [t.cuda() for t in (w, g, m)]
    how = dict(parts=parts, lr=lr, beta=beta, weight_decay=decay, nesterov=nesterov)
    w1, m1 = muon_update(*dev, pattern, **how)
    assert all(torch.equal(t.cpu(), o) for t, o in zip(dev, (w, g, m)))
    # (the rounding of the weights, and the error of the step)
    tol = TOL[prec] if prec == "fp16" else 1e-6
    assert rel(m1, m64) <= 1e-6 and rel(w1, (1 - lr * decay) * w.double() - step) <= tol
    master = (torch.randn(w.shape, generator=torch.Generator().manual_seed(4)) * 0.2).cuda()
    want = (1 - lr * decay) * master.double().cpu() - step
    w2, m2 = muon_update(*dev, pattern, master=master, inplace=True, **how)
    assert w2.data_ptr() == dev[0].data_ptr() and m2.data_ptr() == dev[2].data_ptr()
    assert torch.equal(m2, m1) and rel(master, want) <= 1e-6 and torch.equal(w2, master.to(w2.dtype))


@pytest.mark.parametrize("pattern", [(3, 32, 16, 1), (2, 150, 150, 1)])
def test_zeros_and_extremes(pattern):
    """A block of zeros stays zero, one of 1e-20 or 1e15 becomes orthogonal, one with a NaN spoils itself alone."""
    from ksmm_amd import orthogonalize

    a, b, c, d = pattern
    u = random_factor(pattern, 1)
    clean = orthogonalize(u.cuda(), pattern)
    u[:c] = 0.0
    got = orthogonalize(u.cuda(), pattern)
    assert not got[:c].any() and torch.equal(got[c:], clean[c:])
    u[1, 1] = float("nan")
    got = orthogonalize(u.cuda(), pattern)
    assert got[:c].isnan().any() and torch.equal(got[c:], clean[c:])
    for scale in (1e-15, 1e15):
        v = random_factor(pattern, 1) * scale
        assert rel(orthogonalize(v.cuda(), pattern, eps=0.0), orthogonal64(v, pattern, 1, eps=0.0)) <= TOL["fp32"]


def test_streams_alignment_and_graphs():
    from ksmm_amd import muon_update

    for pattern in ((2, 48, 32, 1), (1, 200, 150, 1)):
        g, m, w = random_factor(pattern, 1, torch.float16, 0.01, 1).cuda(), random_factor(pattern, 1, seed=2).cuda(), random_factor(pattern, 1, torch.float16, 0.2, 3).cuda()
        here = muon_update(w, g, m, pattern)

        def moved(v):
            room = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
            room[1:] = v.reshape(-1)
            return room[1:].view(v.shape)

        assert all(torch.equal(x, y) for x, y in zip(muon_update(moved(w), moved(g), moved(m), pattern), here))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            there = muon_update(w, g, m, pattern)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(x, y) for x, y in zip(there, here))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = muon_update(w, g, m, pattern)
        for i in range(3):
            g.mul_(-0.5)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, muon_update(w, g, m, pattern))), i


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
def test_block_is_trained(prec):
    """A feed-forward block learns a target: gated projection, KSLinear and norms with their gradients, KSMuon on the factors; the
    loss falls below a third in 40 steps."""
    from ksmm_amd import KSFeedForward, KSMuon

    torch.manual_seed(0)
    block = KSFeedForward((1, 64, 16, 2), [(2, 16, 64, 1)], dtype=DT[prec], bias=True)
    assert {tuple(f[1:]) for f in KSMuon.factors_of(block)} == {((1, 64, 16, 2), 2), ((2, 16, 64, 1), 1)}
    opt, rest = KSMuon(block, lr=0.02), torch.optim.SGD(KSMuon.others(block), lr=0.02)
    assert len(KSMuon.others(block)) + 2 == len(list(block.parameters()))
    r = torch.randn(256, 32, device="cuda").to(DT[prec])
    target = (r.float() + torch.tanh(r.float().roll(1, 1))).to(DT[prec])
    losses = []
    with torch.enable_grad():
        for _ in range(40):
            _, out = block(block.begin(r), r)
            loss = (out.float() - target.float()).square().mean()
            opt.zero_grad()
            rest.zero_grad()
            loss.backward()
            opt.step()
            rest.step()
            losses.append(float(loss.detach()))
    assert losses[-1] < losses[0] / 3, losses
    if prec == "fp16":
        for p, state in opt.state.items():
            assert torch.equal(p.detach(), state["master"].half())


def test_refusals():
    from ksmm_amd import KSMuon, muon_update, orthogonalize

    pattern = (2, 8, 4, 2)
    g = random_factor(pattern, 1).cuda()
    for error, call in [
        (RuntimeError, lambda: orthogonalize(g.cpu(), pattern)),
        (RuntimeError, lambda: orthogonalize(g.t().contiguous().t(), pattern)),
        (ValueError, lambda: orthogonalize(g, pattern, parts=2)),
        (ValueError, lambda: orthogonalize(g, (2, 8, 4, 1))),
        (ValueError, lambda: orthogonalize(g, pattern, steps=0)),
        (ValueError, lambda: orthogonalize(g, pattern, coefficients=(1.5, -0.5))),
        (AssertionError, lambda: orthogonalize(g.bfloat16(), pattern)),
        (RuntimeError, lambda: muon_update(g.half(), g, g, pattern)),
        (ValueError, lambda: muon_update(g, g, g.half(), pattern)),
        (ValueError, lambda: muon_update(g, g, g[:-1], pattern)),
        (ValueError, lambda: muon_update(g, g, g, pattern, master=g.half())),
        (ValueError, lambda: KSMuon([])),
        (ValueError, lambda: KSMuon([(torch.nn.Parameter(g), (2, 8, 4, 1), 1)])),
    ]:
        with pytest.raises(error):
            call()
