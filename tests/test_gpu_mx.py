"""Microscaled 4-bit numbers (quantize_mx, pack_mx, mx_linear and their modules) against the definitions in float64.

Tolerances, relative Frobenius.  Codes and scales: equal.  Products: what the codes stand for is multiplied exactly (three bits by three)
and summed in fp32; in order a sum of k terms is off by at most k 2^-24 of the sum of magnitudes, at random by sqrt(k) of it: 2e-6 for
k up to 1024 with the fp32 activations' 1e-6.  fp16 results: the last rounding, 2^-11, or for a result below 6e-5 half of 6e-8: 4.9e-4.
fp16 gradients of gated products: dz is rounded before the sums over it and they are once more, 2 * 2^-11 at most."""
import pytest
import torch

from tests import mx_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
TOL = {"fp32": 2e-6, "fp16": 4.9e-4}


def rel(x, y):
    x, y = x.double().cpu(), y.double().cpu()
    assert x.shape == y.shape
    x, y = x.detach(), y.detach()
    n = float(torch.linalg.vector_norm(y))
    e = float(torch.linalg.vector_norm(x - y))
    return e / n if n else e


def rows(n, features, bs_last, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, features, generator=g) * scale * torch.exp2(torch.randint(-3, 4, (n, features), generator=g).float())
    return (x.t() if bs_last else x).contiguous().to(dtype)


def factor(pattern, gated, dtype, seed=1):
    a, b, c, d = pattern
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(a * d * c, 2 * b if gated else b, generator=g) / c ** 0.5).to(dtype)


def factor_rows(f, pattern):
    """(a, d, rows, c)"""
    a, _, c, d = pattern
    return f.detach().cpu().reshape(a, d, c, -1).transpose(2, 3).contiguous()


SIZES = [(1, 1, 1), (2, 31, 1), (1, 32, 1), (3, 33, 2), (1, 96, 5), (2, 64, 16), (1, 17, 40), (1, 200, 3), (4, 192, 1), (1, 256, 8), (1, 70, 64)]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("sizes", SIZES)
def test_codes_and_scales(sizes, prec, bs_last):
    from ksmm_amd import quantize_mx

    a, c, d = sizes
    for n in (1, 2, 31, 65, 200):
        x = rows(n, a * c * d, bs_last, DT[prec], n)
        q = quantize_mx(x.cuda(), sizes, bs_last)
        code, scale = R.quantize(R.operand(x, a, c, d, bs_last).reshape(a * d, n, c))
        assert q.codes.shape == (a * d, n, 16 * scale.shape[-1]) and q.scales.shape == scale.shape
        assert torch.equal(q.scales.cpu().long(), scale)
        got = R.unpacked(q.codes)
        assert torch.equal(R.GRID[got & 7], R.GRID[code & 7]) and torch.equal(got >= 8, code >= 8)
        back = R.tensor(R.values(code, scale, c).reshape(a, d, n, c), x.shape, bs_last)
        assert torch.equal(q.dequantize().cpu(), back.to(DT[prec])) and q.dequantize().shape == x.shape
        assert torch.equal(q.dequantize(torch.float32).cpu(), back.float())


@pytest.mark.parametrize("bs_last", [False, True])
def test_every_fp16_number_and_scale(bs_last):
    """Each fp16 number as the largest of its block and beside each power of two above it."""
    from ksmm_amd import quantize_mx

    h = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    h = h[torch.isfinite(h)]
    blocks = [torch.stack([h, torch.full_like(h, 2.0 ** e)], 1) for e in range(-24, 16, 3)] + [torch.stack([h, -h], 1)]
    x = torch.cat(blocks)
    x = x.t().contiguous() if bs_last else x
    q = quantize_mx(x.cuda(), (1, 2, 1), bs_last)
    code, scale = R.quantize(R.operand(x, 1, 2, 1, bs_last)[0])
    assert torch.equal(q.scales.cpu().long(), scale)
    back = R.tensor(R.values(code, scale, 2)[:, None], x.shape, bs_last)
    assert torch.equal(q.dequantize(torch.float32).cpu().double(), back)


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("sizes", [(1, 64, 1), (2, 40, 3), (1, 96, 2)])
def test_infinities_and_nans_stay_in_their_block(sizes, bs_last, prec):
    from ksmm_amd import quantize_mx

    a, c, d = sizes
    x = rows(9, a * c * d, False, DT[prec])
    x[0, 5 * d], x[3, (c - 1) * d], x[4, 1] = float("inf"), float("nan"), -float("inf")
    x = (x.t() if bs_last else x).contiguous()
    q = quantize_mx(x.cuda(), sizes, bs_last)
    code, scale = R.quantize(R.operand(x, a, c, d, bs_last))
    assert (scale == 255).sum() == 3
    assert torch.equal(q.scales.cpu().long().reshape(scale.shape), scale)
    back = R.tensor(R.values(code, scale, c), x.shape, bs_last)
    got = q.dequantize().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(back))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(back.to(DT[prec])))


def test_ends_of_the_fp32_range():
    from ksmm_amd import quantize_mx

    x = torch.zeros(7, 32)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 0], x[5, 0] = 3.4e38, 2.0 ** -122, 2.0 ** -123, 1e-45, -(2.0 ** -119), 2.0 ** -126
    q = quantize_mx(x.cuda(), (1, 32, 1))
    code, scale = R.quantize(x)
    assert torch.equal(q.scales.cpu().long()[0], scale)
    assert torch.equal(q.dequantize().cpu().double(), R.values(code, scale, 32))


PATTERNS = [(1, 1, 1, 1), (2, 5, 3, 2), (1, 32, 32, 1), (3, 33, 40, 1), (1, 64, 192, 2), (2, 20, 65, 3), (1, 100, 64, 6), (1, 16, 48, 16), (1, 130, 300, 4),
            (6, 64, 64, 1), (1, 200, 1030, 1), (1, 8, 16, 37), (2, 96, 72, 3), (1, 48, 96, 64), (1, 768, 192, 2), (5, 34, 128, 8), (1, 9, 5000, 1), (1, 9, 1400, 4), (40, 16, 16, 1), (70, 4, 4, 1),
            (1, 40, 70, 17), (1, 33, 33, 20), (1, 24, 3000, 5), (2, 64, 64, 7), (1, 70, 384, 4)]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", PATTERNS)
def test_products(pattern, prec, bs_last):
    from ksmm_amd import MXKernel, mx_linear, pack_mx, quantize_mx

    a, b, c, d = pattern
    for n, gated, act, with_bias in ((1, False, None, True), (2, True, "silu", False), (7, False, "gelu", True), (33, True, "gelu", True), (64, False, None, False),
                                     (131, True, "silu", True), (200, True, None, False), (517, False, "gelu", False)):
        x, f = rows(n, a * c * d, bs_last, DT[prec], n), factor(pattern, gated, DT[prec])
        g = torch.Generator().manual_seed(2)
        bias = (torch.randn(a * f.shape[1] * d, generator=g) * 0.1).to(DT[prec]) if with_bias else None
        w = pack_mx(f.cuda(), pattern, gated)
        code, scale = R.quantize(factor_rows(f, pattern).reshape(a * d, -1, c))
        assert torch.equal(w.scales.cpu().long(), scale)
        cuda_bias = None if bias is None else bias.cuda()
        y = mx_linear(x.cuda(), w, bias=cuda_bias, act=act, bs_last=bs_last)
        want = R.product(R.rounded(R.operand(x, a, c, d, bs_last)), R.rounded(factor_rows(f, pattern)), None if bias is None else bias.double(), pattern, act, gated,
                         bs_last)
        want = R.tensor(want, y.shape, bs_last)
        assert y.dtype == DT[prec] and rel(y, want) <= TOL[prec], (n, gated, act)
        # the same numbers, however they were made, and handed out as they are
        q = quantize_mx(x.cuda(), (a, c, d), bs_last)
        z, codes, scales = MXKernel.forward(x.cuda(), w, cuda_bias, act, bs_last, need_codes=True)
        assert torch.equal(z, y) and torch.equal(codes, q.codes) and torch.equal(scales, q.scales)
        assert torch.equal(mx_linear(q, w, bias=cuda_bias, act=act, bs_last=bs_last), y)
        assert torch.equal(mx_linear(x.cuda(), f.cuda(), pattern, bias=cuda_bias, act=act, gated=gated, bs_last=bs_last), y)


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", [(1, 64, 192, 2), (3, 40, 33, 1), (1, 20, 64, 5)])
def test_a_nan_stays_in_its_row(pattern, prec, bs_last):
    from ksmm_amd import mx_linear, pack_mx

    a, b, c, d = pattern
    n = 70
    x = rows(n, a * c * d, False, DT[prec])
    clean = x.clone()
    x[3, 2 * d] = float("nan")
    x[68, 0] = float("inf")
    clean[3], clean[68] = 0, 0
    x, clean = ((t.t() if bs_last else t).contiguous().cuda() for t in (x, clean))
    w = pack_mx(factor(pattern, False, DT[prec]).cuda(), pattern)
    y, z = (mx_linear(t, w, bs_last=bs_last) for t in (x, clean))
    y, z = ((t.t() if bs_last else t) for t in (y, z))
    bad = torch.zeros(n, dtype=torch.bool)
    bad[3] = bad[68] = True
    assert torch.equal(y[~bad], z[~bad])
    first = y[bad].reshape(2, a, b, d)[:, 0, :, 0]  # the block that the two belong to
    assert torch.isnan(first).all()
    assert int(torch.isnan(y).sum()) == first.numel()


GRADS = [(1, 1, 1, 1), (2, 5, 3, 2), (3, 33, 40, 1), (1, 64, 192, 2), (2, 96, 72, 3), (1, 16, 48, 16)]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", GRADS)
def test_gradients_go_straight_through(pattern, prec, bs_last):
    from ksmm_amd import mx_linear, pack_mx

    a, b, c, d = pattern
    for n, gated, act, with_bias in ((1, False, None, True), (35, True, "silu", True), (70, False, "gelu", True), (129, True, "gelu", False), (64, False, "gelu", False)):
        x, f = rows(n, a * c * d, bs_last, DT[prec], n), factor(pattern, gated, DT[prec])
        g = torch.Generator().manual_seed(2)
        bias = (torch.randn(a * f.shape[1] * d, generator=g) * 0.1).to(DT[prec]) if with_bias else None
        dy = rows(n, a * b * d, bs_last, DT[prec], 5)
        leaves = [t.cuda().requires_grad_(True) for t in (x, f, bias) if t is not None]
        with torch.enable_grad():
            y = mx_linear(leaves[0], leaves[1], pattern, bias=leaves[2] if with_bias else None, act=act, gated=gated, bs_last=bs_last)
            got = torch.autograd.grad(y, leaves, dy.cuda())
            xq, wq = R.rounded(R.operand(x, a, c, d, bs_last)).requires_grad_(True), R.rounded(factor_rows(f, pattern)).requires_grad_(True)
            b64 = None if bias is None else bias.double().requires_grad_(True)
            want = R.product(xq, wq, b64, pattern, act, gated, bs_last)
            assert rel(y, R.tensor(want, y.shape, bs_last)) <= TOL[prec]
            grads = torch.autograd.grad(want, [t for t in (xq, wq, b64) if t is not None], R.operand(dy, a, b, d, bs_last).double())
        expected = [R.tensor(grads[0], x.shape, bs_last), grads[1].transpose(2, 3).reshape(f.shape)] + list(grads[2:])
        for u, v, t in zip(got, expected, leaves):
            assert u.dtype == t.dtype and rel(u, v) <= 2 * TOL[prec], (n, gated, act)
        # a packed factor hands the gradient on to the input
        with torch.enable_grad():
            y = mx_linear(leaves[0], pack_mx(f.cuda(), pattern, gated), bias=None if bias is None else bias.cuda(), act=act, bs_last=bs_last)
            assert torch.equal(torch.autograd.grad(y, leaves[0], dy.cuda())[0], got[0])


def test_the_formula_of_the_gradients_against_differences():
    for pattern, gated, name in (((2, 3, 5, 2), False, "gelu"), ((1, 4, 33, 3), True, "silu")):
        a, b, c, d = pattern
        g = torch.Generator().manual_seed(0)
        x, w = torch.randn(a, d, 4, c, generator=g).double(), torch.randn(a, d, 2 * b if gated else b, c, generator=g).double()
        bias = torch.randn(a * w.shape[2] * d, generator=g).double()
        with torch.enable_grad():
            args = [t.requires_grad_(True) for t in (x, w, bias)]
            assert torch.autograd.gradcheck(lambda *t: R.product(*t, pattern, name, gated, False), args)


def test_second_derivatives_and_quantised_inputs_are_refused():
    from ksmm_amd import mx_linear, pack_mx, quantize_mx

    with torch.enable_grad():
        x = torch.randn(4, 64, device="cuda", requires_grad=True)
        f = torch.randn(64, 32, device="cuda", requires_grad=True)
        y = mx_linear(x, f, (1, 32, 64, 1))
        (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.sum().backward()
        with pytest.raises(RuntimeError):
            mx_linear(quantize_mx(x, (1, 64, 1)), f, (1, 32, 64, 1))
    w = pack_mx(f, (1, 32, 64, 1))
    assert torch.equal(mx_linear(quantize_mx(x, (1, 64, 1)), w), mx_linear(x, w))


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("shape", [(0,), (3, 0), (2, 5)])
def test_batches_of_several_axes_and_of_none(shape, bs_last):
    from ksmm_amd import mx_linear, quantize_mx

    g = torch.Generator().manual_seed(0)
    x = torch.randn(*((64, *shape) if bs_last else (*shape, 64)), generator=g).cuda()
    f = torch.randn(64, 40, generator=g).cuda()
    with torch.enable_grad():
        leaves = [x.clone().requires_grad_(True), f.clone().requires_grad_(True), torch.zeros(40, device="cuda", requires_grad=True)]
        y = mx_linear(leaves[0], leaves[1], (1, 40, 64, 1), bias=leaves[2], act="gelu", bs_last=bs_last)
        assert y.shape == ((40, *shape) if bs_last else (*shape, 40))
        dx, df, db = torch.autograd.grad(y.sum(), leaves)
    assert dx.shape == x.shape and df.shape == f.shape
    assert quantize_mx(x, (1, 64, 1), bs_last).dequantize().shape == x.shape
    if x.numel() == 0:
        assert not df.any() and not db.any()
    else:
        flat = x.reshape(64, -1) if bs_last else x.reshape(-1, 64)
        assert torch.equal(y.reshape(40, -1) if bs_last else y.reshape(-1, 40), mx_linear(flat, f, (1, 40, 64, 1), act="gelu", bs_last=bs_last))


def test_unaligned_tensors():
    """Inputs, biases and results that start off a vector's boundary, whose rows are odd."""
    from ksmm_amd import MXKernel, pack_mx, quantize_mx

    for prec in ("fp32", "fp16"):
        for pattern in ((1, 37, 65, 1), (1, 37, 33, 3), (2, 64, 64, 2)):
            a, b, c, d = pattern
            for bs_last in (False, True):
                n = 67
                x, f = rows(n, a * c * d, bs_last, DT[prec]).cuda(), factor(pattern, False, DT[prec]).cuda()
                w = pack_mx(f, pattern)
                bias = torch.randn(a * b * d, device="cuda").to(DT[prec])
                y = MXKernel.forward(x, w, bias, None, bs_last)

                def off(t):
                    room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
                    room[1:].copy_(t.reshape(-1))
                    return room[1:].view(t.shape)

                out = off(torch.zeros_like(y))
                MXKernel.forward(off(x), w, off(bias), None, bs_last, out=out)
                assert torch.equal(out, y)
                q, p = quantize_mx(x, (a, c, d), bs_last), quantize_mx(off(x), (a, c, d), bs_last)
                assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
                p = pack_mx(off(f), pattern)
                assert torch.equal(p.codes, w.codes) and torch.equal(p.scales, w.scales)


def test_refusals():
    from ksmm_amd import MXFactor, MXKernel, MXLinear, MXTensor, mx_linear, pack_mx, quantize_mx

    x, f = torch.randn(4, 128, device="cuda"), torch.randn(128, 40, device="cuda")
    p = (2, 40, 64, 1)
    w = pack_mx(f, p)
    q = quantize_mx(x, (2, 64, 1))
    for call in (lambda: quantize_mx(x, (2, 64)), lambda: quantize_mx(x, (2, 32, 1)), lambda: quantize_mx(x, (0, 64, 1)), lambda: pack_mx(f, (2, 20, 64, 1)),
                 lambda: pack_mx(f, p, gated=True), lambda: mx_linear(x, f), lambda: mx_linear(x, w, (1, 40, 128, 1)), lambda: mx_linear(x, w, gated=True),
                 lambda: mx_linear(x, w, act="silu"), lambda: mx_linear(x, w, act="relu"), lambda: mx_linear(x[:, :64].contiguous(), w),
                 lambda: mx_linear(x, w, bias=torch.zeros(40, device="cuda")), lambda: mx_linear(quantize_mx(x, (1, 128, 1)), w), lambda: mx_linear(q, w, bs_last=True),
                 lambda: MXFactor(w.codes, w.scales, (2, 41, 64, 1)), lambda: MXFactor(w.codes, w.scales[:, :20].contiguous(), p), lambda: MXFactor(w.codes.float(), w.scales, p),
                 lambda: MXTensor(q.codes, q.scales, (2, 64, 1), (5, 128), torch.float32), lambda: MXLinear([]),
                 lambda: MXKernel.forward(x, w, out=torch.empty(4, 81, device="cuda")), lambda: MXLinear([w, w])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: quantize_mx(x.cpu(), (2, 64, 1)), lambda: quantize_mx(x.t(), (2, 64, 1), True), lambda: mx_linear(x, w, bias=torch.zeros(80, device="cuda").half()),
                 lambda: mx_linear(x, w, bias=torch.zeros(80))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(AssertionError):
        quantize_mx(x.double(), (2, 64, 1))
    with pytest.raises(RuntimeError):
        MXKernel.forward(x, w, out=x.view(-1)[:320].view(4, 80))
    for ws in (torch.empty(1 << 20, dtype=torch.uint8), torch.empty(8, 8, dtype=torch.uint8, device="cuda").t()):
        with pytest.raises(ValueError):
            MXKernel.forward(x, w, workspace=ws)


def test_captured_and_replayed():
    """Single rows from a captured graph, with eager work between the replays; two graphs at once."""
    from ksmm_amd import mx_linear, pack_mx

    pattern = (1, 768, 192, 2)
    w = pack_mx(factor(pattern, True, torch.float16).cuda(), pattern, True)
    graphs = []
    for n in (1, 5):
        x = torch.zeros(n, 384, dtype=torch.float16, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mx_linear(x, w, act="silu")
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mx_linear(x, w, act="silu")
        graphs.append((x, graph, y))
    for i in range(4):
        for x, graph, y in graphs:
            new = rows(x.shape[0], 384, False, torch.float16, 10 + i).cuda()
            x.copy_(new)
            graph.replay()
        for x, graph, y in graphs:
            assert torch.equal(y, mx_linear(rows(x.shape[0], 384, False, torch.float16, 10 + i).cuda(), w, act="silu"))
        torch.cuda.synchronize()


def test_other_streams():
    from ksmm_amd import mx_linear, pack_mx

    pattern = (6, 64, 64, 1)
    w = pack_mx(factor(pattern, False, torch.float16).cuda(), pattern)
    x = rows(3000, 384, False, torch.float16).cuda()
    want = mx_linear(x, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(mx_linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


@pytest.mark.parametrize("bs_last", [False, True])
def test_modules(bs_last):
    from ksmm_amd import KSFeedForwardMX, KSGatedLinearMX, KSLinear, KSLinearMX, KSMuon, MXLinear, mx_linear, pack_block

    torch.manual_seed(0)
    patterns = [(6, 64, 64, 1), (1, 768, 192, 2)]
    x = rows(50, 384, bs_last, torch.float16).cuda()
    layer = KSLinearMX(patterns, dtype=torch.float16, bs_last=bs_last, act="gelu")
    y = layer(x)
    z = mx_linear(mx_linear(x, layer.factors[0], patterns[0], bs_last=bs_last), layer.factors[1], patterns[1], bias=layer.bias, act="gelu", bs_last=bs_last)
    assert torch.equal(y, z)
    packed = layer.packed()
    assert torch.equal(packed(x), y) and not list(packed.parameters()) and packed.out_size == 1536
    layer.factors[0].data.zero_()  # (codes are a copy)
    assert torch.equal(packed(x), y)
    plain = KSLinear(patterns, algo="kernel", dtype=torch.float16, bs_last=bs_last, device="cuda")
    of = MXLinear.of(plain)
    again = MXLinear.of(KSLinear(patterns, algo="kernel", dtype=torch.float16, bs_last=bs_last, device="cuda"))
    again.load_state_dict(of.state_dict())
    assert torch.equal(of(x), again(x))

    gated = KSGatedLinearMX((1, 768, 192, 2), bs_last=bs_last)
    assert torch.equal(gated.packed()(x), gated(x))
    block = KSFeedForwardMX((1, 768, 192, 2), [(1, 192, 768, 2), (6, 64, 64, 1)], bs_last=bs_last)
    assert len(KSMuon.factors_of(block)) == 3
    n, r = block(block.begin(x), x)
    served = block.packed()
    m, s = served(served.begin(x), x)
    assert torch.equal(n, m) and torch.equal(r, s)
    assert torch.equal(pack_block(block)(block.begin(x), x)[0], n)
    with torch.enable_grad():
        n, r = block(block.begin(x), x)
        (n.float().sum() + r.float().sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
    assert all(not any(p is q for q in block.parameters()) for p in served.parameters())


@pytest.mark.parametrize("bs_last", [False, True])
def test_without_the_native_module(monkeypatch, bs_last):
    """The same results, gradients among them, through ctypes alone."""
    from ksmm_amd import _lib, mx_linear, pack_mx, quantize_mx

    def everything():
        out = []
        for pattern, gated, act in (((2, 40, 33, 1), False, "gelu"), ((1, 64, 96, 2), True, "silu"), ((1, 24, 64, 3), False, None)):
            a, b, c, d = pattern
            x, f = rows(70, a * c * d, bs_last, torch.float16).cuda(), factor(pattern, gated, torch.float16).cuda()
            bias = torch.linspace(-1, 1, a * f.shape[1] * d).half().cuda()
            q, w = quantize_mx(x, (a, c, d), bs_last), pack_mx(f, pattern, gated)
            out += [q.codes, q.scales, q.dequantize(), w.codes, w.dequantize(), mx_linear(x, w, bias=bias, act=act, bs_last=bs_last)]
            leaves = [t.clone().requires_grad_(True) for t in (x, f, bias)]
            with torch.enable_grad():
                y = mx_linear(leaves[0], leaves[1], pattern, bias=leaves[2], act=act, gated=gated, bs_last=bs_last)
                out += [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
                y = mx_linear(leaves[0], w, bias=leaves[2], act=act, bs_last=bs_last)
                out += [y.detach(), *torch.autograd.grad(y, [leaves[0], leaves[2]], torch.ones_like(y))]
        return out

    native = everything()
    assert _lib.native() is not _lib._NoNative
    monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    for x, y in zip(native, everything()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("pattern", [(1, 6, 9000, 1), (1, 5, 1200, 16), (2, 40, 2500, 2)])
def test_more_than_local_memory_holds(pattern, bs_last):
    """c so large that a workgroup cannot keep the codes of 32 rows."""
    from ksmm_amd import MXKernel, mx_linear, pack_mx, quantize_mx

    a, b, c, d = pattern
    for prec in ("fp16", "fp32"):
        for n, gated, act in ((3, True, "silu"), (70, False, "gelu")):
            x, f = rows(n, a * c * d, bs_last, DT[prec], n).cuda(), factor(pattern, gated, DT[prec]).cuda()
            w, q = pack_mx(f, pattern, gated), quantize_mx(x, (a, c, d), bs_last)
            y, codes, scales = MXKernel.forward(x, w, None, act, bs_last, need_codes=True)
            want = R.product(R.rounded(R.operand(x, a, c, d, bs_last)), R.rounded(factor_rows(f, pattern)), None, pattern, act, gated, bs_last)
            # (sums of 9000 terms in fp32, at random: sqrt(9000) 2^-24, 6e-6 of the sum's deviation)
            assert rel(y, R.tensor(want, y.shape, bs_last)) <= max(TOL[prec], 6e-6)
            assert torch.equal(codes, q.codes) and torch.equal(scales, q.scales) and torch.equal(mx_linear(q, w, act=act, bs_last=bs_last), y)


@pytest.mark.parametrize("bs_last", [False, True])
def test_offsets_beyond_31_bits(bs_last):
    """Tensors of almost 2^31 elements: their last rows as a tensor of their own."""
    from ksmm_amd import MXKernel, mx_linear, pack_mx, quantize_mx

    pattern, n = (1, 64, 64, 1), (1 << 25) - 4096
    w = pack_mx(factor(pattern, False, torch.float16).cuda(), pattern)
    part = rows(100, 64, False, torch.float16).cuda()
    x = torch.zeros((64, n) if bs_last else (n, 64), dtype=torch.float16, device="cuda")
    for at in (0, n // 2 + 7, n - 100):
        if bs_last:
            x[:, at:at + 100] = part.t()
        else:
            x[at:at + 100] = part
    y, codes, scales = MXKernel.forward(x, w, None, None, bs_last, need_codes=True)
    small = (part.t() if bs_last else part).contiguous()
    want, q = mx_linear(small, w, bs_last=bs_last), quantize_mx(small, (1, 64, 1), bs_last)
    big = quantize_mx(x, (1, 64, 1), bs_last)
    assert torch.equal(big.codes, codes) and torch.equal(big.scales, scales)
    back = big.dequantize()
    for at in (0, n // 2 + 7, n - 100):
        assert torch.equal(y[:, at:at + 100] if bs_last else y[at:at + 100], want)
        assert torch.equal(codes[:, at:at + 100], q.codes) and torch.equal(scales[:, at:at + 100], q.scales)
        assert torch.equal(back[:, at:at + 100] if bs_last else back[at:at + 100], q.dequantize())
    assert not (y[:, 200:300] if bs_last else y[200:300]).any()


def test_traced_modules_compute():
    from ksmm_amd import KSLinearMX

    torch.manual_seed(0)
    layer = KSLinearMX([(6, 64, 64, 1), (1, 96, 192, 2)], dtype=torch.float16)
    x, other = (torch.randn(9, 384, device="cuda").half() for _ in range(2))
    traced = torch.jit.trace(layer, (x,), check_trace=False)
    assert torch.equal(traced(other), layer(other))


def test_threads_at_once():
    """Calls of several threads on streams of their own."""
    import threading

    from ksmm_amd import mx_linear, pack_mx

    pattern = (1, 96, 192, 2)
    f = factor(pattern, True, torch.float16).cuda()
    w = pack_mx(f, pattern, True)
    xs = [rows(300 + 7 * i, 384, False, torch.float16, i).cuda() for i in range(4)]
    want = [mx_linear(x, w, act="silu") for x in xs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = mx_linear(xs[i], w, act="silu")
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("gated", [False, True])
def test_captured_training(gated):
    """Forward and backward pass of a captured step, replayed on new inputs."""
    from ksmm_amd import mx_linear

    pattern = (1, 96, 64, 2)
    x = rows(70, 128, False, torch.float16).cuda().requires_grad_(True)
    f = factor(pattern, gated, torch.float16).cuda().requires_grad_(True)
    dy = rows(70, 192, False, torch.float16, 3).cuda()

    def step():
        with torch.enable_grad():
            y = mx_linear(x, f, pattern, act="gelu", gated=gated)
            return (y.detach(), *torch.autograd.grad(y, (x, f), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(rows(70, 128, False, torch.float16, 20 + i).cuda())
            f.copy_(factor(pattern, gated, torch.float16, 30 + i).cuda())
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want), i


@pytest.mark.parametrize("leaf", ["x", "factor", "bias"])
@torch.enable_grad()
def test_captured_backward_beside_an_eager_graph_of_its_leaves(leaf):
    """Refused before anything is enqueued: the eager graph's nodes of the leaves belong to the default stream."""
    from ksmm_amd import mx_linear

    pattern = (1, 40, 64, 2)
    x = rows(9, 128, False, torch.float16).cuda().requires_grad_(leaf == "x")
    f = factor(pattern, False, torch.float16).cuda().requires_grad_(leaf == "factor")
    bias = torch.zeros(80, device="cuda").half().requires_grad_(leaf == "bias")
    leaves = [t for t in (x, f, bias) if t.requires_grad]
    dy = rows(9, 80, False, torch.float16, 3).cuda()
    torch.autograd.grad(mx_linear(x, f, pattern, bias), leaves, dy)
    eager = mx_linear(x, f, pattern, bias)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(mx_linear(x, f, pattern, bias), leaves, dy)
    want = torch.autograd.grad(eager, leaves, dy)
    del eager, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(mx_linear(x, f, pattern, bias), leaves, dy)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0])


def test_packed_blocks_are_their_own():
    from ksmm_amd import KSFeedForward, pack_block

    block = KSFeedForward((1, 64, 32, 2), [(1, 32, 64, 2)])
    new = pack_block(block)
    new.register_buffer("more", torch.zeros(1))
    assert not hasattr(block, "more") and "gated" in block._modules and type(block.gated) is not type(new.gated)


SLOPES = [(1, 1, 1, 1), (2, 5, 3, 2), (1, 32, 32, 1), (3, 33, 40, 1), (1, 64, 192, 2), (2, 96, 72, 2), (1, 130, 120, 1), (1, 768, 192, 2), (6, 64, 64, 1), (1, 200, 250, 1), (4, 192, 192, 1),
          (2, 24, 70, 3), (1, 130, 40, 4), (2, 96, 72, 3), (1, 40, 16, 5), (1, 48, 400, 1)]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", SLOPES)
def test_gradients_of_what_activations_are_applied_to(pattern, prec, bs_last):
    """In fp16 they are rounded once, 2^-11 of each; fp32 as its sums are."""
    from ksmm_amd import _lib, pack_mx, quantize_mx
    from ksmm_amd.mx import _slope

    a, b, c, d = pattern
    for n, gated, act, with_bias in ((1, True, "silu", True), (7, False, "gelu", True), (33, True, "gelu", False), (200, True, None, True), (517, False, "gelu", False),
                                     (1000, True, "silu", False)):
        x, f = rows(n, a * c * d, bs_last, DT[prec], n), factor(pattern, gated, DT[prec])
        total = a * b * d * (1 + gated)
        bias = torch.linspace(-1, 1, total).to(DT[prec]) if with_bias else None
        dy = rows(n, a * b * d, bs_last, DT[prec], n + 1)
        q, w = quantize_mx(x.cuda(), (a, c, d), bs_last), pack_mx(f.cuda(), pattern, gated)
        got = _slope(dy.cuda(), q, w, None if bias is None else bias.cuda(), act, bs_last)
        taken = bs_last and c <= 256 or d <= (4 if prec == "fp16" else 2) and c <= 64
        assert (got is not None) or not taken
        if got is None:
            continue
        xr = R.rounded(R.operand(x, a, c, d, bs_last))
        with torch.enable_grad():
            z = (xr @ R.rounded(factor_rows(f, pattern)).transpose(2, 3)).double()
            if bias is not None:
                z = z + bias.double().reshape(a, -1, d).permute(0, 2, 1).unsqueeze(2)
            z = z.detach().requires_grad_(True)
            y = R.act(act, z[..., :b]) * z[..., b:] if gated else R.act(act, z)
            want, = torch.autograd.grad(y, z, R.operand(dy, a, b, d, bs_last).double())
        assert rel(got, R.tensor(want, got.shape, bs_last)) <= (2.0 ** -11 + 1e-5 if prec == "fp16" else TOL[prec]), (n, gated, act)
        if n == 517:  # nothing behind the end is written
            room = torch.full((got.numel() + 64,), 7.0, dtype=DT[prec], device="cuda")
            out = room[:got.numel()]
            rc = _lib.load().ksmm_mx_slope(q.codes.data_ptr(), q.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), None, dy.cuda().data_ptr(), out.data_ptr(), n, a, b, c, d,
                                           0 if prec == "fp32" else 1, int(bs_last), 1, int(gated), torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and torch.equal(out, got.flatten()) and (room[got.numel():] == 7).all()


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", [(1, 1, 1, 1), (2, 5, 3, 2), (3, 33, 40, 1), (2, 20, 65, 3), (1, 100, 64, 6), (1, 9, 130, 4), (5, 34, 128, 8), (1, 8, 16, 37)])
def test_both_operands_as_values(pattern, prec, bs_last):
    from ksmm_amd import _lib, pack_mx, quantize_mx

    a, b, c, d = pattern
    for n, gated in ((1, False), (70, True), (517, False)):
        q = quantize_mx(rows(n, a * c * d, bs_last, DT[prec], n).cuda(), (a, c, d), bs_last)
        w = pack_mx(factor(pattern, gated, DT[prec]).cuda(), pattern, gated)
        room = [torch.full((a * c * d * k + 64,), 7.0, dtype=DT[prec], device="cuda") for k in (n, w.codes.size(1))]
        rc = _lib.load().ksmm_mx_values(q.codes.data_ptr(), q.scales.data_ptr(), room[0].data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), room[1].data_ptr(), n, w.codes.size(1),
                                        a, c, d, 0 if prec == "fp32" else 1, int(bs_last), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        for got, want in zip(room, (q.dequantize(), w.dequantize(DT[prec]))):
            assert torch.equal(got[:-64], want.flatten()) and (got[-64:] == 7).all()


@pytest.mark.parametrize("bs_last", [False, True])
def test_training_beyond_31_bits(bs_last):
    """Gradients of almost 2^31 elements behind an activation: those of rows alone."""
    from ksmm_amd import pack_mx, quantize_mx
    from ksmm_amd.mx import _slope

    pattern, n = (1, 64, 64, 1), (1 << 25) - 4096
    w = pack_mx(factor(pattern, False, torch.float16).cuda(), pattern)
    part, dpart = rows(100, 64, False, torch.float16).cuda(), rows(100, 64, False, torch.float16, 1).cuda()
    x, dy = (torch.zeros((64, n) if bs_last else (n, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    for at in (0, n // 2 + 7, n - 100):
        for whole, piece in ((x, part), (dy, dpart)):
            if bs_last:
                whole[:, at:at + 100] = piece.t()
            else:
                whole[at:at + 100] = piece
    small, dsmall = ((t.t() if bs_last else t).contiguous() for t in (part, dpart))
    want = _slope(dsmall, quantize_mx(small, (1, 64, 1), bs_last), w, None, "gelu", bs_last)
    got = _slope(dy, quantize_mx(x, (1, 64, 1), bs_last), w, None, "gelu", bs_last)
    for at in (0, n // 2 + 7, n - 100):
        assert torch.equal(got[:, at:at + 100] if bs_last else got[at:at + 100], want)
    assert not (got[:, 200:300] if bs_last else got[200:300]).any()


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", [(200, 4, 4, 1), (300, 4, 4, 1), (1, 40, 48, 200), (1, 40, 3000, 270), (1, 300, 1030, 1), (2, 70, 600, 1)])
def test_last_rows_of_the_batch_feature_major(pattern, prec):
    """One row, and odd numbers of them: rows that are read in pairs."""
    from ksmm_amd import MXKernel, mx_linear, pack_mx, quantize_mx

    a, b, c, d = pattern
    for n in (1, 2, 3, 33) + ((31, 65, 129, 257) if a * c * d < 100000 else ()) + ((12801, 16385) if a * c * d < 1100 else ()):
        x = rows(n, a * c * d, True, DT[prec], n).cuda()
        w, q = pack_mx(factor(pattern, False, DT[prec]).cuda(), pattern), quantize_mx(x, (a, c, d), True)
        y, codes, scales = MXKernel.forward(x, w, None, None, True, need_codes=True)
        assert torch.equal(codes, q.codes) and torch.equal(scales, q.scales) and torch.equal(y, mx_linear(q, w, bs_last=True))
        want = R.product(R.rounded(R.operand(x[:, -3:].contiguous(), a, c, d, True)), R.rounded(factor_rows(factor(pattern, False, DT[prec]), pattern)), None, pattern, None, False, True)
        assert rel(y[:, -3:], R.tensor(want, (a * b * d, min(n, 3)), True)) <= TOL[prec]


@pytest.mark.parametrize("bs_last", [False, True])
def test_local_memory_of_a_kernel_grows_from_call_to_call(bs_last):
    """The same kernel with 70, 100 and 150 KB of it, in that order."""
    from ksmm_amd import mx_linear, pack_mx

    for c in (2100 if bs_last else 3200, 5000, 7200 if bs_last else 8000):
        pattern = (1, 24, c, 1)
        x, f = rows(9, c, bs_last, torch.float32, 1), factor(pattern, True, torch.float32)
        y = mx_linear(x.cuda(), pack_mx(f.cuda(), pattern, True), act="gelu", bs_last=bs_last)
        want = R.product(R.rounded(R.operand(x, 1, c, 1, bs_last)), R.rounded(factor_rows(f, pattern)), None, pattern, "gelu", True, bs_last)
        assert rel(y, R.tensor(want, y.shape, bs_last)) <= 6e-6
