"""Products of 4-bit numbers: calls beside the ordinary ones."""
import pytest
import torch

from tests import mx_ref as R
from tests.test_gpu_mx import DT, TOL, factor, factor_rows, rel, rows

pytestmark = pytest.mark.gpu


def test_a_given_result_counts_as_written():
    """A graph that holds the memory that a result went into raises."""
    from ksmm_amd import MXKernel, pack_mx

    pattern = (1, 40, 64, 1)
    w = pack_mx(factor(pattern, False, torch.float32).cuda(), pattern)
    x = rows(5, 64, False, torch.float32).cuda()
    out = torch.zeros(5, 40, device="cuda")
    before = out._version
    assert MXKernel.forward(x, w, out=out) is out and out._version == before + 1
    with torch.enable_grad():
        leaf = torch.ones(5, 40, device="cuda", requires_grad=True)
        y = leaf * out
        MXKernel.forward(x, w, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():  # (tensors without a count)
        out = torch.empty(5, 40, device="cuda")
        assert torch.equal(MXKernel.forward(x, w, out=out), MXKernel.forward(x, w))


FAR = [(1, 16, 64, 5), (2, 8, 33, 6), (1, 12, 40, 17), (1, 20, 400, 4), (1, 40, 600, 1), (1, 6, 9000, 1)]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("pattern", FAR)
def test_gradients_far_below_zero(monkeypatch, pattern, bs_last, native):
    """GELU of what fp16 does not hold: its result is zero, and so is its slope.  dz is rounded once, the sums over it once more: twice 2^-11."""
    from ksmm_amd import _lib, mx_linear

    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    a, b, c, d = pattern
    n = 37
    x, f = rows(n, a * c * d, bs_last, torch.float16, 1), factor(pattern, False, torch.float16)
    f[:, 0] = -64.0  # z of the first output of a block: -64 |x| summed, below -65504 with the rows made large
    x = x.abs().clamp(max=8.0)
    if bs_last:
        x[:, :5] = 512.0
    else:
        x[:5] = 512.0
    dy = rows(n, a * b * d, bs_last, torch.float16, 5)
    leaves = [t.cuda().requires_grad_(True) for t in (x, f)]
    bias = torch.linspace(-1, 1, a * b * d).half().cuda().requires_grad_(True)
    with torch.enable_grad():
        y = mx_linear(leaves[0], leaves[1], pattern, bias=bias, act="gelu", bs_last=bs_last)
        got = torch.autograd.grad(y, [*leaves, bias], dy.cuda())
        xq, wq = R.rounded(R.operand(x, a, c, d, bs_last)).requires_grad_(True), R.rounded(factor_rows(f, pattern)).requires_grad_(True)
        b64 = bias.detach().cpu().double().requires_grad_(True)
        want = R.product(xq, wq, b64, pattern, "gelu", False, bs_last)
        assert float(R.product(xq, wq, b64, pattern, None, False, bs_last).min()) < -65520
        grads = torch.autograd.grad(want, [xq, wq, b64], R.operand(dy, a, b, d, bs_last).double())
    assert torch.isfinite(y).all()
    for u, v in zip(got, [R.tensor(grads[0], x.shape, bs_last), grads[1].transpose(2, 3).reshape(f.shape), grads[2]]):
        assert torch.isfinite(u).all() and rel(u, v) <= 2 * TOL["fp16"]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("pattern", [(1, 40, 16, 5), (2, 24, 70, 3), (2, 33, 33, 17), (1, 70, 64, 16), (1, 6, 9000, 1), (1, 5, 1200, 16)])
def test_sums_for_gradients(pattern, prec, bs_last):
    """What GELU is applied to: the product's result without it, but that fp16 ends at 65504, and a NaN is none.  Nothing behind the end is written."""
    from ksmm_amd import _lib, mx_linear, pack_mx, quantize_mx
    from ksmm_amd.mx import _ptr

    a, b, c, d = pattern
    for n, with_bias in ((1, True), (33, False), (70, True), (517, False)):
        x, f = rows(n, a * c * d, False, DT[prec], n), factor(pattern, False, DT[prec])
        x[0] *= 1000
        f[:, 0] *= 1000
        f[:, 1] *= -1000
        x[n // 2, 0] = float("nan")
        x = (x.t() if bs_last else x).contiguous()
        bias = torch.linspace(-1, 1, a * b * d).to(DT[prec]).cuda() if with_bias else None
        q, w = quantize_mx(x.cuda(), (a, c, d), bs_last), pack_mx(f.cuda(), pattern)
        y = mx_linear(q, w, bias=bias, bs_last=bs_last)
        room = torch.full((y.numel() + 64,), 7.0, dtype=DT[prec], device="cuda")
        assert _lib.load().ksmm_mx_sums(q.codes.data_ptr(), q.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), _ptr(bias), room.data_ptr(), n, a, b, c, d,
                                        0 if prec == "fp32" else 1, int(bs_last), torch.cuda.current_stream().cuda_stream) == 0
        z = room[:-64].view(y.shape)
        assert torch.isnan(y).any() and (prec == "fp32" or n == 1 or torch.isinf(y).any())
        assert torch.equal(torch.isnan(z), torch.isnan(y))
        want = y.clamp(-65504, 65504) if prec == "fp16" else y
        assert torch.equal(torch.nan_to_num(z), torch.nan_to_num(want)) and (room[-64:] == 7).all()


def wide(gated, d=1, seed=0):
    """A factor in fp32 whose first block lies beyond fp16's range and whose second one below it, and an input and gradient for it.

    Products of the first are 2^8 (gated dz 2^-7), of gradients 2^12; of the second 2^-12."""
    g = torch.Generator().manual_seed(seed)
    pattern, n = (2, 24, 64, d), 41
    a, b, c, d = pattern
    f = torch.randn(a, d * c, 2 * b if gated else b, generator=g) * torch.tensor([2.0 ** 17, 2.0 ** -27]).view(2, 1, 1)
    x = torch.randn(n, a, c * d, generator=g) * torch.tensor([2.0 ** -12, 1.0]).view(1, 2, 1)
    dy = torch.randn(n, a, b * d, generator=g) * torch.tensor([2.0 ** -15, 2.0 ** 13]).view(1, 2, 1)
    return pattern, f.reshape(a * d * c, -1), x.reshape(n, -1).half(), dy.reshape(n, -1).half()


def wide_gradients(pattern, f, x, dy, bias, act, gated):
    a, b, c, d = pattern
    with torch.enable_grad():
        xq, wq = R.rounded(R.operand(x, a, c, d, False)).requires_grad_(True), R.rounded(factor_rows(f, pattern))
        b64 = bias.double().requires_grad_(True)
        want = R.product(xq, wq, b64, pattern, act, gated, False)
        dx, db = torch.autograd.grad(want, [xq, b64], R.operand(dy, a, b, d, False).double())
    return R.tensor(dx, x.shape, False), db


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("gated,act", [(False, None), (False, "gelu"), (True, "silu"), (True, None)])
@pytest.mark.parametrize("made", ["packed", "by hand"])
@pytest.mark.parametrize("d", [1, 5])
def test_gradients_through_values_beyond_fp16(monkeypatch, d, made, gated, act, native):
    """Codes of fp32 weights hold values that fp16 has not: gradients of fp16 inputs are rounded once for all that, at the end."""
    from ksmm_amd import MXFactor, _lib, mx_linear, pack_mx

    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    pattern, f, x, dy = wide(gated, d)
    w = pack_mx(f.cuda(), pattern, gated)
    if made == "by hand":
        w = MXFactor(w.codes, w.scales, pattern, gated)
    bias = torch.linspace(-1, 1, f.shape[1] * 2 * d).half()
    leaves = [t.cuda().requires_grad_(True) for t in (x, bias)]
    with torch.enable_grad():
        y = mx_linear(leaves[0], w, bias=leaves[1], act=act)
        dx, db = torch.autograd.grad(y, leaves, dy.cuda())
    assert y.dtype == dx.dtype == db.dtype == torch.float16
    want, want_b = wide_gradients(pattern, f, x, dy, bias, act, gated)
    for part in (slice(0, 64 * d), slice(64 * d, None)):
        # (a value is rounded to 2^-11 of it, or to 2^-25 where the type has no more)
        assert rel(dx[:, part], want[:, part]) <= TOL["fp16"] + 2.0 ** -25 * want[:, part].numel() ** 0.5 / float(want[:, part].norm())
    fine = want_b.abs() < 65504
    assert fine.sum() >= 24 and rel(db.cpu()[fine], want_b[fine]) <= TOL["fp16"]


def test_gradients_through_loaded_codes():
    from ksmm_amd import KSLinear, MXLinear

    pattern, f, x, dy = wide(False)
    layers = {}
    for dtype in (torch.float32, torch.float16):
        layer = KSLinear([pattern], algo="kernel", bias=False, dtype=dtype, device="cuda")
        layer.factors[0].data.copy_(f.clamp(-60000, 60000))
        layers[dtype] = MXLinear.of(layer)
    layer = KSLinear([pattern], algo="kernel", bias=False, dtype=torch.float32, device="cuda")
    layer.factors[0].data.copy_(f)
    full = MXLinear.of(layer)
    layers[torch.float16].load_state_dict(full.state_dict())
    want, _ = wide_gradients(pattern, f, x, dy, torch.zeros(48), None, False)
    for served in (full, layers[torch.float16]):
        with torch.enable_grad():
            leaf = x.cuda().requires_grad_(True)
            dx, = torch.autograd.grad(served(leaf), leaf, dy.cuda())
        assert rel(dx, want) <= TOL["fp16"] and rel(dx[:, 64:], want[:, 64:]) <= 2 * TOL["fp16"]
    # and back: codes of fp16 weights
    narrow = MXLinear.of(KSLinear([pattern], algo="kernel", bias=False, dtype=torch.float16, device="cuda"))
    full.load_state_dict(narrow.state_dict())
    with torch.enable_grad():
        leaf = x.cuda().requires_grad_(True)
        assert torch.equal(*(torch.autograd.grad(m(leaf), leaf, dy.cuda())[0] for m in (full, narrow)))


def test_forward_mode_is_refused():
    """A tangent would be lost."""
    from torch.autograd import forward_ad

    from ksmm_amd import KSLinearMX, MXLinear, mx_linear, pack_mx, quantize_mx

    pattern = (1, 40, 64, 1)
    x, f, bias = rows(5, 64, False, torch.float32).cuda(), factor(pattern, False, torch.float32).cuda(), torch.zeros(40, device="cuda")
    w = pack_mx(f, pattern)
    layer = KSLinearMX([pattern], dtype=torch.float32, bias=False)
    with forward_ad.dual_level():
        dx, df, db = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, f, bias))
        for call in (lambda: mx_linear(dx, w), lambda: mx_linear(dx, f, pattern), lambda: mx_linear(x, df, pattern), lambda: mx_linear(x, w, bias=db),
                     lambda: mx_linear(quantize_mx(x, (1, 64, 1)), w, bias=db), lambda: layer(dx), lambda: layer.packed()(dx)):
            for on in (False, True):
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert torch.equal(mx_linear(x, w), mx_linear(x, f, pattern))  # (tensors without one)


@pytest.mark.parametrize("native", [True, False])
def test_an_error_from_before_is_not_the_calls_own(monkeypatch, native):
    """What an earlier call on the thread left is neither taken for a launch's own nor cleared."""
    from ksmm_amd import _lib, mx_linear, pack_mx, quantize_mx
    from ksmm_amd.mx import _slope

    lib = _lib.load()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    pattern = (1, 40, 64, 2)
    x, f, dy = rows(70, 128, False, torch.float16).cuda(), factor(pattern, False, torch.float16).cuda(), rows(70, 80, False, torch.float16, 1).cuda()
    got = []
    for before in (False, True):
        w, q = pack_mx(f, pattern), quantize_mx(x, (1, 64, 2))
        torch.cuda.synchronize()
        if before:
            assert lib.hipSetDevice(1 << 20) != 0
        try:
            now = [pack_mx(f, pattern).codes, quantize_mx(x, (1, 64, 2)).codes, q.dequantize(), mx_linear(x, w, act="gelu"), mx_linear(q, w), mx_linear(x, f, pattern),
                   _slope(dy, q, w, None, "gelu", False)]
        finally:
            left = lib.hipGetLastError()
        assert (left != 0) == before
        got.append(now)
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
def test_more_workgroups_than_a_launch_takes(prec, bs_last):
    """2^32 threads and more: blocks of one number each, whose product is that of two numbers."""
    from ksmm_amd import MXKernel, pack_mx, quantize_mx
    from ksmm_amd.mx import _slope

    a = 16_800_000
    g = torch.Generator(device="cuda").manual_seed(0)
    f = torch.randn(a, 1, device="cuda", generator=g).to(DT[prec])
    w = pack_mx(f, (a, 1, 1, 1))
    wq = w.dequantize(torch.float32).flatten()
    assert bool(((wq - f.flatten().float()).abs() <= 0.25 * f.flatten().float().abs()).all())  # (saturation: 7.99 of 8 is 6)
    for n in (1, 3):
        x = torch.randn(*((a, n) if bs_last else (n, a)), device="cuda", generator=g).to(DT[prec])
        q = quantize_mx(x, (a, 1, 1), bs_last)
        xq = q.dequantize(torch.float32)
        z = xq * (wq.unsqueeze(1) if bs_last else wq)  # (exact: three bits by three)
        y, codes, scales = MXKernel.forward(x, w, None, None, bs_last, need_codes=True)
        assert torch.equal(y, z.to(DT[prec])) and torch.equal(codes, q.codes) and torch.equal(scales, q.scales)
        assert torch.equal(MXKernel.forward(q, w, None, None, bs_last), y)
        del y, codes, scales
        dz = _slope(torch.ones_like(x), q, w, None, "gelu", bs_last)
        with torch.enable_grad():
            z.requires_grad_(True)
            want, = torch.autograd.grad(torch.nn.functional.gelu(z).sum(), z)
        assert bool(((dz.float() - want).abs() <= (2.0 ** -11 if prec == "fp16" else 2e-6) * want.abs() + 2e-6).all())


def test_copies_have_hooks_of_their_own():
    from ksmm_amd import KSFeedForwardMX
    from ksmm_amd.train_block import KSStack

    block = KSFeedForwardMX((1, 64, 32, 2), [(1, 32, 64, 2)])
    stack = KSStack((1, 64, 32, 2), [(1, 32, 64, 2)], 1, mx=True)
    for module in (block, stack):
        copy = module.packed()
        calls = []
        copy.register_forward_hook(lambda *a: calls.append("copy"))
        copy.register_forward_pre_hook(lambda *a: calls.append("copy"))
        assert not module._forward_hooks and not module._forward_pre_hooks
        copy.register_buffer("more", torch.zeros(1), persistent=False)
        assert not hasattr(module, "more") and not module._non_persistent_buffers_set


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("pattern", [(1, 2000, 1, 1), (1, 500, 40, 4), (2, 200, 33, 5), (1, 2000, 9000, 1)])
def test_gelu_in_fp32_far_below_zero(pattern, bs_last):
    """Of one factor, relative to its value: 1e-6, and what an exponent of 0.72 z^2 is off by, four times 2^-24 of it: 1.2e-7 z^2."""
    from ksmm_amd import mx_linear, pack_mx

    a, b, c, d = pattern
    w = pack_mx(factor(pattern, False, torch.float32).cuda(), pattern)
    z = torch.linspace(-12, 6, a * b * d)  # (the bias: sums of zeros are exact)
    for n in (1, 300):
        x = torch.zeros((a * c * d, n) if bs_last else (n, a * c * d), device="cuda")
        y = mx_linear(x, w, bias=z.cuda(), act="gelu", bs_last=bs_last).cpu().double()
        want = z.double() * torch.special.erfc(-z.double() * 0.5 ** 0.5) / 2
        off = ((y.t() if bs_last else y) - want).abs()
        assert bool((off <= (1e-6 + 1.2e-7 * z.double().square()) * want.abs()).all())


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("shape", [(0,), (3, 0)])
def test_gated_batches_of_none(shape, bs_last):
    from ksmm_amd import mx_linear

    for d in (1, 5):
        pattern = (1, 40, 64, d)
        x = torch.zeros(*((64 * d, *shape) if bs_last else (*shape, 64 * d)), device="cuda")
        with torch.enable_grad():
            leaves = [x.requires_grad_(True), torch.ones(64 * d, 80, device="cuda", requires_grad=True), torch.zeros(80 * d, device="cuda", requires_grad=True)]
            y = mx_linear(leaves[0], leaves[1], pattern, bias=leaves[2], act="silu", gated=True, bs_last=bs_last)
            dx, df, db = torch.autograd.grad(y.sum(), leaves)
        assert y.shape == ((40 * d, *shape) if bs_last else (*shape, 40 * d)) and dx.shape == x.shape
        assert not df.any() and not db.any() and df.shape == (64 * d, 80)
