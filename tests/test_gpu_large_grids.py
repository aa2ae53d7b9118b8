"""Blocks so many and small that their workgroups have 2^32 threads and more, which one launch does not start: results are right, or the call
is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
A = 16_800_000


def right_or_refused(call, wants, eps, least=1e-7):
    """Within ``eps`` of the value and ``least``: for sums of up to three terms below 30 two steps of 2^-24 of their magnitudes, 1.1e-5; for GELU's
    slope, 3e-7 off, times a gradient below 6, 2e-6."""
    from ksmm_amd import _lib

    try:
        got = call()
    except _lib.KsmmError as e:
        assert e.status == -5
        return
    for u, v in zip(got, wants):
        off = (u.double() - v).abs() - (eps * v.abs() + least)
        assert float(off.max()) <= 0, int((off > 0).sum())


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
def test_products_and_gradients(prec, bs_last, n):
    from ksmm_amd import GatedKernel, Kernel

    g = torch.Generator(device="cuda").manual_seed(0)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g).to(DT[prec])
    shape = (A, n) if bs_last else (n, A)
    eps = 2e-6 if prec == "fp32" else 2.0 ** -10  # (sums of one term, of n for weights; a product with an activation is one rounding more)
    x, dy, w = draw(*shape), draw(*shape), draw(A, 1)
    col = (lambda t: t.double().view(A, 1)) if bs_last else (lambda t: t.double().view(1, A))
    over = (lambda t: t.sum(1)) if bs_last else (lambda t: t.sum(0))
    pattern = (A, 1, 1, 1)
    right_or_refused(lambda: [Kernel.forward(x, w, bs_last, *pattern, dtype=DT[prec])], [x.double() * col(w)], eps)
    right_or_refused(lambda: Kernel.backward(dy, x, w, bs_last, *pattern), [dy.double() * col(w), over(dy.double() * x.double()).view(A, 1)], 4 * eps, 1.1e-5)
    z = draw(*shape)
    with torch.enable_grad():
        leaf = z.double().requires_grad_(True)
        dz, = torch.autograd.grad(torch.nn.functional.gelu(leaf), leaf, dy.double())
    right_or_refused(lambda: Kernel.epilogue_backward(dy, z, bs_last, "gelu"), [dz, over(dz)], 4 * eps, 1.3e-5)
    del z, leaf, dz
    f = draw(A, 2)
    right_or_refused(lambda: [GatedKernel.forward(x, f, pattern, None, None, bs_last)], [x.double() * col(f[:, 0]) * x.double() * col(f[:, 1])], 4 * eps)


@pytest.mark.parametrize("bs_last", [False, True])
def test_training_in_4_bits(bs_last):
    from ksmm_amd import mx_linear, pack_mx, quantize_mx

    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.randn(*((A, 2) if bs_last else (2, A)), device="cuda", generator=g) for _ in range(2))
    f = torch.randn(A, 1, device="cuda", generator=g)
    w, q = pack_mx(f, (A, 1, 1, 1)).dequantize(torch.float32).double(), quantize_mx(x, (A, 1, 1), bs_last).dequantize().double()

    def grads():
        with torch.enable_grad():
            leaves = [x.requires_grad_(True), f.requires_grad_(True)]
            return torch.autograd.grad(mx_linear(*leaves, (A, 1, 1, 1), bs_last=bs_last), leaves, dy)

    def call():
        from ksmm_amd import _lib

        try:
            return grads()
        except RuntimeError as e:
            if "status -5" in str(e):
                raise _lib.KsmmError(-5, "refused")
            raise

    want = [dy.double() * (w.view(A, 1) if bs_last else w.view(1, A)), (dy.double() * q).sum(1 if bs_last else 0).view(A, 1)]
    right_or_refused(call, want, 4e-6, 1.1e-5)
