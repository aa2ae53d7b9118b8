"""Residual norm of rows so narrow that the norm leaves next to nothing of a gradient: one feature, or two behind a mean.

What is left is eps / (var + eps) of it.  fp32, relative Frobenius: a dozen roundings of 2^-24 of values that are products, not differences,
but for dv - mean(dv), half the difference of two random values: 5e-6 as for other rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("features,norm", [(1, "rms"), (2, "layer")])
@pytest.mark.parametrize("batch", [3, 60, 2500])
def test_gradients_of_narrow_rows(features, norm, batch, bs_last):
    from ksmm_amd import residual_norm

    g = torch.Generator().manual_seed(0)
    r, dn = (torch.randn(batch, features, generator=g) * 3 for _ in range(2))
    x, dr = (torch.randn(batch, features, generator=g) for _ in range(2))
    w = torch.randn(features, generator=g) * 0.1 + 1

    def normed(v):
        v = v - v.mean(1, keepdim=True) if norm == "layer" else v
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)

    def laid(t):
        return (t.t() if bs_last else t).contiguous()

    with torch.enable_grad():
        r64, x64 = r.double().requires_grad_(), x.double().requires_grad_()
        want, = torch.autograd.grad(normed(r64) * w.double(), r64, dn.double())
        want_x, = torch.autograd.grad(normed(x64) * w.double(), x64, dr.double())
        ours, x = laid(r).cuda().requires_grad_(), laid(x).cuda().requires_grad_()
        got, = torch.autograd.grad(residual_norm(None, ours, weight=w.cuda(), norm=norm, eps=1e-5, bs_last=bs_last)[1], ours, laid(dn).cuda())
        out = residual_norm(x, ours.detach(), post_weight=w.cuda(), norm=norm, eps=1e-5, bs_last=bs_last, need_norm=False)[0]
        got_x, = torch.autograd.grad(out, x, laid(dr).cuda())
    for a, b in ((got, want), (got_x, want_x)):
        assert float((a.cpu().double() - laid(b)).norm() / b.norm()) <= 5e-6
