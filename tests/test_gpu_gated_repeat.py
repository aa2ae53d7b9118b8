"""Gated projection: every call on the same tensors gives the same bits, forward and backward.  Outputs and rows that no vector divides are
where two workgroups, or two vectors of one, hold the same results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("pattern,batch", [((2, 193, 96, 8), 4001), ((6, 129, 128, 4), 9881), ((3, 97, 64, 1), 6001), ((2, 130, 48, 2), 6001), ((2, 41, 80, 3), 6001),
                                           ((1, 99, 64, 6), 4003), ((1, 203, 40, 5), 4003), ((4, 65, 33, 16), 1003)])
def test_calls_repeat(pattern, batch, dtype, bs_last):
    from ksmm_amd import gated_linear

    a, b, c, d = pattern
    g = torch.Generator(device="cuda").manual_seed(1)

    def make(features, scale=1.0):
        return (torch.randn((features, batch) if bs_last else (batch, features), generator=g, device="cuda") * scale).to(dtype)

    x, dh = make(a * c * d), make(a * b * d)
    w = (torch.randn(a * d * c, 2 * b, generator=g, device="cuda") / c ** 0.5).to(dtype)
    v = (torch.randn(2 * a * b * d, generator=g, device="cuda") * 0.1).to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, v)]

    def results():
        with torch.enable_grad():
            h = gated_linear(x, w, pattern, v, "silu", bs_last)
            return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

    first = results()
    for _ in range(20):
        assert [torch.equal(p, q) for p, q in zip(results(), first)] == [True] * 4
