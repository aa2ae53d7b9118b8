"""The gated projection and the residual norm inside autograd: traced, from several threads, into tensors that are watched."""

import threading
import pytest
import torch

pytestmark = pytest.mark.gpu


def operands():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 32, generator=g).cuda()
    return x, (torch.randn(32, 48, generator=g) / 6).cuda(), torch.randn(6, 32, generator=g).cuda(), torch.ones(32, device="cuda")


def test_results_written_into_a_saved_tensor_are_noticed():
    from ksmm_amd import GatedKernel

    x, w, _, _ = operands()
    held = torch.randn(6, 24, device="cuda")
    p = torch.randn(6, 24, device="cuda", requires_grad=True)
    with torch.enable_grad():
        y = (held * p).sum()
    GatedKernel.forward(x, w, (1, 24, 32, 1), out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
