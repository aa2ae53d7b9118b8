"""The gated projection and the residual norm inside autograd: traced, from several threads, into tensors that are watched."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def operands():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 32, generator=g).cuda()
    return x, (torch.randn(32, 48, generator=g) / 6).cuda(), torch.randn(6, 32, generator=g).cuda(), torch.ones(32, device="cuda")


def test_traced_functions_compute():
    """torch.jit.trace records the operators, not the memory of the traced call's results."""
    from ksmm_amd import gated_linear, residual_norm

    x, w, r, v = operands()

    def gated(x):
        return gated_linear(x, w, (1, 24, 32, 1)) * 1.0

    def norm(x, r):
        out, n = residual_norm(x, r, weight=v)
        return out * 1.0, n * 1.0

    def only_norm(r):
        return residual_norm(None, r, weight=v)[1] * 1.0

    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            for fn, args in ((gated, (x,)), (norm, (x, r)), (only_norm, (r,))):
                traced = torch.jit.trace(fn, args, check_trace=False)
                other = tuple(t * 1.5 + 0.25 for t in args)
                got, want = traced(*other), fn(*other)
                for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                    assert torch.equal(a, b)


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


def test_one_graph_from_two_threads():
    """Each backward pass of a shared graph gives its gradients, or says that the graph is gone."""
    from ksmm_amd import gated_linear, residual_norm

    x, w, r, v = operands()
    for _ in range(20):
        leaves = [t.clone().requires_grad_() for t in (x, r, w, v)]
        with torch.enable_grad():
            out, n = residual_norm(leaves[0], leaves[1], weight=leaves[3])
            total = out.sum() + gated_linear(n, leaves[2], (1, 24, 32, 1)).sum()
        want = torch.autograd.grad(total, leaves, retain_graph=True)
        got, errors = [], []

        def backward():
            try:
                got.append(torch.autograd.grad(total, leaves))
            except RuntimeError as e:
                errors.append(str(e))

        threads = [threading.Thread(target=backward) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=60)
            assert not t.is_alive()
        assert len(got) + len(errors) == 2 and all("second time" in e for e in errors), errors
        for grads in got:
            assert all(torch.equal(a, b) for a, b in zip(grads, want))
