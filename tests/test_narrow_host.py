"""Host side of the 4-bit products and of AdamW without a GPU: what reaches the kernels, and how often."""
import pytest
import torch

from ksmm_amd import KSAdamW, _lib, adamw, adamw_update, mx


class Native:
    """In place of the native module: its AdamW step has the status given."""

    def __init__(self, status):
        self.status, self.calls = status, 0

    def adamw_update(self, *args):
        self.calls += 1
        return self.status


def test_a_step_whose_launch_failed_is_not_made_again(monkeypatch):
    """Tables of tensors before the one that failed are updated: a second call would update them twice."""
    native = Native(-7)
    message = _lib.strerror(-7)
    monkeypatch.setattr(_lib, "native", lambda: native)
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("the step goes to the library a second time"))
    monkeypatch.setattr(_lib, "strerror", lambda status: message if status == -7 else pytest.fail(status))
    t = [torch.zeros(4)]
    with pytest.raises(_lib.KsmmError) as e:
        adamw_update(t, t, t, t)
    assert e.value.status == -7 and native.calls == 1


def test_a_tangent_is_refused(monkeypatch):
    """Forward-mode derivatives, whichever tensor has one: no kernel is reached."""
    from torch.autograd import forward_ad

    class Declines:
        @staticmethod
        def mx_linear(*args):
            return None

    def reached(*args, **kw):
        raise AssertionError("a kernel is reached")

    monkeypatch.setattr(_lib, "native", lambda: Declines)
    monkeypatch.setattr(mx.MXKernel, "forward", staticmethod(reached))
    monkeypatch.setattr(mx.MXFunction, "apply", reached)
    monkeypatch.setattr(mx, "_check_factor", lambda factor, pattern, gated: pattern)
    packed = object.__new__(mx.MXFactor)
    packed.codes = packed.scales = torch.zeros(1, dtype=torch.uint8)
    packed.pattern, packed.gated, packed.dtype = (1, 4, 8, 1), False, torch.float32
    x, factor, bias = torch.ones(2, 8), torch.ones(8, 4), torch.ones(4)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, factor, bias)]
        for args in ((dual[0], packed), (dual[0], factor, packed.pattern), (x, dual[1], packed.pattern), (x, packed, None, dual[2])):
            for on in (False, True):
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="forward-mode"):
                    mx.mx_linear(*args)
        with pytest.raises(AssertionError, match="reached"):
            mx.mx_linear(x, packed)


def test_no_two_tensors_of_a_step_are_rounded_alike(monkeypatch):
    """Seeds and numbers in a call of all groups, types and counts of steps; of one group they are those of its list."""
    seeds = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(adamw, "adamw_update", lambda params, grads, m, v, scales, masters, step, *how, **kw: seeds.append([how[5] + i for i in range(len(params))]))
    ps = [torch.nn.Parameter(torch.zeros(40, dtype=t)) for t in (torch.float32, torch.float16, torch.float32, torch.float32, torch.float16)]

    def step(opt, of):
        seeds.clear()
        for p in ps:
            p.grad = torch.ones_like(p) if any(p is q for q in of) else None
        opt.step()
        return [s for call in seeds for s in call]

    opt = KSAdamW([{"params": ps[:3]}, {"params": ps[3:4], "weight_decay": 0.0}, {"params": ps[4:]}], bits=8, seed=7)
    for of in (ps, ps[1:], ps[::2], ps):  # (counts of steps that differ, too)
        found = step(opt, of)
        assert len(found) == len(of) == len(set(found)), found
    assert sorted(step(KSAdamW(ps[:1] + ps[2:4], bits=8, seed=7), ps)) == [7, 8, 9]
