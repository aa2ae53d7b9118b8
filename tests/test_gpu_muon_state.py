"""KSMuon over its life: saved and resumed, next to autograd, next to others who write the weights."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
PATTERNS = [((2, 24, 16, 1), 1), ((1, 20, 12, 2), 2), ((1, 130, 140, 1), 1)]


def factors(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.nn.Parameter((torch.randn(a * d * c, parts * b, generator=g) * 0.2).to(dtype).cuda()), (a, b, c, d), parts)
            for (a, b, c, d), parts in PATTERNS]


def step(opt, fs, i):
    g = torch.Generator().manual_seed(100 + i)
    for p, _, _ in fs:
        p.grad = (torch.randn(p.shape, generator=g) * 0.01).to(p.dtype).cuda()
    opt.step()


def tensors(opt):
    return [v for s in opt.state.values() for v in (s["momentum"], s.get("master")) if v is not None]


@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("model_first", [True, False])
def test_resumed_steps_are_those_that_were_not_interrupted(prec, model_first):
    from ksmm_amd import KSMuon

    fs = factors(DT[prec])
    opt = KSMuon(fs, lr=0.01, weight_decay=0.1)
    for i in range(3):
        step(opt, fs, i)
    saved = io.BytesIO()
    torch.save([opt.state_dict(), [p.detach() for p, _, _ in fs]], saved)
    for i in range(3, 6):
        step(opt, fs, i)
    saved.seek(0)
    state, weights = torch.load(saved, weights_only=True)
    again = factors(DT[prec], seed=9)
    resumed = KSMuon(again, lr=0.5)
    if not model_first:
        resumed.load_state_dict(state)
    with torch.no_grad():
        for (p, _, _), w in zip(again, weights):
            p.copy_(w)
    if model_first:
        resumed.load_state_dict(state)
    assert all(t.dtype == torch.float32 for t in tensors(resumed))
    before = copy.deepcopy(state)
    for i in range(3, 6):
        step(resumed, again, i)
    for (p, _, _), (q, _, _) in zip(fs, again):
        assert torch.equal(p, q)
    assert all(torch.equal(x, y) for x, y in zip(tensors(opt), tensors(resumed))) and len(tensors(opt)) == (6 if prec == "fp16" else 3)
    for k in state["state"]:  # what was loaded from is not written
        assert torch.equal(state["state"][k]["momentum"], before["state"][k]["momentum"])


def test_autograd_sees_the_new_weights():
    """A graph that was made with the old weights refuses to run backward, as it does behind torch's optimisers."""
    from ksmm_amd import KSMuon, gated_linear, muon_update

    pattern = (1, 16, 8, 2)
    for prec in ("fp32", "fp16"):
        w = torch.nn.Parameter((torch.randn(16, 32) * 0.3).to(DT[prec]).cuda())
        x = torch.randn(5, 16, device="cuda").to(DT[prec]).requires_grad_()
        opt = KSMuon([(w, pattern, 2)])
        with torch.enable_grad():
            h = gated_linear(x, w, pattern)
            h.sum().backward(retain_graph=True)
            opt.step()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                h.sum().backward()
        m, master = torch.zeros(16, 32, device="cuda"), torch.zeros(16, 32, device="cuda")
        at = [t._version for t in (w, m, master)]
        muon_update(w, w.grad, m, pattern, parts=2, master=master, inplace=True)
        assert all(t._version > v for t, v in zip((w, m, master), at))
        at = [t._version for t in (w, m, master)]
        muon_update(w, w.grad, m, pattern, parts=2, master=master)  # writes the master alone
        assert [t._version > v for t, v in zip((w, m, master), at)] == [False, False, True]


def test_inference_tensors_are_updated_too():
    from ksmm_amd import muon_update

    with torch.inference_mode():
        w, g, m = (torch.randn(16, 8, device="cuda") for _ in range(3))
        want, want_m = muon_update(w, g, m, (1, 8, 8, 2))
        muon_update(w, g, m, (1, 8, 8, 2), inplace=True)
        assert torch.equal(w, want) and torch.equal(m, want_m)


@pytest.mark.parametrize("how", ["copy", "data", "some"])
def test_weights_that_others_wrote_count(how):
    """fp32 masters stand behind fp16 weights that are still their rounding; weights loaded or changed afterwards replace them."""
    from ksmm_amd import KSMuon

    fs, new = factors(torch.float16), factors(torch.float16, seed=5)
    opt = KSMuon(fs, lr=0.01)
    for i in range(2):
        step(opt, fs, i)
    masters = [opt.state[p]["master"].clone() for p, _, _ in fs]
    with torch.no_grad():
        for (p, _, _), (q, _, _) in zip(fs, new):
            if how == "copy":
                p.copy_(q)
            elif how == "data":  # (autograd does not see this one)
                p.data.copy_(q)
            else:
                p[1].copy_(q[1])
    # (a written value that is by chance what the master rounds to leaves it its bits)
    want = [torch.where(p.detach() == m.half(), m, p.detach().float()) for (p, _, _), m in zip(fs, masters)]
    assert all(not torch.equal(w, m) for w, m in zip(want, masters))
    ref = [(torch.nn.Parameter(p.detach().clone()), pattern, parts) for p, pattern, parts in fs]
    other = KSMuon(ref, lr=0.01)
    for (p, _, _), (q, _, _), m in zip(fs, ref, want):
        other.state[q] = {"momentum": opt.state[p]["momentum"].clone(), "master": m.clone()}
    step(opt, fs, 2)
    step(other, ref, 2)
    for (p, _, _), (q, _, _) in zip(fs, ref):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], other.state[q]["master"])


def test_coefficients_that_leave_the_range_are_refused():
    """Iterates are held as pairs of fp16 numbers: coefficients with which a singular value of one or less could leave their range."""
    from ksmm_amd import orthogonalize

    u = torch.randn(32, 16, device="cuda")
    for p, steps in (((20.0, 0.0, 0.0), 5), ((3.4445, -4.775, 20.0), 5), ((1.0, 0.0, 1e6), 1), ((float("nan"), 0.0, 0.0), 1)):
        with pytest.raises(RuntimeError):
            orthogonalize(u, (1, 16, 32, 1), steps=steps, coefficients=p)
    assert orthogonalize(u, (1, 16, 32, 1), steps=2, coefficients=(20.0, 0.0, 0.0)).isfinite().all()
