"""What the C ABI of the operators around a feed-forward block refuses before anything is launched, and what its optimiser keeps of its
state (no GPU)."""
import ctypes

import pytest
import torch

ALIAS = -11
FAR = [(i + 1) << 28 for i in range(16)]  # addresses that are never touched: every call here is refused


def test_update_refuses_results_that_lie_in_operands(lib):
    """Only the weights, the momentum and the masters may be written in their own place."""
    from ksmm_amd._lib import KsmmMuonDesc

    desc = KsmmMuonDesc((ctypes.c_float * 3)(1, 0, 0), 1e-7, 0.9, 1, 1, 5, 1)
    for blocks, c, b in ((2, 16, 16), (1, 200, 200)):
        need = lib.ksmm_muon_workspace(blocks, c, b, 1)
        size = 4 * blocks * c * b
        names = ["grad", "momentum", "momentum_out", "weight", "master", "master_out", "out", "workspace"]
        base = dict(zip(names, FAR))
        outs = ["momentum_out", "master_out", "out"] + (["workspace"] if need else [])

        def call(**change):
            p = dict(base, **change)
            return lib.ksmm_muon_update(ctypes.byref(desc), p["grad"], p["momentum"], p["momentum_out"], p["weight"], p["master"], p["master_out"],
                                        p["out"], p["workspace"], need, blocks, c, b, 1, 0, None)

        own = {("momentum_out", "momentum"), ("master_out", "master"), ("out", "weight")}
        for o in outs:
            for other in names:
                if other == o or (other == "workspace" and not need):
                    continue
                # a step into it from below, and from within
                assert call(**{o: base[other] + size - 16}) == ALIAS, (o, other)
                assert call(**{o: base[other] - 16}) == ALIAS, (o, other)
                if (o, other) not in own and other not in outs:
                    assert call(**{o: base[other]}) == ALIAS, (o, other)


def test_norm_refuses_results_that_lie_in_operands(lib):
    from ksmm_amd._lib import KsmmNormDesc

    batch, features, groups = 12, 64, 3
    ins = ["x", "residual", "gate", "post", "weight", "bias"]
    at = dict(zip(ins, FAR))
    rows, vector = 4 * batch * features, 4 * features
    size = {"x": rows, "residual": rows, "gate": groups * vector, "post": vector, "weight": vector, "bias": vector, "stats": 16 * batch, "dr": rows,
            "dn": rows}
    desc = KsmmNormDesc(*(at[k] for k in ins), groups, 1.0, 1e-6, 0)
    outs = dict(zip(["r", "n", "stats"], FAR[6:]))

    def forward(**change):
        p = dict(outs, **change)
        return lib.ksmm_residual_norm_forward(ctypes.byref(desc), p["r"], p["n"], p["stats"], None, 0, batch, features, 0, 0, None)

    for o in outs:
        for other in ins:
            assert forward(**{o: at[other] + size[other] - 4}) == ALIAS, (o, other)
        for other in outs:
            if other != o:
                assert forward(**{o: outs[other]}) == ALIAS, (o, other)

    at.update(zip(["stats", "dr", "dn"], FAR[6:]))
    names = ["dx", "dresidual", "dgate", "dpost", "dweight", "dbias"]
    outs = dict(zip(names + ["workspace"], FAR[9:]))
    for bs_last in (0, 1):
        need = lib.ksmm_residual_norm_backward_workspace(batch, features, groups, 0, bs_last)

        def backward(**change):
            p = dict(outs, **change)
            return lib.ksmm_residual_norm_backward(ctypes.byref(desc), at["stats"], at["dr"], at["dn"], *(p[k] for k in names), p["workspace"], need,
                                                   batch, features, 0, bs_last, None)

        for o in outs:
            for other in at:
                # (a workspace's address is a multiple of 16)
                assert backward(**{o: at[other] + size[other] - 16}) == ALIAS, (o, other)
            for other in outs:
                if other != o:
                    assert backward(**{o: outs[other]}) == ALIAS, (o, other)


def test_update_refuses_sizes_whose_indexes_would_not_fit(lib):
    top = (1 << 31) - 1
    for blocks, c, b, parts in ((1, top, 1, 1), (1, 1, top, 1), (1, top - 100, 1, 1), (1, 1, 1, top), (1 << 62, 1, 1, 1), (top, 1, 1, 1),
                                (1, 46341, 46341, 1)):
        assert lib.ksmm_muon_workspace(blocks, c, b, parts) == -5, (blocks, c, b, parts)


@pytest.mark.parametrize("coefficients,steps,status", [
    ((3.4445, -4.7750, 2.0315), 5, -1), ((3.4445, -4.7750, 2.0315), 2000000000, -1), ((1.5, -0.5, 0.0), 100, -1), ((2.0, -1.5, 0.5), 30, -1),
    ((20.0, 0.0, 0.0), 2, -1), ((20.0, 0.0, 0.0), 3, -6), ((1.0, 0.0, 1e6), 1, -6), ((3.4445, -4.7750, 20.0), 5, -6), ((float("nan"), 0.0, 0.0), 1, -6),
    ((float("inf"), 0.0, 0.0), 1, -6), ((1.0, 0.0, 0.0), 2000000000, -1)])
def test_update_refuses_coefficients_whose_steps_leave_the_range(coefficients, steps, status, lib):
    """-1: accepted as far as the pointers, which are null here."""
    from ksmm_amd._lib import KsmmMuonDesc

    desc = KsmmMuonDesc((ctypes.c_float * 3)(*coefficients), 1e-7, 0.9, 1, 1, steps, 1)
    assert lib.ksmm_muon_update(ctypes.byref(desc), None, None, None, None, None, None, None, None, 0, 1, 8, 8, 1, 0, None) == status


def test_tied_factors_are_one():
    from ksmm_amd import KSGatedLinear, KSMuon

    first, second, other = (KSGatedLinear((2, 6, 4, 1), device="cpu") for _ in range(3))
    second.factor = first.factor
    found = KSMuon.factors_of(torch.nn.Sequential(first, second, other))
    assert [id(f[0]) for f in found] == [id(first.factor), id(other.factor)]


def optimizer(dtype):
    """KSMuon over one CPU parameter, made without its check that factors are on a GPU."""
    from ksmm_amd import KSMuon

    p = torch.nn.Parameter(torch.randn(8, 6).to(dtype))
    opt = KSMuon.__new__(KSMuon)
    torch.optim.Optimizer.__init__(opt, [{"params": [p], "pattern": (1, 6, 8, 1), "parts": 1}], dict(lr=0.02, master=True))
    return p, opt


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_state_is_loaded_in_32_bits(dtype):
    p, opt = optimizer(dtype)
    half = dtype == torch.float16
    opt.state[p] = {"momentum": torch.randn(8, 6), "master": torch.randn(8, 6) if half else None}
    saved = opt.state_dict()
    q, again = optimizer(dtype)
    seen = []
    again.register_load_state_dict_pre_hook(lambda o, s: seen.append("before"))
    again.register_load_state_dict_post_hook(lambda o: seen.append([v.dtype for v in o.state[q].values() if v is not None]))
    again.load_state_dict(saved)
    assert seen == ["before", [torch.float32] * (2 if half else 1)]
    assert list(again.state) == [q] and again.param_groups[0]["lr"] == 0.02
    for name, v in opt.state[p].items():
        if v is None:
            assert again.state[q][name] is None
        else:
            assert torch.equal(again.state[q][name], v) and again.state[q][name].data_ptr() != v.data_ptr()
    again.load_state_dict(saved)  # (the hooks it needs are gone: a second time is as the first)
    assert len(seen) == 4


def test_state_of_another_type_is_widened():
    """As an optimiser that was saved in 16 bits leaves it."""
    p, opt = optimizer(torch.float16)
    opt.state[p] = {"momentum": torch.randn(8, 6).half(), "master": torch.randn(8, 6).half()}
    q, again = optimizer(torch.float16)
    again.load_state_dict(opt.state_dict())
    assert all(v.dtype == torch.float32 for v in again.state[q].values())
    assert torch.equal(again.state[q]["momentum"], opt.state[p]["momentum"].float())
