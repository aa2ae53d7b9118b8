"""Host side of the operators around a feed-forward block: argument checks of the C ABI, layouts, module wiring (no GPU)."""
import ctypes

import pytest
import torch

from ksmm_amd import KSMuon, generate_factor, pack_gated


@pytest.mark.parametrize("change,status", [
    ({}, -1), ({"batch": 0}, -3), ({"a": 0}, -2), ({"b": 1 << 30}, -5), ({"dtype": 2}, -4), ({"dtype": 9}, -4), ({"act": 7}, -12),
    ({"batch": 1 << 40}, -5)])
def test_gated_codes(lib, change, status):
    how = dict(batch=4, a=1, b=8, c=8, d=2, dtype=0, act=2)
    how.update(change)
    a = (how["batch"], how["a"], how["b"], how["c"], how["d"], how["dtype"], 0)
    # (null pointers are found last: nothing is launched)
    assert lib.ksmm_gated_forward(None, None, None, None, *a, how["act"], None) == status
    assert lib.ksmm_gated_backward(None, None, None, None, None, None, None, None, 0, *a, how["act"], None) == status
    if "act" not in change:
        need = lib.ksmm_gated_backward_workspace(*a)
        assert need == status if status != -1 else need >= 4 * 2 * 8 * 2 * 4


def test_gated_backward_refuses_a_small_workspace(lib):
    p = ctypes.c_void_p(64)
    need = lib.ksmm_gated_backward_workspace(4, 1, 8, 8, 2, 1, 0)
    for ws, size in ((None, need), (p, need - 1), (ctypes.c_void_p(72), need)):
        assert lib.ksmm_gated_backward(p, p, p, None, p, p, None, ws, size, 4, 1, 8, 8, 2, 1, 0, 2, None) == -9


@pytest.mark.parametrize("change,status", [
    ({}, -1), ({"batch": 0}, -3), ({"features": 0}, -3), ({"groups": 3}, -3), ({"groups": 0}, -3), ({"dtype": 2}, -4), ({"kind": 5}, -12),
    ({"residual": None}, -1), ({"features": 16385}, -5)])
def test_norm_codes(lib, change, status):
    from ksmm_amd._lib import KsmmNormDesc

    how = dict(batch=4, features=16, groups=1, dtype=0, kind=0, residual=64)
    how.update(change)
    desc = KsmmNormDesc(None, how["residual"], None, None, None, None, how["groups"], 1.0, 1e-6, how["kind"])
    assert lib.ksmm_residual_norm_forward(ctypes.byref(desc), None, None, None, None, 0, how["batch"], how["features"], how["dtype"], 0, None) == status
    assert lib.ksmm_residual_norm_backward(ctypes.byref(desc), None, None, None, None, None, None, None, None, None, None, 0, how["batch"],
                                           how["features"], how["dtype"], 0, None) == status
    assert lib.ksmm_residual_norm_forward(None, None, None, None, None, 0, 1, 1, 0, 0, None) == -1


def test_norm_backward_refuses_gradients_of_what_is_not_there(lib):
    from ksmm_amd._lib import KsmmNormDesc

    p = ctypes.c_void_p(64)
    desc = KsmmNormDesc(None, 64, None, None, None, None, 1, 1.0, 1e-6, 0)
    need = lib.ksmm_residual_norm_backward_workspace(4, 16, 1, 0, 0)
    assert need > 0
    for i in range(6):
        outs = [p if j == i else None for j in range(6)]
        want = -9 if i == 1 else -1  # (dresidual is always there: the call gets to its workspace)
        assert lib.ksmm_residual_norm_backward(ctypes.byref(desc), p, None, p, *outs, None, 0, 4, 16, 0, 0, None) == want


@pytest.mark.parametrize("change,status", [
    ({}, -1), ({"blocks": 0}, -2), ({"c": 0}, -2), ({"parts": 0}, -2), ({"dtype": 2}, -4), ({"steps": 0}, -6), ({"blocks": 1 << 40}, -5)])
def test_muon_codes(lib, change, status):
    from ksmm_amd._lib import KsmmMuonDesc

    how = dict(blocks=2, c=8, b=8, parts=1, dtype=0, steps=5)
    how.update(change)
    desc = KsmmMuonDesc((ctypes.c_float * 3)(1, 0, 0), 1e-7, 0.9, 1, 1, how["steps"], 1)
    assert lib.ksmm_muon_update(ctypes.byref(desc), None, None, None, None, None, None, None, None, 0, how["blocks"], how["c"], how["b"],
                                how["parts"], how["dtype"], None) == status
    assert lib.ksmm_muon_update(None, None, None, None, None, None, None, None, None, 0, 1, 8, 8, 1, 0, None) == -1


def test_muon_workspace_of_blocks_that_fit_a_compute_unit_and_of_larger_ones(lib):
    from ksmm_amd._lib import KsmmMuonDesc

    assert lib.ksmm_muon_workspace(100, 64, 64, 2) == 0 and lib.ksmm_muon_workspace(100, 16, 256, 1) == 0
    need = lib.ksmm_muon_workspace(2, 384, 1536, 2)
    assert need >= 4 * 2 * 2 * 384 * 1536
    desc = KsmmMuonDesc((ctypes.c_float * 3)(1, 0, 0), 1e-7, 0.9, 1, 1, 5, 1)
    p = ctypes.c_void_p(64)
    assert lib.ksmm_muon_update(ctypes.byref(desc), p, None, None, None, None, None, p, p, need - 1, 2, 384, 1536, 2, 0, None) == -9


def test_packed_weights_are_one_factor_of_twice_the_outputs():
    """What the gradients run on: kernel format of pattern (a, 2b, c, d)."""
    a, b, c, d = 2, 3, 4, 5
    gate, up = torch.randn(a, b, c, d), torch.randn(a, b, c, d)
    both = torch.cat([gate, up], 1)
    assert torch.equal(pack_gated(gate, up, torch.float32), generate_factor(a, 2 * b, c, d, "kernel", both, torch.float32))


def test_muon_takes_the_factors_of_kernel_layers():
    from ksmm_amd import KSGatedLinear, KSLinear

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gated = KSGatedLinear((2, 6, 4, 1), device="cpu")
            self.dense = KSLinear([(1, 4, 4, 1)], algo="dense")

    model = Model()
    found = KSMuon.factors_of(model)
    assert len(found) == 1 and found[0][0] is model.gated.factor and found[0][1:] == ((2, 6, 4, 1), 2)
    assert {id(p) for p in KSMuon.others(model)} == {id(p) for p in model.parameters()} - {id(model.gated.factor)}
    with pytest.raises(RuntimeError):
        model.gated(torch.randn(3, 8).half())


def test_norms_in_steps_need_a_workspace(lib):
    from ksmm_amd._lib import KsmmNormDesc

    assert lib.ksmm_residual_norm_forward_workspace(25088, 768, 1, 0) == 0 and lib.ksmm_residual_norm_forward_workspace(500, 384, 0, 1) == 0
    need = lib.ksmm_residual_norm_forward_workspace(500, 8000, 1, 1)
    assert need >= 500 * 8000 // 256 * 16
    desc, p = KsmmNormDesc(64, 64, None, None, None, None, 1, 1.0, 1e-6, 0), ctypes.c_void_p(64)
    assert lib.ksmm_residual_norm_forward(ctypes.byref(desc), p, p, None, p, need - 1, 500, 8000, 1, 1, None) == -9


def test_train_block_refuses_nothing_to_do():
    from ksmm_amd import train_block

    assert train_block.pattern("1,2,3,4") == (1, 2, 3, 4)
    for bad in (["--steps", "0"], ["--rows", "0"], ["--dtype", "fp8"]):
        with pytest.raises(SystemExit):
            train_block.main(bad)


def test_outputs_that_lie_in_inputs_are_refused(lib):
    from ksmm_amd._lib import KsmmNormDesc

    f = lib.ksmm_gated_forward  # 4 rows of 8 features -> 8 in fp32: 128 bytes each, 512 of weights
    assert f(4096, 8192, None, 4096 + 64, 4, 1, 8, 8, 1, 0, 0, 2, None) == -11
    assert f(4096, 8192, None, 8192 + 500, 4, 1, 8, 8, 1, 0, 0, 2, None) == -11
    assert f(4096, 8192, 16384, 16384 + 60, 4, 1, 8, 8, 1, 0, 0, 2, None) == -11
    need = lib.ksmm_gated_backward_workspace(4, 1, 8, 8, 1, 0, 0)
    g = lib.ksmm_gated_backward
    assert g(1 << 20, 1 << 21, 1 << 22, None, 1 << 23, (1 << 23) + 64, None, 1 << 24, need, 4, 1, 8, 8, 1, 0, 0, 2, None) == -11
    assert g(1 << 20, 1 << 21, 1 << 22, None, 1 << 23, None, None, (1 << 20) - 16, need, 4, 1, 8, 8, 1, 0, 0, 2, None) == -11
    desc = KsmmNormDesc(1 << 20, 1 << 21, None, None, None, None, 1, 1.0, 1e-6, 0)
    n = lib.ksmm_residual_norm_forward
    for r, out in ((1 << 20, 1 << 22), ((1 << 21) + 60, 1 << 22), (1 << 22, 1 << 22), (1 << 22, 1 << 21)):
        assert n(ctypes.byref(desc), r, out, None, None, 0, 4, 8, 0, 0, None) == -11
    need = lib.ksmm_residual_norm_backward_workspace(4, 8, 1, 0, 0)
    for dx, dr in ((1 << 20, 1 << 23), (1 << 23, 1 << 22), (1 << 23, (1 << 23) + 4)):
        assert lib.ksmm_residual_norm_backward(ctypes.byref(desc), 1 << 19, 1 << 22, None, dx, dr, None, None, None, None, 1 << 24, need, 4, 8, 0, 0,
                                               None) == -11
