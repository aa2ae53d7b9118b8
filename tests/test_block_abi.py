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
