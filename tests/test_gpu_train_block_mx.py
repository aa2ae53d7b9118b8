"""``python -m ksmm_amd.train_block`` with 4-bit products and AdamW beside KSMuon: it runs, and answers single rows as it does eagerly."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", [("--mx",), ("--mx", "--rest", "adamw", "--bits", "8"), ("--rest", "adamw"), ("--mx", "--bs-last", "1", "--rest", "adamw"),
                                 ("--mx", "--dtype", "fp32")])
def test_trains_and_answers(how, capsys):
    from ksmm_amd.train_block import main

    with torch.enable_grad():
        result = main(["--gated", "1,96,48,2", "--down", "1,48,96,2", "3,32,32,1", "--rows", "200", "--batches", "2", "--steps", "3", *how])
    assert all(math.isfinite(result[k]) for k in ("first_loss", "last_loss", "ms_per_step", "us_per_row"))
    assert result["graph_minus_eager"] == 0
    assert result["mx"] == ("--mx" in how)


def test_every_parameter_moves():
    from ksmm_amd.train_block import KSStack, train

    torch.manual_seed(0)
    model = KSStack((1, 96, 48, 2), [(1, 48, 96, 2)], 2, mx=True)
    before = [p.detach().clone() for p in model.parameters()]
    x = torch.randn(100, 96, device="cuda").half()
    train(model, [(x, x.roll(1, 0).contiguous())], 3, rest="adamw", bits=8)
    assert all(not torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(model.parameters(), before))
    packed = model.packed()
    assert torch.equal(packed(x), model(x))
