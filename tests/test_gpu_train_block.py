"""The gated feed-forward blocks, their norms and the optimiser together: training lowers the loss, and a captured single row
answers what the eager one does."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bs_last", [("fp16", 0), ("fp32", 0), ("fp16", 1), ("fp32", 1)])
def test_blocks_learn_and_answer(dtype, bs_last):
    from ksmm_amd import train_block

    result = train_block.main(["--gated", "1,96,32,2", "--down", "1,32,96,2", "4,16,16,1", "--blocks", "2", "--rows", "200", "--steps", "60",
                               "--batches", "4", "--dtype", dtype, "--bs-last", str(bs_last)])
    assert result["last_loss"] < 0.5 * result["first_loss"]
    assert result["graph_minus_eager"] == 0.0


def test_replays_between_other_work():
    import torch
    from ksmm_amd import train_block

    torch.manual_seed(1)
    model = train_block.KSStack((1, 96, 32, 2), [(1, 32, 96, 2)], 1)
    one = train_block.OneRow(model, 64, torch.float16)
    for i in range(6):
        row = torch.randn(1, 64, device="cuda").half()
        with torch.no_grad():
            want = model(row)
            model(torch.randn(64, 64, device="cuda").half())
        torch.cuda.synchronize()
        assert torch.equal(one(row), want), i
