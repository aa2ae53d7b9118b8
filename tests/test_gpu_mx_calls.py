"""Products of 4-bit numbers: calls beside the ordinary ones."""
import pytest
import torch

from tests import mx_ref as R
from tests.test_gpu_mx import DT, TOL, factor, factor_rows, rel, rows

pytestmark = pytest.mark.gpu


def test_a_given_result_counts_as_written():
    """A graph that holds the memory that a result went into raises."""
    from ksmm_amd import MXKernel, pack_mx

    pattern = (1, 40, 64, 1)
    w = pack_mx(factor(pattern, False, torch.float32).cuda(), pattern)
    x = rows(5, 64, False, torch.float32).cuda()
    out = torch.zeros(5, 40, device="cuda")
    before = out._version
    assert MXKernel.forward(x, w, out=out) is out and out._version == before + 1
    with torch.enable_grad():
        leaf = torch.ones(5, 40, device="cuda", requires_grad=True)
        y = leaf * out
        MXKernel.forward(x, w, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():  # (tensors without a count)
        out = torch.empty(5, 40, device="cuda")
        assert torch.equal(MXKernel.forward(x, w, out=out), MXKernel.forward(x, w))
