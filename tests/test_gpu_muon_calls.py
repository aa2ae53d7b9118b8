"""Orthogonalised updates: what a call makes of an error that an earlier one left."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pattern", [(2, 8, 16, 1), (1, 100, 60, 2), (1, 512, 384, 1)])
def test_an_error_from_before_is_not_the_updates_own(pattern):
    """The step is in place: it is made, and an error that is none of its launches' neither raised nor cleared."""
    from ksmm_amd import _lib, muon_update

    lib = _lib.load()
    a, b, c, d = pattern
    g = torch.Generator().manual_seed(0)
    first = [torch.randn(a * d * c, b, generator=g).cuda() for _ in range(3)]
    sets = [[t.clone() for t in first] for _ in range(2)]
    for (w, grad, m), before in zip(sets, (False, True)):
        torch.cuda.synchronize()
        if before:
            assert lib.hipSetDevice(1 << 20) != 0
        try:
            muon_update(w, grad, m, pattern, inplace=True)
        finally:
            left = lib.hipGetLastError()
        assert (left != 0) == before
    assert not torch.equal(sets[0][0], first[0]) and all(torch.equal(x, y) for x, y in zip(*sets))
