"""AdamW over many tensors: how often a step is made, and what its calls leave behind."""
import pytest
import torch

from tests.test_gpu_adamw import HOW, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("bits", [8, 32])
def test_an_error_from_before_is_not_the_steps_own(monkeypatch, bits, native):
    """An error that an earlier call on the thread left is neither taken for the launch's (the step would be made twice) nor cleared."""
    from ksmm_amd import _lib, adamw_moments, adamw_update

    lib = _lib.load()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    _lib.native()
    sets = [make([300, 40], "fp16", bits, True) for _ in range(2)]
    decoded = []
    for s, before in zip(sets, (False, True)):
        torch.cuda.synchronize()
        if before:
            assert lib.hipSetDevice(1 << 20) != 0
        try:
            adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], s["master"], step=3, **HOW)
            decoded.append(adamw_moments(s["m"], s["v"], s["scales"]) if bits == 8 else None)
        finally:
            left = lib.hipGetLastError()
        assert (left != 0) == before
    for k in ("w", "m", "v", "master") + (("scales",) if bits == 8 else ()):
        assert all(torch.equal(x, y) for x, y in zip(sets[0][k], sets[1][k])), k
    if bits == 8:
        assert all(torch.equal(x, y) for one, other in zip(*decoded) for x, y in zip(one, other))
