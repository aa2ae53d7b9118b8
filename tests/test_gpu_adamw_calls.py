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


def test_groups_round_apart():
    """Equal parameters with equal gradients in two groups, and of two types in one: their 8-bit moments are not rounded alike."""
    from ksmm_amd import KSAdamW

    g = torch.randn(4096, generator=torch.Generator().manual_seed(0)).cuda()
    for split in (True, False):
        ps = [torch.nn.Parameter(torch.zeros(4096, device="cuda", dtype=t)) for t in (torch.float32, torch.float32 if split else torch.float16)]
        opt = KSAdamW([{"params": [p]} for p in ps] if split else ps, bits=8, weight_decay=0.0)
        for p in ps:
            p.grad = g.half().to(p.dtype)
        opt.step()
        m, v = ([opt.state[p][k] for p in ps] for k in ("exp_avg", "exp_avg_sq"))
        # a value goes up with the probability p of its place between two codes: two of them differ with 2 p (1 - p), 1/3 on the mean of
        # all places (4096 of them: 0.007 off), which values of a normal distribution are not quite evenly at
        for x, y in (m, v):
            assert abs(float((x != y).float().mean()) - 1 / 3) <= 0.1
