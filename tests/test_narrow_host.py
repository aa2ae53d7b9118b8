"""Host side of the 4-bit products and of AdamW without a GPU: what reaches the kernels, and how often."""
import pytest
import torch

from ksmm_amd import KSAdamW, _lib, adamw_update


class Native:
    """In place of the native module: its AdamW step has the status given."""

    def __init__(self, status):
        self.status, self.calls = status, 0

    def adamw_update(self, *args):
        self.calls += 1
        return self.status


def test_a_step_whose_launch_failed_is_not_made_again(monkeypatch):
    """Tables of tensors before the one that failed are updated: a second call would update them twice."""
    native = Native(-7)
    message = _lib.strerror(-7)
    monkeypatch.setattr(_lib, "native", lambda: native)
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("the step goes to the library a second time"))
    monkeypatch.setattr(_lib, "strerror", lambda status: message if status == -7 else pytest.fail(status))
    t = [torch.zeros(4)]
    with pytest.raises(_lib.KsmmError) as e:
        adamw_update(t, t, t, t)
    assert e.value.status == -7 and native.calls == 1
