"""Derivatives that the learner's operators do not have are refused, not dropped (the checks in front of the device, on the CPU)."""
import pytest
import torch
from torch.autograd import forward_ad

from sustaingym_amd import learner


@pytest.fixture(autouse=True)
def anywhere(monkeypatch):
    monkeypatch.setattr(learner, '_on_device', lambda name, t, device=None: None)


def test_forward_mode_tangents_are_refused():
    z, l, x = torch.zeros(4, 5), torch.zeros(4, dtype=torch.int64), torch.zeros(6, 4, 3)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for name, call in (('logits', lambda: learner.level_logprobs(dual(z), l)), ('x', lambda: learner.gated_scan(dual(x), 0.5)),
                           ('gate', lambda: learner.gated_scan(x, dual(x))), ('gate', lambda: learner.gated_scan(x, dual(x[:1, :1]))),
                           ('initial', lambda: learner.gated_scan(x, 0.5, dual(x[0])))):
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(ValueError, match=f'{name}: there is no forward-mode derivative'):
                    call()
