"""A Muon group's ``momentum``, changed between steps (a warm-up), is what the next step uses."""
import pytest
import torch

from dphubert_amd import optim
from dphubert_amd.optim import FusedMuon


def _opt():
    return FusedMuon([{"params": [torch.nn.Parameter(torch.randn(3))]},
                      {"params": [torch.nn.Parameter(torch.randn(3, 4))], "muon": True, "momentum": 0.85}])


def test_changed_momentum_reaches_the_kernels_scalars(monkeypatch):
    o = _opt()
    seen = []
    monkeypatch.setattr(optim.FusedAdamW, "launch", lambda self: seen.append([g["betas"][0] for g in self.param_groups]))
    for m in (0.85, 0.9, 0.95):
        o.param_groups[1]["momentum"] = m
        o.begin_step()                       # (what the per-step upload reads afterwards)
        assert o.param_groups[1]["betas"][0] == m
        o.launch()
    o.param_groups[1]["momentum"] = 0.5      # a launch alone
    o.launch()
    assert seen == [[0.9, 0.85], [0.9, 0.9], [0.9, 0.95], [0.9, 0.5]]


@pytest.mark.parametrize("bad", [1.0, -0.1, float("nan")])
def test_refused_before_anything_is_stepped(bad):
    o = _opt()
    o.param_groups[1]["momentum"] = bad
    for f in (o.begin_step, o.launch, o.step):
        with pytest.raises(ValueError, match="momentum"):
            f()
    assert o._step == 0


def test_loaded_groups_bring_theirs():
    a, b = _opt(), _opt()
    a.param_groups[1]["momentum"] = 0.7
    b.load_state_dict(a.state_dict())
    b.begin_step()
    assert b.param_groups[1]["betas"][0] == 0.7
