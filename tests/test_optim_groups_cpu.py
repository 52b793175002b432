"""The optimisers hold the scalars of four parameter groups: a fifth is refused when it is added, not at the next step."""
import pytest
import torch

from dphubert_amd.optim import FusedAdamW, FusedMuon


def _g(**kw):
    return dict(params=[torch.nn.Parameter(torch.randn(3, 4))], **kw)


@pytest.mark.parametrize("make", [lambda: FusedAdamW([_g() for _ in range(4)]), lambda: FusedMuon([_g(muon=True) for _ in range(4)])])
def test_a_fifth_group_is_refused_and_leaves_the_four(make):
    o = make()
    for group in (_g(), _g(muon=True)):
        with pytest.raises(ValueError, match="at most 4"):
            o.add_param_group(group)
    assert len(o.param_groups) == 4


@pytest.mark.parametrize("cls", [FusedAdamW, FusedMuon])
def test_five_groups_at_once_are_refused(cls):
    with pytest.raises(ValueError, match="at most 4"):
        cls([_g() for _ in range(5)])
