"""FusedMuon's arguments and where it stands in the framework (no device needed)."""
import copy

import pytest
import torch

from dphubert_amd.optim import FusedAdamW, FusedMuon


def _p(*s):
    return torch.nn.Parameter(torch.randn(*s))


@pytest.mark.parametrize("group", [[_p(5)], [_p(3, 4), torch.nn.Parameter(torch.randn(()))], [_p(0, 3)],
                                   [torch.nn.Parameter(torch.randn(3, 4).bfloat16())], [torch.nn.Parameter(torch.randn(4, 3).t())]])
def test_refuses_what_is_no_matrix(group):
    with pytest.raises(ValueError):
        FusedMuon([{"params": group, "muon": True}])


@pytest.mark.parametrize("kw", [dict(momentum=1.0), dict(momentum=-0.1), dict(ns_steps=0), dict(ns_steps=65)])
def test_refuses_bad_settings(kw):
    with pytest.raises(ValueError):
        FusedMuon([{"params": [_p(3, 4)], "muon": True}], **kw)


def test_groups_keep_their_settings():
    o = FusedMuon([{"params": [_p(3)]}, {"params": [_p(3, 4), _p(2, 3, 3)], "muon": True, "momentum": 0.8}], momentum=0.9)
    assert o.param_groups[0]["betas"] == (0.9, 0.999) and o.param_groups[1]["betas"][0] == 0.8
    assert o._state_keys(0) == ("exp_avg", "exp_avg_sq") and o._state_keys(1) == ("momentum_buffer",)
    o = FusedMuon([{"params": [_p(3, 4)], "muon": True}], momentum=0.9)
    assert o.param_groups[0]["momentum"] == 0.9


def test_groups_added_later_are_checked_too():
    o = FusedMuon([{"params": [_p(3, 4)], "muon": True}], momentum=0.9)
    o.add_param_group({"params": [_p(5, 4)], "muon": True})
    o.add_param_group({"params": [_p(5)]})
    assert o.param_groups[1]["momentum"] == 0.9 and o.param_groups[1]["betas"] == (0.9, 0.0) and not o._is_muon(2)
    for bad in ({"params": [_p(5)], "muon": True}, {"params": [_p(5, 2)], "muon": True, "momentum": 1.0}):
        with pytest.raises(ValueError):
            o.add_param_group(bad)
    assert len(o.param_groups) == 3


def _module(**kw):
    from dphubert_amd.synthetic import HUBERT_BASE_CONFIG
    from dphubert_amd.trainer import build_distill_module
    cfg = copy.deepcopy(HUBERT_BASE_CONFIG)
    cfg.update(encoder_num_layers=1, encoder_use_attention=[True], encoder_use_feed_forward=[True], encoder_num_heads=[12],
               encoder_ff_interm_features=[256])
    return build_distill_module(cfg, distill_layers="0.1", **kw)


def test_distill_module_chooses_the_optimizer():
    m = _module(optimizer="muon", muon_momentum=0.9)
    o = m.configure_optimizers(clip_norm=10.0)["optimizer"]
    assert isinstance(o, FusedMuon) and [g["name"] for g in o.param_groups] == ["main_params", "log_alpha", "lambda", "muon"]
    mats = o.param_groups[3]["params"]
    assert sorted(tuple(p.shape) for p in mats) == sorted([(768, 768)] * 4 + [(256, 768), (768, 256)])
    assert o.param_groups[3]["momentum"] == 0.9 and o.param_groups[3]["lr"] == o.param_groups[0]["lr"]
    every = [p for g in o.param_groups for p in g["params"]]
    plain = _module().configure_optimizers(clip_norm=10.0)["optimizer"]
    assert type(plain) is FusedAdamW and len(plain.param_groups) == 3
    assert len({id(p) for p in every}) == len(every) == sum(len(g["params"]) for g in plain.param_groups)
    with pytest.raises(ValueError):
        _module(optimizer="sgd")


def test_flags():
    from dphubert_amd.cli import distill_parser, final_distill_parser
    for p in (distill_parser(), final_distill_parser()):
        a = p.parse_args([])
        assert a.optimizer == "adamw" and not a.teacher_int8 and a.muon_momentum == 0.95
        a = p.parse_args(["--optimizer", "muon", "--teacher_int8", "--muon_momentum", "0.9"])
        assert a.optimizer == "muon" and a.teacher_int8 and a.muon_momentum == 0.9


def test_quantize_int8_refuses_on_the_host_and_with_gates():
    m = _module()
    with pytest.raises(ValueError, match="device"):
        m.teacher_model.quantize_int8()
    with pytest.raises(ValueError, match="gates"):
        m.student_model.quantize_int8()
    m.teacher_model.quantize_int8(False)
    assert not any(layer.int8 for layer in m.teacher_model.encoder.transformer.layers)
