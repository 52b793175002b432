"""An encoder layer in 8-bit integers refuses a forward whose gradients are wanted, whoever wants them."""
import copy

import pytest
import torch


def _layer(family):
    from dphubert_amd.synthetic import HUBERT_BASE_CONFIG, WAVLM_BASE_CONFIG
    from dphubert_amd.trainer import seeded_model
    c = copy.deepcopy(WAVLM_BASE_CONFIG if family == "wavlm" else HUBERT_BASE_CONFIG)
    c.update(encoder_num_layers=2, encoder_use_attention=[True] * 2, encoder_use_feed_forward=[True] * 2, encoder_ff_interm_features=[256] * 2)
    if family == "wavlm":
        c.update(encoder_total_num_heads=[12] * 2, encoder_remaining_heads=[list(range(12))] * 2)
    else:
        c.update(encoder_num_heads=[12] * 2)
    layer = seeded_model(c, 3).eval().encoder.transformer.layers[1]
    layer.requires_grad_(False)
    layer.int8 = True
    return layer


@pytest.mark.parametrize("family", ["hubert", "wavlm"])
def test_gradients_wanted_by_what_lies_before_a_frozen_layer(family, monkeypatch):
    from dphubert_amd import ops
    monkeypatch.setattr(ops, "encoder_layer_int8", lambda cfg, h, layer, wl: h.detach())
    layer = _layer(family)
    x = torch.randn(1, 4, 768)
    with pytest.raises(RuntimeError, match="forward only"):
        layer(x.clone().requires_grad_())
    if family == "wavlm":
        with pytest.raises(RuntimeError, match="forward only"):
            layer(x, position_bias=torch.randn(12, 4, 4, requires_grad=True))
    for grad, t in ((True, x), (False, x.clone().requires_grad_())):
        with torch.set_grad_enabled(grad):
            assert torch.equal(layer(t)[0], t)
