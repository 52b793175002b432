"""An encoder in 8-bit integers (Wav2Vec2Model.quantize_int8) against its bf16 self.

Tolerance: a step of a row's integers is max|x| / 127; of 768 normal numbers the largest is about 3.5 standard deviations,
so an operand is off by 3.5 / 127 / sqrt(12) = 0.8 % (root mean square), a product of two by 1.1 %, and with a few larger
channels by twice that.  Each of a layer's two branches makes two such products in a row (1.6 - 3 %), added to a residual of
about its size: 2 % of a layer's output, growing with the square root of the layers through the norms -- 3 % after two,
taken as 6 %."""
import copy

import pytest
import torch

from dphubert_amd import kernels as K
from helpers import rel_l2

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cfg(family, layers=2, **kw):
    from dphubert_amd.synthetic import HUBERT_BASE_CONFIG, WAVLM_BASE_CONFIG
    c = copy.deepcopy(WAVLM_BASE_CONFIG if family == "wavlm" else HUBERT_BASE_CONFIG)
    c.update(encoder_num_layers=layers, encoder_use_attention=[True] * layers, encoder_use_feed_forward=[True] * layers,
             encoder_ff_interm_features=[1533, 1201][:layers] if family == "pruned" else [2048] * layers)
    if family == "wavlm":
        c.update(encoder_total_num_heads=[12] * layers, encoder_remaining_heads=[list(range(12))] * layers)
    elif family == "large":
        c.update(extractor_mode="layer_norm", encoder_embed_dim=1024, encoder_num_heads=[16] * layers,
                 encoder_layer_norm_first=True, encoder_ff_interm_features=[4096] * layers, normalize_waveform=True)
    else:
        c.update(encoder_num_heads=[7, 12][:layers] if family == "pruned" else [12] * layers)
    c.update(kw)
    return c


def _model(family, **kw):
    from dphubert_amd.trainer import seeded_model
    return seeded_model(_cfg(family, **kw), 3).to(DEV).eval()


def _wave(B=3, S=16000, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (0.1 * torch.randn(B, S, generator=g)).to(DEV), torch.tensor([S, S - 3000, S // 2][:B], device=DEV)


@pytest.mark.parametrize("family", ["hubert", "pruned", "wavlm", "large"])
def test_hidden_states_near_bf16(family):
    m = _model(family)
    w, ln = _wave()
    with torch.no_grad():
        want, lw = m.extract_features(w, ln)
        got, lg = m.quantize_int8().extract_features(w, ln)
        back, _ = m.quantize_int8(False).extract_features(w, ln)
    assert torch.equal(lw, lg) and len(want) == len(got) == 3
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape
        for u in range(len(ln)):
            n = int(lw[u])
            assert rel_l2(a[u, :n].float(), b[u, :n].float()) < 0.06, (i, u)
        if i:
            assert not torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(back, want))


def test_single_frame_and_sublayers_pruned_away():
    m = _model("hubert", encoder_use_attention=[False, True], encoder_use_feed_forward=[True, False])
    w, _ = _wave(1, 400)              # one frame
    with torch.no_grad():
        want, _ = m.extract_features(w)
        got, _ = m.quantize_int8().extract_features(w)
    assert got[-1].shape == (1, 1, 768)
    for a, b in zip(got, want):
        assert rel_l2(a.float(), b.float()) < 0.06


def test_weights_are_laid_out_again_when_they_change():
    m = _model("hubert", layers=1)
    w, ln = _wave()
    lay = m.encoder.transformer.layers[0]
    with torch.no_grad():
        m.quantize_int8()
        a = lay.int8_weights()
        assert lay.int8_weights()["qkv"] is a["qkv"]
        y = m.extract_features(w, ln)[0][-1]
        lay.attention.q_proj.weight.mul_(1.5)
        b = lay.int8_weights()
        assert b["qkv"] is not a["qkv"] and b["out"] is a["out"]
        assert torch.equal(b["qkv"].q, K.quant_rows_i8(torch.cat([lay.attention.q_proj.weight, lay.attention.k_proj.weight,
                                                                   lay.attention.v_proj.weight])).q)
        assert not torch.equal(m.extract_features(w, ln)[0][-1], y)


def test_weights_that_changed_unseen_are_laid_out_by_the_next_quantize():
    """A replayed optimiser step, or new storage, changes weights without their versions."""
    m = _model("hubert", layers=1).quantize_int8()
    a, lay = m.encoder.transformer.layers[0].int8_weights(), m.encoder.transformer.layers[0]
    g = torch.cuda.CUDAGraph()
    p = lay.feed_forward.output_dense.weight
    with torch.no_grad(), torch.cuda.graph(g):
        p.mul_(2.0)
    m.quantize_int8(False).quantize_int8()
    g.replay()
    b = m.quantize_int8(False).quantize_int8().encoder.transformer.layers[0].int8_weights()
    assert torch.equal(b["down"].scale, 2 * a["down"].scale)
    p.data = p.data * 3
    assert torch.equal(lay.int8_weights()["down"].q, K.quant_rows_i8(p.detach()).q)
    # another key projection (whose identity may be the freed one's)
    lay.attention.k_proj.weight = torch.nn.Parameter(torch.zeros_like(lay.attention.k_proj.weight))
    assert not lay.int8_weights()["qkv"].q[768:1536].any()


def test_forward_only():
    m = _model("hubert", layers=1).quantize_int8()
    w, ln = _wave()
    with pytest.raises(RuntimeError, match="forward only"):
        m.extract_features(w, ln)                     # gradients wanted
    with torch.no_grad():
        m.train()
        with pytest.raises(RuntimeError, match="forward only"):
            m.extract_features(w, ln)
        m.eval()
        m.extract_features(w, ln)


def test_captured_forward():
    m = _model("large", layers=1, normalize_waveform=False).quantize_int8()
    w, ln = _wave()
    with torch.no_grad():
        want = [h.clone() for h in m.extract_features(w, ln)[0]]
        held = w.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got, _ = m.extract_features(held, ln)
        for k in range(3):
            held.copy_(w.flip(0) if k == 1 else w)
            g.replay()
            eager, _ = m.extract_features(held, ln)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_distill_step_with_int8_teacher():
    """The loss against an int8 teacher is near the bf16 teacher's, and the student's gradients are all there."""
    from dphubert_amd.trainer import build_distill_module
    cfg = _cfg("hubert", encoder_projection_dropout=0.0, encoder_attention_dropout=0.0, encoder_dropout=0.0, encoder_layer_drop=0.0)
    losses = []
    for int8 in (False, True):
        dm = build_distill_module(cfg, use_reg=False, distill_layers="0.1,2", seed=3).to(DEV)
        if int8:
            dm.teacher_model.quantize_int8()
        dm.train()
        loss = dm._step(_wave(), 0, "train")
        loss.backward()
        losses.append(loss.item())
        assert all(p.grad is not None and p.grad.isfinite().all() for p in dm.student_model.parameters() if p.requires_grad)
    # L1 and cosine of two nearly equal models: the bf16 teacher is the student itself (L1 0, cosine 1), the int8 one is a
    # few per cent off, |s - t| a few per cent of |t| ~ 1
    assert abs(losses[0] - losses[1]) < 0.2 and losses[1] > losses[0]
