"""optim.FusedMuon against its formulas in 64 bits, as an optimiser of its own and inside the trainer.

Tolerance of a step: the direction's (an element within 2^-8 of itself and 8 standard deviations of 2.5e-3 of the root
mean square, tests/test_newton_schulz_gpu.py) times lr 0.2 sqrt(max(rows, columns)), and 6 fp32 roundings (2^-24) of the
parameter and of the step."""
import copy
import math

import pytest
import torch

from dphubert_amd import ops
from dphubert_amd.optim import FusedAdamW, FusedMuon
from test_newton_schulz_gpu import exact

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def params(shapes, g, scale=0.05):
    return [torch.nn.Parameter((torch.randn(*s, generator=g) * scale).to(DEV)) for s in shapes]


@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_against_the_formulas(nesterov):
    g = gen(1)
    mats, rest = params([(96, 64), (64, 200), (50, 3), (33, 4, 5), (1, 9), (130, 131)], g), params([(64,), (7, 5)], g)
    adam = [p.detach().clone().requires_grad_(True) for p in rest]
    opt = FusedMuon([{"params": rest, "lr": 1e-2, "weight_decay": 0.1},
                     {"params": mats, "lr": 2e-2, "weight_decay": 0.05, "muon": True, "momentum": 0.9}],
                    max_grad_norm=1.0, nesterov=nesterov)
    plain = FusedAdamW([{"params": adam, "lr": 1e-2, "weight_decay": 0.1}])
    want = [p.detach().cpu().double() for p in mats]
    mom = [torch.zeros_like(w) for w in want]
    slack = [torch.zeros_like(w) for w in want]
    for step in range(4):
        grads = [torch.randn(*p.shape, generator=g) * (3.0 if step % 2 else 1e-3) for p in rest + mats]
        norm = math.sqrt(sum(t.double().square().sum().item() for t in grads))
        clip = min(1.0, 1.0 / (norm + 1e-6))
        for p, t in zip(rest + mats, grads):
            p.grad = t.to(DEV)
        for p, t in zip(adam, grads):
            p.grad = (t * clip).to(DEV)
        opt.step()
        plain.step()
        for k, (t, p) in enumerate(zip(grads[len(rest):], mats)):
            t = t.double() * clip
            mom[k] += (t - mom[k]) * (1 - 0.9)
            u = (t + (mom[k] - t) * 0.9 if nesterov else mom[k]).reshape(t.shape[0], -1)
            o = exact(u).reshape(t.shape)
            scale = 0.2 * math.sqrt(max(u.shape)) * 2e-2
            want[k] = want[k] * (1 - 2e-2 * 0.05) - scale * o
            slack[k] += scale * (o.abs() * 2.0 ** -8 + 8 * 2.5e-3 * o.square().mean().sqrt()) + \
                6 * 2.0 ** -24 * (want[k].abs() + scale * o.abs())
            got = p.detach().cpu().double()
            assert ((got - want[k]).abs() <= slack[k]).all(), (step, tuple(p.shape))
            assert torch.allclose(opt.state[p]["momentum_buffer"].cpu().double(), mom[k], rtol=1e-5, atol=1e-9)
            assert torch.allclose(p.grad.cpu().double(), t, rtol=1e-5, atol=0)      # clipped in place, as AdamW's
    for p, q in zip(rest, adam):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-7)


def test_parameter_without_gradient_is_left_alone():
    g = gen(2)
    a, b = params([(40, 30), (40, 30)], g)
    opt = FusedMuon([{"params": [a, b], "lr": 1e-2, "weight_decay": 0.1, "muon": True}])
    before = b.detach().clone()
    a.grad = torch.randn_like(a)
    opt.step()
    assert torch.equal(b, before) and not opt.state[b]["momentum_buffer"].any()
    moved = a.detach().clone()
    a.grad, b.grad = None, torch.randn_like(b)
    opt.step()
    assert torch.equal(a, moved) and not torch.equal(b, before)


def test_group_added_after_a_step_moves():
    g = gen(12)
    a, b, c = params([(40, 30), (7,), (20, 50)], g)
    opt = FusedMuon([{"params": [a], "lr": 1e-2, "muon": True}])
    a.grad = torch.randn_like(a)
    opt.step()
    opt.add_param_group({"params": [b], "lr": 1e-2, "weight_decay": 0.0})
    for add in (None, {"params": [c], "lr": 1e-2, "muon": True}):
        if add:
            opt.add_param_group(add)
        ps = [a, b, c] if add else [a, b]
        old = [p.detach().clone() for p in ps]
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
        assert all((p != q).any() for p, q in zip(ps, old))


def test_writes_bf16_images():
    g = gen(3)
    ps = params([(96, 64), (96, 64), (96, 64), (50, 3)], g)
    img = ops.bf16_image(*ps[:3])
    odd = ops.bf16_image(ps[3])
    opt = FusedMuon([{"params": ps, "lr": 1e-2, "muon": True}])
    for _ in range(2):
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
    assert ops.bf16_image(*ps[:3]).data_ptr() == img.data_ptr()
    assert torch.equal(ops.bf16_image(*ps[:3]), torch.cat([p.detach() for p in ps[:3]]).bfloat16())
    assert ops.bf16_image(ps[3]).data_ptr() == odd.data_ptr() and torch.equal(odd, ps[3].detach().bfloat16())


def test_state_dict_resumes():
    g = gen(4)
    grads = [torch.randn(60, 44, generator=g).to(DEV) for _ in range(4)]
    a = params([(60, 44)], gen(5))[0]
    b = a.detach().clone().requires_grad_(True)
    oa = FusedMuon([{"params": [a], "lr": 1e-2, "muon": True, "momentum": 0.8}])
    for t in grads[:2]:
        a.grad = t.clone()
        oa.step()
    with torch.no_grad():
        b.copy_(a)
    ob = FusedMuon([{"params": [b], "lr": 1e-2, "muon": True}])
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for t in grads[2:]:
        a.grad, b.grad = t.clone(), t.clone()
        oa.step()
        ob.step()
    assert torch.equal(a, b) and ob.param_groups[0]["momentum"] == 0.8


def _trainer(graphs, **kw):
    from test_graph_gpu import _cfg
    from dphubert_amd.synthetic import seeded_tensor
    from dphubert_amd.trainer import Trainer, build_distill_module
    dm = build_distill_module(_cfg(), pruning_units="conv,head,interm", distill_layers="0.1,2", seed=3, learning_rate=2e-3,
                              warmup_updates=2, max_updates=10, sparsity_warmup_updates=4, optimizer="muon")
    with torch.no_grad():
        dm.lambda1.fill_(0.3)
        dm.lambda2.fill_(0.2)
        for n, p in dm.student_model.named_parameters():
            if "log_alpha" not in n and p.numel() > 1:
                p.add_(0.1 * p.abs().mean() * seeded_tensor("offset." + n, tuple(p.shape), 4).sign())
    dm.global_step = 1
    g = torch.Generator().manual_seed(11)
    dm = dm.to(DEV)
    for name, mod in dm.student_model.named_modules():
        if hasattr(mod, "set_noise"):
            mod.set_noise((torch.rand(mod.log_alpha.shape, generator=g) * 0.98 + 0.01).to(DEV))
    if kw.get("teacher_int8"):
        dm.teacher_model.quantize_int8()
    return Trainer(dm, clip_norm=10.0, graphs=graphs, graph_warmup=1)


@pytest.mark.parametrize("teacher_int8", [False, True])
def test_trainer_graph_replay_matches_eager(teacher_int8):
    """Muon steps (and the int8 teacher) captured into the step graphs: losses and parameters bitwise those of eager
    steps, with the two trainers' steps interleaved."""
    from test_graph_gpu import _batch
    from dphubert_amd import _lib
    prev = _lib.deterministic()
    _lib.set_deterministic(True)
    try:
        batch = _batch()
        ea, gr = _trainer(False, teacher_int8=teacher_int8), _trainer(True, teacher_int8=teacher_int8)
        before = {n: p.detach().clone() for n, p in gr.module.student_model.named_parameters()}
        for step in range(5):
            le, lg = ea.step(batch).item(), gr.step(batch).item()
            assert le == lg and math.isfinite(le), step
        torch.cuda.synchronize()
        assert gr._graph is not None
        assert isinstance(gr.optimizer, FusedMuon)
        for (n, p), (_, q) in zip(ea.module.named_parameters(), gr.module.named_parameters()):
            assert torch.equal(p, q), n
        for p in gr.optimizer.param_groups[-1]["params"]:
            n = next(k for k, v in gr.module.student_model.named_parameters() if v is p)
            assert not torch.equal(p, before[n]), n
    finally:
        _lib.set_deterministic(prev)
