"""Captured FusedMuon steps replayed after what they read has moved: bitwise the steps that a second optimiser, on clones,
takes eagerly (every kernel of a step adds in a fixed order)."""
import copy

import pytest
import torch

from dphubert_amd.optim import FusedMuon

pytestmark = pytest.mark.gpu
SHAPES = [(96, 64), (64, 200), (130, 131), (7,)]


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _params():
    g = gen(5)
    return [torch.nn.Parameter((torch.randn(*s, generator=g) * 0.05).cuda()) for s in SHAPES]


def _opt(ps):
    return FusedMuon([{"params": ps[:3], "lr": 1e-2, "weight_decay": 0.1, "muon": True},
                      {"params": ps[3:], "lr": 1e-2, "weight_decay": 0.0}], max_grad_norm=1e9)


def _grads(ps, seed):
    g = gen(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).cuda()


def _same(a, b):
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def _captured():
    """(parameters, optimiser, its captured step) and the eager pair, both after one step."""
    a, b = _params(), _params()
    oa, ob = _opt(a), _opt(b)
    for ps, o in ((a, oa), (b, ob)):
        _grads(ps, 1)
        o.step()
    graph = torch.cuda.CUDAGraph()
    oa.begin_step()
    with torch.cuda.graph(graph):
        oa.launch()
    return a, oa, graph, b, ob


def _replay(graph, ob):
    """The captured AdamW step is the second one whatever came before (its count is an argument): so is the eager one."""
    graph.replay()
    ob._step = 1
    ob.step()


def test_gradients_that_moved():
    a, oa, graph, b, ob = _captured()
    _replay(graph, ob)
    _same(a, b)
    for seed in (2, 3):
        oa._step = ob._step = seed
        for ps, o in ((a, oa), (b, ob)):
            _grads(ps, seed)             # (the old ones' memory is free for others)
            o.step()
        junk = [torch.full((1 << 16,), float("nan"), device="cuda") for _ in range(16)]
        _replay(graph, ob)
        _same(a, b)
        assert len(junk) == 16


def test_states_that_were_loaded():
    a, oa, graph, b, ob = _captured()
    for ps, o in ((a, oa), (b, ob)):
        o.load_state_dict(copy.deepcopy(o.state_dict()))
        _grads(ps, 4)
        o._step = 1
        o.step()
    junk = [torch.full((1 << 16,), float("nan"), device="cuda") for _ in range(16)]
    _replay(graph, ob)
    _same(a, b)
    assert len(junk) == 16


def test_a_group_added_later():
    a, oa, graph, b, ob = _captured()
    more = [torch.nn.Parameter(torch.randn(50, 80, generator=gen(9)).cuda()) for _ in range(2)]
    oa.add_param_group({"params": [more[0]], "lr": 1e-2, "muon": True})
    more[0].grad = torch.randn(50, 80, generator=gen(10)).cuda()
    oa._step = ob._step = 1
    oa.step()
    ob.step()
    held = more[0].detach().clone()
    junk = [torch.full((1 << 16,), float("nan"), device="cuda") for _ in range(16)]
    for _ in range(2):
        _replay(graph, ob)               # (steps the groups it knew)
        _same(a, b)
        assert torch.equal(more[0], held)
    assert not torch.equal(held, more[1]) and len(junk) == 16


def test_without_a_muon_group():
    a, b = _params(), _params()
    oa, ob = (FusedMuon([{"params": ps, "lr": 1e-2}], max_grad_norm=1.0) for ps in (a, b))
    for ps, o in ((a, oa), (b, ob)):
        _grads(ps, 1)
        o.step()
    graph = torch.cuda.CUDAGraph()
    oa.begin_step()
    with torch.cuda.graph(graph):
        oa.launch()
    for _ in range(3):
        _replay(graph, ob)
        _same(a, b)


def test_momentum_that_was_changed():
    p = torch.nn.Parameter(torch.randn(40, 30, generator=gen(2)).cuda())
    opt = FusedMuon([{"params": [p], "lr": 1e-2, "muon": True, "momentum": 0.8}])
    m = torch.zeros(40, 30, dtype=torch.float64)
    for k, beta in enumerate((0.8, 0.95, 0.5)):
        opt.param_groups[0]["momentum"] = beta
        g = torch.randn(40, 30, generator=gen(k))
        p.grad = g.cuda()
        opt.step()
        m += (g.double() - m) * (1 - beta)
        # beta and 1 - beta in fp32, a difference, a product and a sum a step: 5 roundings of numbers up to |g| + |m| < 8
        assert (opt.state[p]["momentum_buffer"].cpu().double() - m).abs().max() <= (k + 1) * 5 * 8 * 2.0 ** -24
