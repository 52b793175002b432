"""The device tables that FusedMuon's launches read by address, on the host: a captured step goes on reading them, so they
are written in place where a pointer moves, and kept where they are replaced."""
import ctypes
import gc
import weakref

import pytest
import torch

from dphubert_amd import _lib, kernels, optim
from dphubert_amd.optim import FusedMuon

CAPTURING = [False]


class Plan:
    """A NewtonSchulzPlan's attributes without a device."""

    def __init__(self, mats, **_):
        self.mats, self.out = mats, [torch.zeros(m.shape, dtype=torch.bfloat16) for m in mats]

    def run(self):
        return self.out


@pytest.fixture(autouse=True)
def host(monkeypatch):
    CAPTURING[0] = False
    monkeypatch.setattr(kernels, "NewtonSchulzPlan", Plan)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: CAPTURING[0])
    monkeypatch.setattr(optim, "call", lambda *a: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda *a: 0)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **k: empty(*a, **k))
    monkeypatch.setattr(torch.cuda, "Event", lambda: type("E", (), {"record": lambda s: None, "synchronize": lambda s: None})())


def _p(*s):
    p = torch.nn.Parameter(torch.randn(*s))
    p.grad = torch.randn(*s)
    return p


def _update(opt, capture=False):
    """What launch() does before and around the kernels."""
    plist = opt._params()
    CAPTURING[0] = capture
    opt._ensure_chunks(plist)
    opt._slot_table(plist)
    opt._update(plist, {}, torch.zeros(1), (optim.DphAdamGroup * 4)(), False, 0)
    CAPTURING[0] = False


def _slots(opt):
    n = opt._m_slots.numel() // ctypes.sizeof(_lib.DphMuonSlot)
    return (_lib.DphMuonSlot * n).from_buffer_copy(opt._m_slots.numpy().tobytes())


def _muon(**kw):
    return FusedMuon([{"params": [_p(8, 4), _p(3, 5)], "muon": True}, {"params": [_p(7)]}], **kw)


@pytest.mark.parametrize("what", ["grad", "momentum", "parameter"])
def test_a_moved_pointer_is_written_into_the_same_tables(what):
    opt = _muon()
    _update(opt)
    _update(opt, capture=True)
    tables = [getattr(opt, n) for n in ("_m_slots", "_m_cslot", "_m_cstart", "_a_cslot", "_a_cstart", "_plan", "_slots_dev", "_cslot")]
    p = opt.param_groups[0]["params"][1]
    if what == "grad":
        p.grad = torch.randn(3, 5)
    elif what == "momentum":
        opt.state[p]["momentum_buffer"] = opt.state[p]["momentum_buffer"].clone()
    else:
        p.data = p.data.clone()
    _update(opt)
    assert all(getattr(opt, n) is t for n, t in zip(("_m_slots", "_m_cslot", "_m_cstart", "_a_cslot", "_a_cstart", "_plan",
                                                     "_slots_dev", "_cslot"), tables))
    s = _slots(opt)
    assert (s[1].param, s[1].grad, s[1].momentum) == (p.data_ptr(), p.grad.data_ptr(), opt.state[p]["momentum_buffer"].data_ptr())


def test_what_a_capture_read_outlives_a_longer_list():
    opt = _muon()
    _update(opt)
    _update(opt, capture=True)
    names = ("_m_slots", "_m_cslot", "_m_cstart", "_a_cslot", "_a_cstart", "_plan", "_slots_dev", "_cslot", "_cstart")
    old = [weakref.ref(getattr(opt, n)) for n in names]
    opt.add_param_group({"params": [_p(6, 6)], "muon": True})
    _update(opt)
    gc.collect()
    assert all(r() is not None for r in old)
    assert len(opt._plan.mats) == 3


def test_without_a_capture_nothing_is_kept():
    opt = _muon()
    _update(opt)
    old = weakref.ref(opt._plan)
    opt.add_param_group({"params": [_p(6, 6)], "muon": True})
    _update(opt)
    gc.collect()
    assert old() is None


def test_without_a_muon_group_it_is_captured_like_adamw():
    opt = FusedMuon([{"params": [_p(7), _p(3, 4)]}])
    _update(opt)
    _update(opt, capture=True)
    opt.param_groups[0]["params"][0].grad = torch.randn(7)
    _update(opt)
    _update(opt, capture=True)


def test_a_larger_parameter_beside_the_matrices_is_stepped_to_its_end():
    opt = _muon()
    _update(opt)
    assert opt._a_cslot.tolist() == [2] and opt._a_cstart.tolist() == [0]
    opt.param_groups[1]["params"][0] = _p(2 * optim.CHUNK + 5)
    _update(opt)
    assert opt._a_cslot.tolist() == [2, 2, 2] and opt._a_cstart.tolist() == [0, optim.CHUNK, 2 * optim.CHUNK]


def test_a_capture_that_would_need_other_tables_is_refused_and_leaves_them():
    opt = _muon()
    _update(opt)
    old = [getattr(opt, n) for n in ("_slots_dev", "_cslot", "_m_slots", "_plan")]
    opt.add_param_group({"params": [_p(6, 6)]})
    with pytest.raises(RuntimeError, match="capture"):
        _update(opt, capture=True)
    CAPTURING[0] = False
    assert all(getattr(opt, n) is t for n, t in zip(("_slots_dev", "_cslot", "_m_slots", "_plan"), old))
    _update(opt)
    assert opt._cslot.tolist() == [0, 1, 2, 3]
