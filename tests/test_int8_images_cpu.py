"""The cached 8-bit weights (ops.i8_image) that a captured forward reads by address, on the host."""
import ctypes
import gc
import weakref

import pytest
import torch

from dphubert_amd import kernels as K
from dphubert_amd import ops

CAPTURING = [False]


def quant(x):
    s = x.abs().amax(1) / 127
    return K.I8Rows(torch.round(x / s[:, None]).to(torch.int8), s)


@pytest.fixture(autouse=True)
def host(monkeypatch):
    CAPTURING[0] = False
    monkeypatch.setattr(K, "quant_rows_i8", quant)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: CAPTURING[0])


def _weights():
    return [torch.nn.Parameter(torch.randn(4, 16)) for _ in range(3)]


def _read_by_a_graph(*ts):
    rows = ops.i8_image(*ts)
    CAPTURING[0] = True
    assert ops.i8_image(*ts) is rows
    CAPTURING[0] = False
    return rows


@pytest.mark.parametrize("how", ["in place", "again", "storage", "another source"])
def test_captured_integers_are_written_in_place(how):
    ts = _weights()
    old = _read_by_a_graph(*ts)
    at = (old.q.data_ptr(), old.scale.data_ptr())
    with torch.no_grad():
        if how == "in place":
            ts[1].mul_(3)
        elif how == "storage":
            ts[2].data = ts[2].data * 3
        elif how == "another source":
            ts[2] = torch.nn.Parameter(torch.randn(4, 16))
        else:
            ts[0].data.mul_(3)
            ts[0]._dph_i8.key = tuple((t.device, t.data_ptr(), t._version) for t in ts)     # (changed unseen)
    new = ops.i8_image(*ts, again=how == "again")
    want = quant(torch.cat([t.detach() for t in ts]))
    assert (new.q.data_ptr(), new.scale.data_ptr()) == at
    assert torch.equal(new.q, want.q) and torch.equal(new.scale, want.scale)
    assert new is not old and ops.i8_image(*ts) is new


def test_captured_integers_outlive_another_shape():
    ts = _weights()
    _read_by_a_graph(*ts)
    old = [weakref.ref(t) for t in ops.i8_image(*ts)]
    for n in (6, 5):
        ts[0].data = torch.randn(n, 16)
        new = ops.i8_image(*ts)
        assert new.q.shape == (n + 8, 16)
        del new
        gc.collect()
        assert all(r() is not None for r in old)


def test_integers_that_no_graph_reads_are_left_to_their_holder():
    ts = _weights()
    old = ops.i8_image(*ts)
    q = old.q.clone()
    with torch.no_grad():
        ts[0].mul_(-1)
    new = ops.i8_image(*ts)
    assert torch.equal(old.q, q) and torch.equal(new.q[:4], -q[:4])
    again = ops.i8_image(*ts, again=True)
    assert again is not new and torch.equal(again.q, new.q)


def test_a_capture_does_not_lay_out():
    ts = _weights()
    ops.i8_image(*ts)
    with torch.no_grad():
        ts[0].mul_(2)
    CAPTURING[0] = True
    with pytest.raises(RuntimeError, match="capture"):
        ops.i8_image(*ts)


def test_laid_out_in_inference_mode_and_written_outside_it():
    ts = _weights()
    with torch.inference_mode():
        old = _read_by_a_graph(*ts)
    new = ops.i8_image(*ts, again=True)
    assert new.q is old.q
    with torch.inference_mode():
        assert ops.i8_image(*ts, again=True).q is old.q


def test_the_biases_that_a_captured_forward_reads(monkeypatch):
    """Their concatenation is cached beside the integers."""
    monkeypatch.setattr(ops, "_table", lambda rows: rows)
    monkeypatch.setattr(ops, "ptr", lambda t: t)
    monkeypatch.setattr(ops, "_s", lambda: 0)
    copy = lambda name, rows, n, most, s: [ctypes.memmove(to, at, 4 * k) for at, to, k in rows]  # noqa: E731
    monkeypatch.setattr(ops, "call", copy)
    ts = [torch.nn.Parameter(torch.randn(4), requires_grad=False) for _ in range(3)]
    free, want = ops.f32_cat(*ts), torch.cat(ts)
    assert torch.equal(free, want) and ops.f32_cat(*ts) is free
    ts[1].mul_(2)
    old = ops.f32_cat(*ts)
    assert old is not free and torch.equal(free, want)        # (no graph reads it: left to its holder)
    CAPTURING[0] = True
    assert ops.f32_cat(*ts) is old
    CAPTURING[0] = False
    ts[2].mul_(3)
    assert ops.f32_cat(*ts) is old and torch.equal(old, torch.cat(ts))
    ts[0].data.mul_(5)                                        # (unseen)
    assert not torch.equal(ops.f32_cat(*ts), torch.cat(ts))
    assert ops.f32_cat(*ts, again=True) is old and torch.equal(old, torch.cat(ts))
    at = weakref.ref(old)
    del old
    for n in (6, 5):
        ts[0].data = torch.randn(n)
        ts[1].mul_(2)
        assert ops.f32_cat(*ts).numel() == n + 8
        gc.collect()
        assert at() is not None
