"""Refusals of the 8-bit products and of the orthogonalisation: decided on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from dphubert_amd import _lib
from dphubert_amd import kernels as K


@pytest.mark.parametrize("call", [
    lambda: K.quant_rows_i8(torch.randn(4, 8)),
    lambda: K.quant_rows_i8([1, 2]),
    lambda: K.linear_i8(torch.randn(4, 8), K.I8Rows(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2))),
    lambda: K.linear_i8(None, None),
    lambda: K.layernorm_linear_i8(torch.randn(4, 8), torch.ones(8), torch.zeros(8), None),
    lambda: K.newton_schulz([torch.randn(4, 8)]),
    lambda: K.newton_schulz([None]),
    lambda: K.newton_schulz([torch.randn(4, 8)], steps=0),
    lambda: K.newton_schulz([torch.randn(4, 8)], coeffs=(1, 2)),
])
def test_no_cpu_path(call):
    with pytest.raises(ValueError):
        call()


def test_nothing_to_do():
    assert K.newton_schulz([]) == []


def _args(**kw):
    a = _lib.DphLinearI8Args()
    d = dict(M=4, N=4, K=32, q=4096, ldq=32, q_scale=4096, w=4096, ldw=32, w_scale=4096, out=4096, ldo=4, out_dtype=K.OUT_BF16)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(K=0), dict(N=-2), dict(K=131073, ldq=131088, ldw=131088), dict(M=1 << 40), dict(q=None), dict(ldq=31), dict(ldq=40),
    dict(q=4100), dict(ldq=16), dict(act=7), dict(out_dtype=2), dict(w=None), dict(w=4104), dict(ldw=8), dict(ldw=36), dict(out=None),
    dict(ldo=3), dict(residual=4096, ldr=3), dict(w_scale=None), dict(q_scale=None), dict(residual=4096, residual_f32=1), dict(x=4096, ldx=31),
    dict(x=4096, ldx=32, ln_weight=4096), dict(x=4096, ldx=4096, ln_weight=4096, ln_bias=4096, K=2049, ldq=2064, ldw=2064),
    dict(M=17, x=4096, ldx=32, ln_weight=4096, ln_bias=4096, ldq=1024), dict(M=17, x=4096, ldx=32, q=None),
    dict(x=4096, ldx=32, ln_weight=4096, ln_bias=4096, norm_out=4096, ld_norm=31), dict(x=4096, ldx=32, w=None),
    dict(x=4096, ldx=32, ln_weight=4096, ln_bias=4096, out_dtype=K.OUT_F32),
    dict(x=4096, ldx=32, ln_weight=4096, ln_bias=4096, residual=4096, ldr=4),
])
def test_c_entry_refuses(kw):
    """The C entry's own checks (nothing is launched: there is no device here)."""
    assert _lib.lib().dph_linear_i8(C.byref(_args(**kw)), None) == -1
    assert _lib.lib().dph_last_error()


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(K=0), dict(x=None), dict(q=None), dict(q=4097), dict(ldq=24), dict(ldq=16), dict(ldx=31),
                                dict(scale=None), dict(rows=1 << 26)])
def test_c_quant_refuses(kw):
    d = dict(x=4096, f32=0, rows=4, K=32, ldx=32, q=4096, ldq=32, scale=4096)
    d.update(kw)
    assert _lib.lib().dph_quant_rows_i8(d["x"], d["f32"], d["rows"], d["K"], d["ldx"], d["q"], d["ldq"], d["scale"], None) == -1


@pytest.mark.parametrize("x,out,small", [(4096, 1 << 16, True), (4096, 4096, False), (4096, 4096 + 254, False),
                                         (4096, 4096 + 256, True), (4096 + 30, 4096, False), (4096 + 32, 4096, True)])
def test_c_entry_needs_q_where_out_lies_over_x(x, out, small):
    """Up to 16 rows need no q (a null w is then what is refused), unless bytes of out are bytes of x: 4 rows of 32 bf16
    columns are 256 bytes, 4 of 4 are 32."""
    assert _lib.lib().dph_linear_i8(C.byref(_args(x=x, ldx=32, out=out, q=None, q_scale=None, ldw=8)), None) == -1
    assert (b"rows of w" in _lib.lib().dph_last_error()) == small
    assert (b"null operand" in _lib.lib().dph_last_error()) == (not small)


def test_workspace():
    """Nothing for up to 16 rows that fit the LDS, else the integers (rows of whole 16 bytes) and the scales."""
    ws = _lib.lib().dph_linear_i8_workspace
    assert ws(1, 8, 1024) == ws(16, 1, 64) == ws(0, 8, 8) == ws(16, 5, 3500) == 0
    assert ws(17, 8, 33) == 17 * (48 + 4) and ws(16, 8, 4096) == 16 * (4096 + 4)


def test_c_empty_calls():
    assert _lib.lib().dph_quant_rows_i8(None, 0, 0, 32, 32, None, 32, None, None) == 0
    assert _lib.lib().dph_linear_i8(C.byref(_args(M=0)), None) == 0
    assert _lib.lib().dph_linear_i8(None, None) == -1
    assert _lib.lib().dph_newton_schulz(None, None, 0, 5, None, 0.0, None, 0, None) == 0


def _ns(rows=8, cols=8, count=1, out=4096, p=4096, rs=8, cs=1, steps=5, ws=4096, nbytes=None, c=True):
    g = (_lib.DphNsGroup * 1)()
    g[0].rows, g[0].cols, g[0].count, g[0].out = rows, cols, count, out
    m = (_lib.DphNsMat * 1)()
    m[0].p, m[0].row_stride, m[0].col_stride = p, rs, cs
    need = _lib.lib().dph_newton_schulz_workspace(g, 1)
    co = (C.c_float * 3)(*K.NS_COEFFS) if c else None
    return _lib.lib().dph_newton_schulz(m, g, 1, steps, co, 1e-7, ws, need if nbytes is None else nbytes, None)


@pytest.mark.parametrize("kw", [dict(rows=0), dict(cols=0), dict(count=0), dict(rows=1 << 21), dict(out=None), dict(out=4100), dict(p=None), dict(rs=7),
                                dict(cs=2), dict(rs=1, cs=7), dict(steps=0), dict(steps=65), dict(ws=None), dict(ws=4100), dict(nbytes=100), dict(c=False)])
def test_c_newton_schulz_refuses(kw):
    assert _ns(**kw) == -1
    assert _lib.lib().dph_last_error()


def test_workspace_is_refused_for_bad_groups():
    g = (_lib.DphNsGroup * 1)()
    assert _lib.lib().dph_newton_schulz_workspace(g, 1) == -1
    assert _lib.lib().dph_newton_schulz_workspace(None, 1) == -1
    g[0].rows, g[0].cols, g[0].count = 70, 64, 2
    # partial sums, Y twice (128 x 64), E and F of 64 x 64, the lower halves of all (up to 128 rows); above, 8 bits more of Y
    assert _lib.lib().dph_newton_schulz_workspace(g, 1) == 2 * (64 * 8 + 4 * 64 * 128 * 2 + 4 * 64 * 64 * 2)
    g[0].rows, g[0].cols = 129, 200
    assert _lib.lib().dph_newton_schulz_workspace(g, 1) == 2 * (64 * 8 + 2 * 192 * 256 * 2 + 192 * 256 + 2 * 192 * 192 * 2)
