"""8-bit products and Newton-Schulz on the tiles of large calls, 128 x 128 and 256 x 256 (test_tiles_cpu.py: that these
sizes take them), against 64 bits and against the same rows or matrices on 64 x 64 tiles.

Tolerances: those of test_int8_gpu.py, with |scale scale sum| for the sum of magnitudes (the integer sum is exact, so the
first rounding is its conversion), and those of test_newton_schulz_gpu.py.  The same numbers on other tiles are the same
bits: integer sums are exact and every float sum runs along k in one order."""
import math

import pytest
import torch

from dphubert_amd import kernels as K
from test_int8_gpu import acts, check, gen, rows64
from test_newton_schulz_gpu import check as ns_check, noise, strong

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# tile, M, N, K: rows, columns and K that end inside a tile, 16 bytes or a step of 128; one step (the schedule runs two), two, more
LINEAR = [(128, 4003, 1101, 100), (128, 4100, 1024, 129), (128, 3001, 1500, 16), (128, 7984, 1022, 257), (128, 2500, 1160, 1533),
          (256, 4001, 3907, 77), (256, 8100, 1901, 200), (256, 7900, 1920, 1000), (256, 4090, 3904, 128), (256, 3841, 4001, 1)]
EPILOGUES = [(act, res, odt) for act in (K.ACT_NONE, K.ACT_GELU) for res, odt in ((None, BF16), (None, F32), (BF16, BF16), (F32, F32))]
LN = [(128, 4003, 1101, 100, True), (128, 4100, 1024, 768, False), (256, 4001, 3907, 513, False), (256, 7900, 1920, 1024, True)]
# tile, (rows, columns, matrices)
LISTS = [(128, [(300, 421, 20), (419, 290, 20)]), (256, [(990, 1090, 12), (1091, 1001, 12)])]


def some_rows(M):
    """40 rows here and there, the first and the last among them (on 64 x 64 tiles, computed alone)."""
    return [slice(min(at, M - 40), min(at, M - 40) + 40) for at in range(0, M + 996, 997)]


@pytest.mark.parametrize("tile,M,N,C", LINEAR)
def test_linear(tile, M, N, C):
    g = gen(M + 3 * N + C)
    x = acts(M, C, F32 if M % 2 else BF16, g)
    w = K.quant_rows_i8((torch.randn(N, C, generator=g) / math.sqrt(C)).cuda())
    bias = torch.randn(N, generator=g).cuda()
    q, s = (t.cuda() for t in rows64(x))
    sums = torch.mm(q, w.q.double().t().contiguous()) * s.double()[:, None] * w.scale.double()
    for act, res, odt in EPILOGUES:
        r = torch.randn(M, N, generator=g).to(res).cuda() if res else None
        b = bias if act == K.ACT_GELU or res else None
        y = K.linear_i8(x, w, b, act=act, residual=r, out_dtype=odt)
        assert y.dtype == odt
        want = sums if b is None else sums + b.double()
        if act == K.ACT_GELU:
            want = want * 0.5 * torch.special.erfc(want * -math.sqrt(0.5))
        mag = sums.abs() + (0 if b is None else b.double().abs())
        if r is not None:
            want, mag = want + r.double(), mag + r.double().abs()
        tol = want.abs() * (torch.finfo(odt).eps / 2) + (9 * 2.0 ** -24 + 2e-7) * mag
        err = (y.double() - want).abs()
        assert y.isfinite().all() and (err <= tol).all(), (act, res, odt, (err / tol.clamp_min(1e-300)).max().item())
        for few in some_rows(M):
            again = K.linear_i8(x[few], w, b, act=act, residual=r[few] if r is not None else None, out_dtype=odt)
            assert torch.equal(again, y[few])


@pytest.mark.parametrize("tile", [128, 256])
def test_linear_what_lies_behind_a_row_and_past_the_end(tile):
    """The bytes behind K are other rows' integers, and out lies in a larger buffer that is left as it was."""
    M, N = (4003, 1101) if tile == 128 else (4001, 3907)
    g = gen(tile)
    mem = torch.randint(-127, 128, (M + N, 160), generator=g, dtype=torch.int8).cuda()
    s = (torch.rand(M + N, generator=g) + 0.5).cuda()
    for C in (77, 129, 144):
        x, w = K.I8Rows(mem[:M, :C], s[:M]), K.I8Rows(mem[M:, :C], s[M:])
        room = torch.full((M + 2, N + 9), 7.0, dtype=F32, device="cuda")
        y = K.linear_i8(x, w, out=room[1:M + 1, 4:N + 4], out_dtype=F32)
        want = torch.mm(x.q.double(), w.q.double().t().contiguous()) * s[:M, None].double() * s[M:].double()
        assert ((y.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()
        y.fill_(7.0)
        assert (room == 7.0).all()


@pytest.mark.parametrize("tile,M,N,C,keep", LN)
@pytest.mark.parametrize("act", [K.ACT_NONE, K.ACT_GELU])
def test_layernorm_linear(tile, M, N, C, keep, act):
    g = gen(M + N + C)
    x = acts(M, C, F32 if C % 2 else BF16, g)
    lw, lb = (1 + 0.2 * torch.randn(C, generator=g)).cuda(), (0.1 * torch.randn(C, generator=g)).cuda()
    w = K.quant_rows_i8((torch.randn(N, C, generator=g) / math.sqrt(C)).cuda())
    b = torch.randn(N, generator=g).cuda()
    y, n = K.layernorm_linear_i8(x, lw, lb, w, b, act=act, keep_norm=keep)
    assert (n is not None) == keep and y.isfinite().all()
    # 40 rows at a time: those calls are compared with 64 bits in test_int8_gpu.py
    for few in some_rows(M):
        ya, na = K.layernorm_linear_i8(x[few], lw, lb, w, b, act=act, keep_norm=keep)
        assert torch.equal(ya, y[few]) and (na is None or torch.equal(na, n[few]))


def exact(t, steps):
    x = t.double()
    x = x.t().contiguous() if t.shape[0] > t.shape[1] else x
    a, b, c = K.NS_COEFFS
    x = x / (x.square().sum().sqrt() + 1e-7)
    for _ in range(steps):
        gram = torch.mm(x, x.t().contiguous())
        x = a * x + torch.mm(b * gram + c * torch.mm(gram, gram), x)
    return (x.t() if t.shape[0] > t.shape[1] else x).cpu()


@pytest.mark.parametrize("tile,shapes", LISTS)
@pytest.mark.parametrize("steps", [5, 3])
def test_newton_schulz(tile, shapes, steps):
    g = gen(tile + steps)
    mats = []
    for i, (m, n, count) in enumerate(shapes):
        mats += [(strong if k % 3 == 2 else noise)(m, n, g, BF16 if i else F32) for k in range(count)]
    got = K.newton_schulz(mats, steps=steps)
    for x, y in zip(mats, got):
        ns_check(y, exact(x, steps))
    # the result of a matrix does not depend on its list: alone it takes 64 x 64 tiles
    for k in (0, 2, shapes[0][2] - 1, shapes[0][2], len(mats) - 1):
        assert torch.equal(got[k], K.newton_schulz([mats[k]], steps=steps)[0]), k
    # nor on its place
    back = K.newton_schulz(mats[::-1], steps=steps)
    assert all(torch.equal(a, b) for a, b in zip(got, back[::-1]))
