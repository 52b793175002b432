"""8-bit integer products (kernels.quant_rows_i8 / linear_i8 / layernorm_linear_i8) against the definition in 64 bits.

Tolerances: the integers and scales are exact by definition (the quotient's rounding is decided exactly), the integer
sums are exact; what follows is fp32 (a handful of roundings of 2^-24 each) and one rounding to the output type, at most
half a step: finfo.eps / 2 of the value (2^-8 in bf16)."""
import math

import pytest
import torch

from dphubert_amd import kernels as K

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
TINY = 2.0 ** -126


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def rows64(x):
    """(q, scale) of the definition: x any float type, computed in 64 bits on the CPU."""
    x = x.detach().cpu()
    amax = x.float().abs().amax(1)
    scale = torch.clamp(amax * (torch.ones(()) / 127.0), min=TINY)     # (fp32: 1 / 127 rounded, then the product)
    bad = ~torch.isfinite(x.float()).all(1)
    q = torch.round(x.double() / scale.double()[:, None])
    q[bad] = 0
    scale[bad] = math.nan
    return q, scale


def linear64(q, qs, w, bias, act, residual):
    y = q.double() @ w.q.cpu().double().t() * qs.double()[:, None] * w.scale.cpu().double()
    if bias is not None:
        y = y + bias.cpu().double()
    if act == K.ACT_GELU:
        y = y * torch.special.ndtr(y)
    return y if residual is None else y + residual.cpu().double()


def check(got, want, mag):
    t = got.dtype
    half = torch.finfo(t).eps / 2
    # fp32: int -> float, two scales, bias, residual: 5 roundings; GELU: its erf approximation, 1.5e-7 of |x|, + 4
    tol = half * want.abs() + (9 * 2.0 ** -24 + 2e-7) * mag
    err = (got.cpu().double() - want).abs()
    assert got.isfinite().all()
    assert (err <= tol).all(), (err / tol.clamp_min(1e-300)).max().item()


def acts(M, K_, dt, g):
    c = torch.exp(0.5 * torch.randn(K_, generator=g))
    return (torch.randn(M, K_, generator=g) * c).to(dt).cuda()


# ---- the integers ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 16), (3, 15), (5, 17), (7, 127), (64, 512), (33, 768), (9, 1533), (4, 4096), (2, 5003)])
def test_quant_rows(R, C, dt):
    g = gen(R * 10007 + C)
    x = acts(R, C, dt, g)
    r = K.quant_rows_i8(x)
    q, s = rows64(x)
    assert r.q.shape == (R, C) and r.q.stride(0) % 16 == 0
    assert torch.equal(r.scale.cpu(), s)
    assert torch.equal(r.q.cpu().double(), q)
    # the bytes between the row's end and the next row are zeros
    whole = r.q.as_strided((R, r.q.stride(0)), (r.q.stride(0), 1)) if R > 1 else r.q
    assert not whole[:, C:].any()


def test_quant_rows_ties_and_borders():
    # 127 makes the scale 1: exact ties go to even, their fp32 neighbours to the nearest
    v = torch.arange(-126.5, 127, 1.0)
    up, dn = torch.nextafter(v, torch.tensor(1e9)), torch.nextafter(v, torch.tensor(-1e9))
    x = torch.stack([torch.cat([torch.tensor([127.0]), t]) for t in (v, up, dn)])
    # the same times numbers that are no powers of two, and a scale at the end of the range
    x = torch.cat([x, x * 0.3, x * 1e-3 / 7, x * 2.0 ** -126, x * 2.0 ** 120]).cuda()
    r = K.quant_rows_i8(x)
    q, s = rows64(x)
    assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), q)
    assert r.q[0, 1:5].tolist() == [-126, -126, -124, -124]


def test_quant_rows_special_rows():
    x = torch.randn(8, 100, generator=gen(1))
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 99] = -math.inf
    x[3, 64] = math.nan
    x[4] = 1e-42
    x[5] = 3.4e38
    x[6] = -0.0
    for dt in (F32, BF16):
        xd = x.to(dt).cuda()
        r = K.quant_rows_i8(xd)
        q, s = rows64(xd)
        assert torch.equal(r.scale.isnan().cpu(), s.isnan()) and r.scale.isnan().tolist() == \
            [False, True, True, True, False, (dt == BF16 and xd[5].isinf().any().item()), False, False]
        ok = ~s.isnan()
        assert torch.equal(r.scale.cpu()[ok], s[ok]) and torch.equal(r.q.cpu().double(), q)
        assert r.scale[0].item() == TINY and not r.q[0].any()


def test_quant_rows_strided_and_empty():
    g = gen(3)
    big = acts(11, 300, BF16, g)
    for v in (big[:, 1:77], big[::2, :64], big[3:4, 5:30], big[:, :1]):
        r = K.quant_rows_i8(v)
        q, s = rows64(v)
        assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), q)
    e = K.quant_rows_i8(big[:0])
    assert e.q.shape == (0, 300) and e.scale.shape == (0,)


# ---- the product -------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 1024), (2, 16, 129), (3, 7, 5), (4, 257, 768), (5, 130, 127), (8, 96, 2048), (16, 384, 512),
         (17, 65, 33), (31, 128, 128), (63, 200, 4100), (64, 768, 768), (100, 100, 100), (127, 129, 256), (128, 128, 1000),
         (129, 768, 1533), (255, 257, 64), (300, 384, 640), (499, 770, 200), (1030, 260, 96)]


@pytest.mark.parametrize("M,N,C", SIZES)
@pytest.mark.parametrize("dt", [BF16, F32])
def test_linear(M, N, C, dt):
    g = gen(M * 31 + N * 7 + C)
    x = acts(M, C, dt, g)
    w = K.quant_rows_i8((torch.randn(N, C, generator=g) / math.sqrt(C)).cuda())
    bias = torch.randn(N, generator=g).cuda()
    q, s = rows64(x)
    for act, res, odt in ((K.ACT_NONE, None, BF16), (K.ACT_GELU, None, F32), (K.ACT_GELU, BF16, None), (K.ACT_NONE, F32, None)):
        r = torch.randn(M, N, generator=g).to(res).cuda() if res else None
        b = bias if act == K.ACT_GELU or res else None
        y = K.linear_i8(x, w, b, act=act, residual=r, out_dtype=odt or BF16)
        assert y.dtype == (res or odt) and y.shape == (M, N)
        want = linear64(q, s, w, b, act, r)
        mag = linear64(q.abs(), s, K.I8Rows(w.q.cpu().abs(), w.scale), b.abs() if b is not None else None, K.ACT_NONE,
                       r.abs() if r is not None else None)
        check(y, want, mag)


def test_linear_of_given_integers_ignores_what_lies_behind_a_row():
    g = gen(5)
    M, N, C = 70, 50, 77
    mem = torch.randint(-127, 128, (M + N, 96), generator=g, dtype=torch.int8).cuda()
    s = torch.rand(M + N, generator=g).cuda()
    x, w = K.I8Rows(mem[:M, :C], s[:M]), K.I8Rows(mem[M:, :C], s[M:])
    y = K.linear_i8(x, w, out_dtype=F32)
    want = linear64(x.q.cpu().double(), s[:M].cpu(), w, None, K.ACT_NONE, None)
    check(y, want, want.abs() + 1)
    # all at the ends of the range: the sums do not wrap
    q = torch.full((3, 131072), 127, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    assert (K.linear_i8(K.I8Rows(q, one), K.I8Rows(-q, one), out_dtype=F32) == -127.0 * 127 * 131072).all()


def test_linear_strides_out_and_in_place():
    g = gen(6)
    M, N, C = 150, 90, 200
    big = acts(M, 3 * C, BF16, g)
    x = big[:, C + 3:2 * C + 3]
    w = K.quant_rows_i8((torch.randn(N, C, generator=g) / 14).cuda())
    q, s = rows64(x)
    room = torch.full((M, 2 * N + 1), 7.0, dtype=F32, device="cuda")
    out = room[:, 5:5 + N]
    out.copy_(torch.randn(M, N, generator=g))
    want = linear64(q, s, w, None, K.ACT_NONE, out)
    y = K.linear_i8(x, w, residual=out, out=out)
    assert y is out
    check(y, want, want.abs() + 3)
    assert (room[:, :5] == 7).all() and (room[:, 5 + N:] == 7).all()


@pytest.mark.parametrize("M", [4, 16, 40])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_linear_out_over_x(M, dt):
    """The residual stream in place: x, the residual and out are one tensor."""
    g = gen(16)
    x = acts(M, 640, dt, g)
    w = K.quant_rows_i8((torch.randn(640, 640, generator=g) / 25).cuda())
    q, s = rows64(x)
    want = linear64(q, s, w, None, K.ACT_NONE, x)
    alone = K.linear_i8(x, w, residual=x)
    assert K.linear_i8(x, w, residual=x, out=x) is x
    assert torch.equal(x, alone)
    check(x, want, want.abs() + 4)
    # out over x's columns of one buffer, and between them
    buf = acts(M, 200, dt, g)
    w = K.quant_rows_i8(torch.randn(50, 100, generator=g).cuda())
    want = K.linear_i8(buf[:, :100].clone(), w, out_dtype=dt)
    keep = buf.clone()
    for c in (150, 50, 0):
        K.linear_i8(buf[:, :100], w, out=buf[:, c:c + 50], out_dtype=dt)
        assert torch.equal(buf[:, c:c + 50], want)
        buf.copy_(keep)
    # beside the residual in one buffer; across it is refused
    want = K.linear_i8(buf[:, :100], w, residual=buf[:, 100:150])
    K.linear_i8(buf[:, :100], w, residual=buf[:, 100:150], out=buf[:, 150:])
    assert torch.equal(buf[:, 150:], want) and torch.equal(buf[:, :150], keep[:, :150])
    for bad in (buf[:, 101:151], buf[:, 51:101], buf.view(-1)[100:100 + 50 * M].view(M, 50)):
        with pytest.raises(ValueError, match="overlaps"):
            K.linear_i8(buf[:, :100], w, residual=buf[:, 100:150], out=bad)
    with pytest.raises(ValueError, match="overlaps"):
        K.linear_i8(buf[:1, :100], w, out=w.scale.view(1, 50), out_dtype=F32)


def test_linear_one_row_in_place():
    g = gen(17)
    x = acts(1, 64, BF16, g)
    w = K.quant_rows_i8(torch.randn(64, 64, generator=g).cuda())
    want = K.linear_i8(x, w, residual=x)
    # (a row's distance to the next one means nothing where there is none)
    for row in (x.clone(), x.clone().as_strided((1, 64), (7, 1)), x.clone().as_strided((1, 64), (0, 1))):
        same = row.as_strided((1, 64), (64, 1))
        assert K.linear_i8(row, w, residual=same, out=row) is row and torch.equal(row, want)
    buf = torch.zeros(1, 96, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        K.linear_i8(x, w, residual=buf[:, :64], out=buf[:, 32:])


def test_gelu_of_sums_past_the_range():
    """Finite operands whose sum is infinite in fp32: GELU(inf) = inf, and GELU(-inf) has the limit 0."""
    for M in (3, 40):
        x = torch.full((M, 4096), 3e38, device="cuda")
        w = K.quant_rows_i8(torch.stack([torch.ones(4096), -torch.ones(4096), torch.zeros(4096)]).cuda())
        y = K.linear_i8(x, w, act=K.ACT_GELU, out_dtype=F32)
        assert (y[:, 0] == math.inf).all() and not y[:, 1:].any()
        x[1, 7] = math.nan
        assert K.linear_i8(x, w, act=K.ACT_GELU).isnan().all(1).tolist() == [r == 1 for r in range(M)]


def test_linear_rows_do_not_touch_each_other():
    g = gen(7)
    x = acts(40, 256, F32, g)
    w = K.quant_rows_i8((torch.randn(96, 256, generator=g) / 16).cuda())
    y = K.linear_i8(x, w)
    bad = x.clone()
    bad[3, 9], bad[17, 0], bad[30, 255] = math.nan, math.inf, -math.inf
    z = K.linear_i8(bad, w)
    rows = torch.ones(40, dtype=torch.bool)
    rows[[3, 17, 30]] = False
    assert z[~rows].isnan().all() and torch.equal(z[rows], y[rows])
    # a row of zeros gives the bias
    bad[5] = 0
    b = torch.randn(96, generator=g).cuda()
    assert torch.equal(K.linear_i8(bad, w, b, out_dtype=F32)[5], b)


def test_linear_empty():
    w = K.quant_rows_i8(torch.randn(10, 32).cuda())
    assert K.linear_i8(torch.empty(0, 32, device="cuda"), w).shape == (0, 10)
    none = K.I8Rows(w.q[:0], w.scale[:0])
    assert K.linear_i8(torch.randn(4, 32, device="cuda"), none).shape == (4, 0)


# ---- LayerNorm + product -------------------------------------------------------------------------------------------
def norm64(x, w, b, eps):
    x = x.cpu().double()
    m = x.mean(1, keepdim=True)
    return (x - m) / torch.sqrt((x - m).square().mean(1, keepdim=True) + eps) * w.cpu().double() + b.cpu().double()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("M,N,C", [(1, 64, 64), (2, 33, 17), (4, 768, 768), (49, 130, 768), (65, 257, 513), (130, 64, 1024), (20, 96, 1280),
                                   (9, 40, 2048), (600, 384, 100)])
def test_layernorm_linear(M, N, C, dt):
    g = gen(M + N + C)
    x = (acts(M, C, F32, g) + 0.5).to(dt)
    lw, lb = (1 + 0.2 * torch.randn(C, generator=g)).cuda(), (0.1 * torch.randn(C, generator=g)).cuda()
    w = K.quant_rows_i8((torch.randn(N, C, generator=g) / math.sqrt(C)).cuda())
    b = torch.randn(N, generator=g).cuda()
    n = norm64(x, lw, lb, 1e-5)
    for act, keep in ((K.ACT_NONE, True), (K.ACT_GELU, False)):
        y, norm = K.layernorm_linear_i8(x, lw, lb, w, b, act=act, keep_norm=keep)
        assert (norm is not None) == keep
        # fp32 statistics: about 2 + log2(64) + C / 64 roundings of a sum of C terms, on |x - mean| rstd |w| + |b|
        err = (24 + C / 64) * 2.0 ** -24 * (n.abs() + x.cpu().double().abs().amax() + 1)
        if keep:
            d = (norm.cpu().double() - n).abs()
            assert (d <= n.abs() * torch.finfo(BF16).eps / 2 + err).all()
        # a value within err of a rounding border may go either way: each such flip moves a sum by one step s |w|
        amax = n.abs().amax(1)
        s = amax / 127
        q = torch.round(n / s[:, None])
        near = ((n / s[:, None] - torch.floor(n / s[:, None]) - 0.5).abs() <= (err + amax[:, None] * 2.0 ** -22) / s[:, None])
        wa = w.q.cpu().double().abs() * w.scale.cpu().double()[:, None]
        slack = (near.double() @ wa.t()) * s[:, None]
        want = linear64(q, s, w, b, act, None)
        mag = linear64(q.abs(), s, K.I8Rows(w.q.cpu().abs(), w.scale), b.abs(), K.ACT_NONE, None)
        # (the scale itself carries the statistics' error)
        tol = want.abs() * torch.finfo(BF16).eps / 2 + mag * (2e-7 + (40 + C / 64) * 2.0 ** -24) + 1.13 * slack
        assert ((y.cpu().double() - want).abs() <= tol).all()


def test_layernorm_linear_odd_rows():
    g = gen(9)
    C = 320
    x = acts(6, C, F32, g)
    x[1] = 4.25           # a constant row: the LayerNorm is its bias
    x[2, 7] = math.nan
    x[3] = 1e4 + torch.randn(C, generator=g).cuda()
    lw, lb = torch.ones(C, device="cuda"), torch.randn(C, generator=g).cuda()
    w = K.quant_rows_i8(torch.eye(C).cuda())
    y, n = K.layernorm_linear_i8(x, lw, lb, w, keep_norm=True)
    assert n[2].isnan().all() and y[2].isnan().all()
    assert torch.equal(n[1], lb.bfloat16())
    rest = [0, 1, 3, 4, 5]
    assert y[rest].isfinite().all()
    want = norm64(x, lw, lb, 1e-5)[rest]
    # one step of the integers, half a step of bf16; row 3: 1e4 costs 14 bits of the difference
    tol = want.abs().amax(1, keepdim=True) / 127 * 0.51 + want.abs() * 2.0 ** -8 + 1e4 * 2.0 ** -22
    assert ((y[rest].cpu().double() - want).abs() <= tol).all()


# ---- streams, graphs, both together ---------------------------------------------------------------------------------
def test_graph_replays_and_streams():
    g = gen(11)
    x = acts(200, 256, BF16, g)
    w1 = K.quant_rows_i8((torch.randn(512, 256, generator=g) / 16).cuda())
    w2 = K.quant_rows_i8((torch.randn(256, 512, generator=g) / 22).cuda())
    lw, lb = torch.ones(256, device="cuda"), torch.zeros(256, device="cuda")

    def block(h):
        u, n = K.layernorm_linear_i8(h, lw, lb, w1, act=K.ACT_GELU, keep_norm=True)
        return K.linear_i8(u, w2, residual=n)

    want = block(x).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block(x)
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    held = x.clone()
    with torch.cuda.graph(graph):
        got = block(held)
    for k in range(3):
        held.copy_(x if k != 1 else x.flip(0))
        graph.replay()
        eager = block(held)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
    assert torch.equal(got, want)
