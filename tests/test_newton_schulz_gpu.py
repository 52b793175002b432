"""kernels.newton_schulz against the iteration in 64 bits.

Tolerance: the result's rounding to bf16 is at most 2^-8 of an element and 2^-8 / sqrt(3) = 2.3e-3 in the 2-norm.  The
fp16 operands add, per step, the rounding of X (2^-11 / sqrt(3) = 2.8e-4), of E (2.8e-4 of it, times |b + 2 c d + 2 c E|,
at most 4.8 while E is of a few singular values' squares, 0.7 in the last two steps) and of F (2.8e-4): in the last two
steps about 2.8e-4 (1 + 0.7 + 1) each, 5e-4 together, and from the steps before at most what a singular value grows by
in the steps that follow (below 1.5 from the fourth step on) times 4.8 * 2.8e-4 = 1.4e-3: 2e-3.  Root of the squares'
sum with the output's rounding: 3.1e-3, taken as 4e-3.  Strong directions over weak ones amplify the first steps'
roundings of the operands (not of X, which has 22 bits there): another 1.5e-3 for a ratio of 100, in the 4e-3 as well.
An element is off by its own rounding and by 8 standard deviations of the rest (2.5e-3 of the root mean square)."""
import math

import pytest
import torch

from dphubert_amd import kernels as K

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
TOL = 4e-3


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def exact(t, steps=5, coeffs=K.NS_COEFFS, eps=1e-7):
    x = t.detach().cpu().double()
    if x.shape[0] > x.shape[1]:
        return exact(t.t(), steps, coeffs, eps).t()
    a, b, c = coeffs
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def check(got, want, tol=TOL):
    assert got.dtype == BF16 and got.shape == want.shape and got.isfinite().all()
    d = got.cpu().double() - want
    rms = want.square().mean().sqrt()
    assert d.norm() <= tol * want.norm(), (d.norm() / want.norm()).item()
    assert (d.abs() <= want.abs() * 2.0 ** -8 + 8 * 2.5e-3 * rms).all()


def noise(m, n, g, dt=F32, scale=1e-3):
    return (torch.randn(m, n, generator=g) * scale).to(dt).cuda()


def strong(m, n, g, dt=F32):
    r = max(1, min(m, n) // 8)
    u, v = torch.randn(m, r, generator=g), torch.randn(r, n, generator=g)
    return ((u @ v + 0.1 * torch.randn(m, n, generator=g)) * 1e-5).to(dt).cuda()


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (5, 3), (16, 64), (64, 16), (63, 65), (64, 64), (100, 100), (128, 128), (129, 127), (129, 400),
          (257, 255), (384, 1000), (1000, 129), (512, 512), (300, 2047),
          (3, 1024), (1500, 64), (130, 1100), (100, 5000), (256, 9000), (20000, 5)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("m,n", SHAPES)
def test_sizes(m, n, dt):
    g = gen(m * 4099 + n)
    a, b = noise(m, n, g, dt), strong(m, n, g, dt)
    got = K.newton_schulz([a, b])
    for x, y in zip((a, b), got):
        assert y.is_contiguous()
        check(y, exact(x))


def test_singular_values():
    """Near one -- but five steps multiply a small singular value by 3.4445^5 = 485 at the most, so one below 1 / 485 of the
    norm stays small (the weak directions of the second matrix, 0.002 of its norm, come to 0.13): the bound is the exact
    factor's value, from which none can be further than the difference's Frobenius norm (Weyl)."""
    g = gen(2)
    mats = [noise(200, 300, g), strong(300, 200, g)]
    for x, t in zip(mats, K.newton_schulz(mats)):
        s, e = torch.linalg.svdvals(t.cpu().double()), torch.linalg.svdvals(exact(x))
        assert s.max() < 1.3 and (s - e).abs().max() <= TOL * exact(x).norm()
    assert torch.linalg.svdvals(K.newton_schulz(mats[:1])[0].float()).min() > 0.6


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 9])
def test_steps(steps):
    g = gen(steps)
    t = [noise(150, 260, g), strong(260, 150, g)]
    for x, y in zip(t, K.newton_schulz(t, steps=steps)):
        check(y, exact(x, steps))


def test_other_coefficients_reach_the_polar_factor():
    g = gen(4)
    x = noise(120, 310, g)
    y = K.newton_schulz([x], steps=12, coeffs=(15 / 8, -10 / 8, 3 / 8))[0]
    u, _, v = torch.linalg.svd(x.cpu().double(), full_matrices=False)
    check(y, u @ v)
    check(y, exact(x, 12, (15 / 8, -10 / 8, 3 / 8)))
    check(K.newton_schulz([x], steps=16, coeffs=(1.5, -0.5, 0.0))[0], exact(x, 16, (1.5, -0.5, 0.0)))


def test_strides_and_transposed_views():
    g = gen(5)
    big = noise(400, 500, g)
    views = [big[3:103, 7:207], big[::2, 100:180], big.t()[5:105, 6:300], big[:50, :300].t(), big[10:11, 5:300], big[:, 3:4],
             big[:64].view(64, 20, 25).reshape(64, 500)]
    got = K.newton_schulz(views)
    for x, y in zip(views, got):
        check(y, exact(x))
    # a transposed view is the same problem: the very same numbers
    a, b = K.newton_schulz([big, big.t()])
    assert torch.equal(a, b.t())


def test_scale_of_the_input_does_not_matter():
    g = gen(6)
    x = torch.randn(96, 160, generator=g).cuda()
    base = exact(x)
    for s in (1e-15, 1e-6, 1.0, 1e6, 1e18):
        check(K.newton_schulz([x * s], eps=0.0)[0], base)
    # eps counts against the norm
    tiny = x * 1e-9
    check(K.newton_schulz([tiny])[0], exact(tiny))


def test_spikes():
    g = gen(7)
    x = noise(200, 333, g)
    x[7, 11] = 5.0
    x[150] *= 300
    check(K.newton_schulz([x])[0], exact(x))


def test_identity():
    """Every number of a row is the same one here, so no rounding averages out, and TOL (root mean squares) does not hold:
    the bound is the sum of the largest roundings, u = 2^-11 of an fp16 operand.  The singular value goes 0.088, 0.30,
    0.91, 0.81, 0.96, 0.73; f' = a + 3 b s^2 + 5 c s^4 along it is 3.33, 2.24, -1.46, -1.61, -1.10.  An error of the third step
    (no shift yet, s^2 = 0.82): X 2 u / s^2-part counted in E, E 0.82 |b + 2 c 0.82| u = 1.2 u, F = 2.55 u, of X 0.9, X itself
    (hi + lo) none, its product 2.55 u: 6.3 u 0.9 / 0.81; it reaches the end times 1.61 * 1.10 and relative to 0.73 against
    0.81: 14 u at the very most if all fall on one side; half of it (7 u) is granted, and 2 u for each of the last two
    steps (E - 1 and F below 0.7): 11 u = 5.4e-3, and the output's own 2^-8: 9.3e-3."""
    for m, n in ((130, 140), (300, 256)):
        e = torch.eye(m, n).cuda()
        check(K.newton_schulz([e])[0], exact(e), 9.3e-3)


def test_zero_and_nonfinite_matrices_keep_to_themselves():
    g = gen(8)
    a, b, c, z = noise(130, 90, g), noise(130, 90, g), noise(130, 90, g), torch.zeros(130, 90, device="cuda")
    b[4, 5], c[129, 89] = math.nan, math.inf
    got = K.newton_schulz([a, b, z, c])
    assert got[1].isnan().all() and got[3].isnan().all() and not got[2].any()
    assert torch.equal(got[0], K.newton_schulz([a])[0])


def test_many_shapes_and_matrices_in_one_call():
    g = gen(9)
    mats = [noise(8 + 5 * (i % 23), 70 - 3 * (i % 19), g, BF16 if i % 3 else F32) for i in range(150)] + \
           [noise(33, 44, g) for _ in range(70)]
    got = K.newton_schulz(mats)
    for x, y in zip(mats, got):
        check(y, exact(x))
    for i in (0, 17, 149, 160, 219):
        assert torch.equal(got[i], K.newton_schulz([mats[i]])[0])


def test_same_tensor_twice_and_repeatable():
    g = gen(10)
    x = noise(256, 384, g)
    a, b = K.newton_schulz([x, x])
    assert torch.equal(a, b) and a.data_ptr() != b.data_ptr()
    assert torch.equal(a, K.newton_schulz([x])[0])


def test_graph_replays_on_other_inputs_and_streams():
    g = gen(11)
    hold = [noise(160, 200, g), noise(200, 160, g, BF16), noise(64, 64, g)]
    fresh = [[t.clone() for t in hold], [t.flip(0).contiguous() for t in hold], [t * 3 + 1e-4 for t in hold]]
    K.newton_schulz(hold)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.newton_schulz(hold)
    with torch.cuda.graph(other):
        got2 = K.newton_schulz(hold[:1])
    for new in fresh + fresh[:1]:
        for t, v in zip(hold, new):
            t.copy_(v)
        graph.replay()
        other.replay()
        eager = K.newton_schulz(new)
        torch.cuda.synchronize()
        for x, y in zip(got, eager):
            assert torch.equal(x, y)
        assert torch.equal(got2[0], eager[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = K.newton_schulz(fresh[0])
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(there, eager):
        assert torch.equal(x, y)


def test_plan_on_another_stream_and_after_a_move():
    g = gen(13)
    mats = [noise(100, 70, g), noise(130, 300, g)]
    plan = K.NewtonSchulzPlan(mats)
    want = [t.clone() for t in plan.run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = plan.run()
    del plan                                       # (its workspace is still being read)
    junk = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(8)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(junk) == 8
    plan = K.NewtonSchulzPlan(mats)
    mats[1].data = mats[1].clone()
    with pytest.raises(RuntimeError, match="moved"):
        plan.run()


def test_refuses_what_it_does_not_take():
    x = torch.randn(8, 9, device="cuda")
    for bad in ([x.half()], [x[0]], [x.double()], [x[:0]], [x.cpu()], [x, x.cpu()], [x[:, ::2][::2]], [x.expand(8, 9)[:1].expand(8, 9)]):
        with pytest.raises(ValueError):
            K.newton_schulz(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(coeffs=(1.0, 2.0)), dict(coeffs=(257.0, 0.0, 0.0)), dict(coeffs=(1.0, math.nan, 0.0)), dict(eps=-1.0), dict(eps=math.nan)):
        with pytest.raises(ValueError):
            K.newton_schulz([x], **kw)
