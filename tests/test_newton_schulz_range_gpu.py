"""Matrices at the ends of fp32's range (eps = 0): the factor does not depend on the matrix's scale, as long as the numbers
themselves keep their digits.  Tolerances: test_newton_schulz_gpu.py's; the comparison is with the 64-bit iteration of
the numbers as they are (those near 2^-149 have few digits left, but they are what is given)."""
import pytest
import torch

from dphubert_amd import kernels as K
from test_newton_schulz_gpu import BF16, F32, check, exact, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(1, 1), (5, 3), (96, 160), (300, 421)])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("up", [-140, -133, -127, -100, 100, 125])
def test_scales(m, n, dt, up):
    x = torch.randn(m, n, generator=gen(m + n)).clamp(-3.9, 3.9)
    # (by two factors that fp32 holds; exact but for the digits that leave at the bottom)
    x = (x.to(dt).float() * 2.0 ** (up // 2) * 2.0 ** (up - up // 2)).to(dt).cuda()
    assert x.isfinite().all()
    if not x.any():
        pytest.skip("nothing is left of such numbers in this type")
    check(K.newton_schulz([x], eps=0.0)[0], exact(x, eps=0.0))
