"""Which tiles the sizes of test_tiles_gpu.py take, by the rule of csrc/mfma_tile.h itself (its two functions, compiled
for the host): a rule that is tuned anew has to leave every tile with sizes of its own there."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

import test_tiles_gpu as T

CSRC = Path(T.K.__file__).resolve().parent / "csrc"


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    head = (CSRC / "mfma_tile.h").read_text()
    rule = re.search(r"^inline double pairs\(.*?^}\n.*?^inline int choose_tile\(.*?^}\n", head, re.M | re.S).group(0)
    at = tmp_path_factory.mktemp("tile")
    (at / "t.cpp").write_text("#include <cstdint>\nstatic int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }\n"
                              + rule + 'extern "C" int f(int64_t a, int64_t b, int64_t c) { return choose_tile(a, b, c); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(at / "t.so"), str(at / "t.cpp")], check=True)
    f = ctypes.CDLL(str(at / "t.so")).f
    f.argtypes = [ctypes.c_int64] * 3
    return lambda count: f(*(count(b) for b in (256, 128, 64)))


def cdiv(a, b):
    return -(-a // b)


@pytest.mark.parametrize("tile,M,N,C", T.LINEAR)
def test_linear_sizes(choose, tile, M, N, C):
    assert choose(lambda b: cdiv(M, b) * cdiv(N, b)) == tile


@pytest.mark.parametrize("tile,M,N,C,keep", T.LN)
def test_layernorm_sizes(choose, tile, M, N, C, keep):
    assert choose(lambda b: cdiv(M, b) * cdiv(N, b)) == tile


@pytest.mark.parametrize("tile,shapes", T.LISTS)
def test_lists(choose, tile, shapes):
    """All four products of the list on the tile; one of its matrices alone on 64 x 64."""
    def products(groups):
        sides = [(min(m, n), max(m, n), c) for m, n, c in groups]
        assert all(m > 256 for m, _, _ in sides)          # (operands in one part, the Gram sum in one)
        square = lambda b: sum(cdiv(m, b) * (cdiv(m, b) + 1) // 2 * c for m, _, c in sides)  # noqa: E731
        return choose(square), choose(lambda b: sum(cdiv(m, b) * cdiv(n, b) * c for m, n, c in sides))

    assert products(shapes) == (tile, tile)
    for m, n, _ in shapes:
        assert products([(m, n, 1)]) == (64, 64)


def test_every_epilogue_is_there():
    assert len({(a, r, o) for a, r, o in T.EPILOGUES}) == 8
    for tile in (128, 256):
        cases = [(M, N, C) for t, M, N, C in T.LINEAR if t == tile]
        assert any(N % 2 for _, N, _ in cases) and any(N % 8 == 0 for _, N, _ in cases)
        assert any(M % 64 for M, _, _ in cases) and any(C % 16 for _, _, C in cases)
        assert any(C <= 128 for _, _, C in cases) and any(128 < C <= 256 for _, _, C in cases) and any(C > 256 for _, _, C in cases)
