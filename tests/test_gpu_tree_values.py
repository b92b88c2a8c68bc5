"""Tree attention's numerics: how many bits a probability keeps, and where infinities and NaN of v
go."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from test_gpu_tree import (BOTH, HQ, SCALE, U, A, Case, bf, f64,  # noqa: E402, F401
                           tree_bits)

pytestmark = pytest.mark.gpu


@BOTH
@pytest.mark.parametrize("m", [1, 4, 5, 8, 11, 16, 17, 32, 40])
def test_probabilities_keep_16_bits(A, fp8, m):  # noqa: F811
    """|out - exact| <= u |exact| + (e + 2 d) A as test_gpu_tree.py has it, but for e: probabilities in
    two bf16 pieces are off by u^2 = 2^-16 of themselves, the fp32 sums and exponentials by 2^-14.
    Where |exact| is small beside A (values of both signs) roundings to one piece, 2^-8 A at most,
    are far past the bound's second part.  (The 8-bit cache's tiles of 32 tokens have one piece,
    and the wider bound.)"""
    for cached in (0, 3, 40, 1500):
        c = Case(300 + m, fp8, [cached], [m], scale=0.3, spread=0.3)
        e = 2.0 ** -14 + (U if fp8 and m > 16 else U * U)
        for bound in (False, True):
            got = f64(c.run(A, 0, bound))
            ref, mag, size = AO.attention_seen(f64(c.q), c.kd[0], c.vd[0], c.seen(0, 0),
                                               f64(c.sinks), SCALE)
            tol = U * np.abs(ref) + (e + 2 * 2.0 ** -17 * size[..., None]) * mag
            assert (np.abs(got - ref) <= tol).all(), np.max((np.abs(got - ref) - tol) / mag)
