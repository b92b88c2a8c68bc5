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


def kinds(x):
    return np.where(np.isnan(x), 2, np.where(np.isposinf(x), 1, np.where(np.isneginf(x), -1, 0)))


@pytest.mark.parametrize("m", [3, 7, 14, 30, 45])
@pytest.mark.parametrize("window", [0, 70])
def test_infinities_and_nan_of_v(A, m, window):  # noqa: F811
    """v of a bf16 cache holds infinities of both signs and NaN, in blocks that every node sees whole,
    at a window's edge and in the tree: who sees +inf alone in a dimension gets +inf, -inf alone
    -inf, both or a NaN gets NaN, whatever block the key lies in; who does not see it a number."""
    rng = np.random.default_rng(m)
    special = np.array([0x7F80, 0xFF80, 0x7FC0, 0xFFC1, 0x7F81], dtype=np.uint16)
    cached, nodes = [0, 50, 130, 700], [m, m, m, max(1, m - 2)]
    for seed in range(3):
        k = [bf(rng.standard_normal((c + n, 8, 64)) * 0.5) for c, n in zip(cached, nodes)]
        v = [bf(rng.standard_normal((c + n, 8, 64))) for c, n in zip(cached, nodes)]
        for b, (c, n) in enumerate(zip(cached, nodes)):
            for key in [c + i for i in range(0, n, 2)] + [c - 1, c - 2, c - 40, c - 64, c - 70, 5, 64]:
                if 0 <= key < c + n:       # a few dimensions of one kv head
                    h = rng.integers(0, 8)
                    d = rng.choice(64, 3, replace=False)
                    v[b][key, h, d] = rng.choice(special, 3)
            if c:                          # the same dimension twice: infinities that meet
                v[b][c // 2, 3, 10], v[b][min(c + n - 1, c // 2 + 33), 3, 10] = 0x7F80, 0xFF80
                v[b][c // 2, 3, 11], v[b][c // 2 + 1, 3, 11] = 0xFF80, 0xFF80
        c = Case(400 + m + seed, False, cached, nodes, k=k, v=v, scale=0.5)
        for bound in (False, True):
            got = f64(c.run(A, window, bound))
            for b, n in enumerate(nodes):
                at = np.arange(c.starts[b], c.starts[b + 1])
                with np.errstate(invalid="ignore"):
                    ref, _, _ = AO.attention_seen(f64(c.q[at]), c.kd[b], c.vd[b], c.seen(b, window),
                                                  f64(c.sinks), SCALE)
                np.testing.assert_array_equal(kinds(got[at]), kinds(ref))
        assert (kinds(got) != 0).any()
        finite = Case(400 + m + seed, False, cached, nodes, k=k, scale=0.5,
                      v=[np.where((x & 0x7F80) == 0x7F80, np.uint16(0), x) for x in v])
        clean = f64(finite.run(A, window))
        number = kinds(got) == 0
        # (keys that a row does not see have nothing to do with it: the same bits)
        for b, n in enumerate(nodes):
            at = np.arange(c.starts[b], c.starts[b + 1])
            np.testing.assert_array_equal(got[at][number[at]], clean[at][number[at]])
