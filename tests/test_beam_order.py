"""The oracle's order of continuations of equal scores is the documented one."""
import numpy as np

from oracle import attn_oracle as AO


def test_equal_scores_by_beam_logit_token():
    """Beside a logit of 1e38 every other score is -1e38 in fp64 (its step there is 2^74)."""
    x = np.array([[1.0, 3.0, 1e38, 3.0, -2.0], [5.0, 1e38, 0.0, 7.0, 7.0]])
    s, b, t = AO.beam_top_k(x, np.zeros(2), 10)
    assert s.tolist() == [0.0] * 2 + [-1e38] * 8
    assert b.tolist() == [0, 1] + [0] * 4 + [1] * 4
    assert t.tolist() == [2, 1] + [1, 3, 0, 4] + [3, 4, 0, 2]


def test_minus_infinity_by_beam_and_token():
    """Beams that have ended, rows without a maximum, tokens that are ruled out."""
    inf = np.inf
    x = np.array([[1.0, 3.0, 2.0], [-inf, 4.0, -inf], [np.nan, 9.0, 1.0], [inf, 9.0, 1.0]])
    s, b, t = AO.beam_top_k(x, np.array([-inf, 0.0, 0.0, 0.0]), 12)
    assert s.tolist() == [0.0] + [-inf] * 11
    assert b.tolist() == [1] + [0] * 3 + [1] * 2 + [2] * 3 + [3] * 3
    assert t.tolist() == [1] + [0, 1, 2] + [0, 2] + [0, 1, 2] + [0, 1, 2]


def test_scores_that_differ_go_by_score():
    rng = np.random.default_rng(0)
    x, scores = rng.standard_normal((5, 40)), rng.standard_normal(5)
    s, b, t = AO.beam_top_k(x, scores, 200)
    every = scores[:, None] + x - np.log(np.exp(x).sum(axis=1, keepdims=True))
    np.testing.assert_allclose(s, np.sort(every.ravel())[::-1])
    np.testing.assert_allclose(s, every[b, t])
