"""The selection's log-sum-exp where a workgroup adds up a whole row: few rows share a row out over
workgroups, many do not."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from test_gpu_beams import A, TYPES, VOCAB  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def rows():
    """Rows whose fp32 sums go wrong by many roundings to one side, and ones that ascend."""
    rng = np.random.default_rng(0)
    at = np.arange(VOCAB)
    for low, first in ((-12.25, 8192), (-11.0, 900), (-7.0, 20), (-19.5, 3), (-0.5, 1000)):
        yield np.where(at < first, 0.0, low)
    yield at * (3.0 / VOCAB)
    yield at * (40.0 / VOCAB)
    yield np.full(VOCAB, 3.25)
    yield np.where(at % 8192 == 0, at / 8192 * 0.9, -30.0 + at / 8192)
    yield rng.standard_normal(VOCAB) * 3


@TYPES
@pytest.mark.parametrize("count", [4, 128, 512])
def test_sums_of_whole_rows(A, count, f32):  # noqa: F811
    """Scores within the bound of test_gpu_beams.py: 2^-24 of themselves for their own rounding and
    2^-20 for the logarithm; beams whose scores are 4 2^-20 apart in their order."""
    width, k = 4, 8
    for x in rows():
        x = x.astype(np.float32) if f32 else O.bf16_to_f32(O.f32_to_bf16(x.astype(np.float32)))
        x64 = x.astype(np.float64)
        lse = x64.max() + np.log(np.exp(x64 - x64.max()).sum())
        s = np.array([-4, 0, -8, -1000], dtype=np.float32) * np.float32(2.0 ** -20)
        line = torch.from_numpy(x).cuda().to(torch.float32 if f32 else torch.bfloat16)
        logits = line.repeat(count, 1)
        got = [t.cpu().numpy() for t in
               A.beam_top_k(logits, torch.from_numpy(np.tile(s, (count // width, 1))).cuda(), k)]
        want, beams, tokens = AO.beam_top_k(np.tile(x, (width, 1)), s, k)
        assert abs(want[0] - (x64.max() - lse)) < 1e-9
        for i in range(count // width):
            np.testing.assert_array_equal(got[1][i], beams)
            np.testing.assert_array_equal(got[2][i], tokens)
            off = np.abs(got[0][i] - want)
            assert (off <= 2.0 ** -24 * np.abs(want) + 2.0 ** -20).all(), (off.max(), x[:3])
