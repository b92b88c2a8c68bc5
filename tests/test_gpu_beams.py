"""Beam search on the GPU: the selection against the oracle's in fp64, the pages that beams copy,
and the engine's search and tree verification."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from gpu_util import bf16_dev, f32_dev, host_bf16, i32_dev, u8_dev  # noqa: E402

pytestmark = pytest.mark.gpu

VOCAB = 201088


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import attn_native
    return attn_native


def select(A, logits, scores, k, f32=False):
    """logits [batch, width, vocab] fp32 (bf16 values unless f32), checked against the oracle:
    beams and tokens exactly; scores within 2^-24 of their size for the one rounding, and
    2^-20 for the logarithm of a sum of fp32 exponentials (each off by a few 2^-24 of
    itself and of its exponent)."""
    batch, width, vocab = logits.shape
    flat = logits.reshape(batch * width, vocab)
    dev = f32_dev(flat) if f32 else bf16_dev(O.f32_to_bf16(flat))
    got = [t.cpu().numpy() for t in A.beam_top_k(dev, f32_dev(scores), k)]
    assert got[0].shape == got[1].shape == got[2].shape == (batch, k)
    for b in range(batch):
        want, beams, tokens = AO.beam_top_k(logits[b], scores[b], k)
        np.testing.assert_array_equal(got[1][b], beams)
        np.testing.assert_array_equal(got[2][b], tokens)
        fine = np.isfinite(want)
        np.testing.assert_array_equal(got[0][b][~fine], want[~fine].astype(np.float32))
        assert (np.abs(got[0][b][fine] - want[fine])
                <= 2.0 ** -24 * np.abs(want[fine]) + 2.0 ** -20).all()
    return got


def draw(rng, batch, width, vocab, f32=False, sigma=2.5):
    x = (rng.standard_normal((batch, width, vocab)) * sigma).astype(np.float32)
    scores = -np.sort(rng.random((batch, width)) * 20, axis=1).astype(np.float32)
    return (x if f32 else O.bf16_to_f32(O.f32_to_bf16(x))), scores


TYPES = pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])


@TYPES
@pytest.mark.parametrize("batch,width,k", [(1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 8, 16)])
def test_full_vocabulary(A, batch, width, k, f32):
    for sigma in (0.3, 2.5, 12.0):
        select(A, *draw(np.random.default_rng(width), batch, width, VOCAB, f32, sigma), k, f32)


@TYPES
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1000, 1001, 4097, 16383, 16385, 50257])
def test_sizes(A, vocab, f32):
    """Rows that begin at any element, up to every candidate there is."""
    rng = np.random.default_rng(vocab)
    for width, k in ((1, 1), (3, 6), (7, 14), (64, 64)):
        if width * vocab > 500000:
            continue
        select(A, *draw(rng, 2, width, vocab, f32), min(k, width * vocab), f32)


@TYPES
def test_equal_scores(A, f32):
    """Ties go to the lowest beam, then the lowest token: constant rows, the same rows in
    several beams, the best ones together in one place."""
    for vocab in (5, 700, 40000):
        x = np.zeros((2, 4, vocab), dtype=np.float32)
        got = select(A, x, np.zeros((2, 4), dtype=np.float32), 20 if vocab == 5 else 32, f32)
        assert got[1][0, 0] == 0 and got[2][0, 1] == 1
        x[:, :, vocab // 2:vocab // 2 + 40] = 3.0
        select(A, x, np.zeros((2, 4), dtype=np.float32), 20, f32)
        x[1, 2] += 0.5                                # a constant more changes no row's scores
        x[:, :, -1] = 9.0
        select(A, x, np.array([[0, -1, 0, -1], [-3, -3, -3, -3]], dtype=np.float32), 20, f32)
    rng = np.random.default_rng(5)
    x = rng.integers(0, 4, (1, 6, 30000)).astype(np.float32)      # thousands of the largest value
    select(A, x, np.zeros((1, 6), dtype=np.float32), 64, f32)
    x[0, :, 12345:12345 + 70] = 5.0
    select(A, x, np.zeros((1, 6), dtype=np.float32), 64, f32)
    x = np.sort(x, axis=2)                                        # the best at one end
    select(A, x, np.zeros((1, 6), dtype=np.float32), 64, f32)
    select(A, x[:, :, ::-1].copy(), np.zeros((1, 6), dtype=np.float32), 64, f32)


@TYPES
def test_masked_and_bad_rows(A, f32):
    """Tokens ruled out by -inf or the type's lowest value, beams that have ended, rows without
    a maximum."""
    rng = np.random.default_rng(6)
    for vocab in (300, 20001):
        x, s = draw(rng, 2, 8, vocab, f32)
        lowest = np.finfo(np.float32).min if f32 else np.float32(-3.3895314e38)
        x[:, :, rng.random(vocab) < 0.9] = -np.inf
        x[0, 1], x[0, 2, 5], x[0, 3, vocab - 1] = -np.inf, np.nan, np.inf
        x[0, 4, 3:] = -np.inf
        x[1, 0, 7:] = lowest
        s[0, 5], s[0, 6], s[1, 3] = -np.inf, np.nan, -np.inf
        select(A, x, s, 16, f32)
        s[:, 1:] = -np.inf                            # a request's first step: one beam alone
        select(A, x, s, 16, f32)
        x[:] = -np.inf                                # nothing at all: the first candidates
        got = select(A, x, s, 16, f32)
        assert (got[0] == -np.inf).all() and (got[2] == np.arange(16)).all()


def test_one_beam_leads(A):
    """All of the best ones in one beam, or one stretch of it; far scores."""
    rng = np.random.default_rng(7)
    x, s = draw(rng, 1, 8, 60000)
    for lead in (0, 3, 7):
        t = s.copy()
        t[0] -= 1000.0
        t[0, lead] = 0.0
        select(A, x, t, 16)
    x[0, 2, 777:777 + 64] = 40.0
    select(A, x, s, 64)


def test_beams_stream_and_graph(A):
    rng = np.random.default_rng(8)
    x, s = draw(rng, 3, 4, 30001)
    logits, scores = bf16_dev(O.f32_to_bf16(x.reshape(12, -1))), f32_dev(s)

    def call():
        return A.beam_top_k(logits, scores, 8)

    want = [t.clone() for t in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(4):
        logits.copy_(logits.roll(777, dims=1).flip(0))
        scores.mul_(1.25)
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("n,layers", [(1, 1), (2, 24), (37, 3), (300, 2)])
def test_copy_pages(A, fp8, n, layers):
    rng = np.random.default_rng(n)
    pool = 2 * n + 2
    shape = (layers, pool, AO.FP8_PAGE_BYTES) if fp8 else (layers, pool, 2, 8, 16, 64)
    cache = rng.integers(0, 256 if fp8 else 65536, shape, dtype=np.uint8 if fp8 else np.uint16)
    dev = u8_dev(cache) if fp8 else bf16_dev(cache)
    ids = rng.permutation(pool)
    src, dst = ids[:n][rng.integers(0, n, n)], ids[n:2 * n].copy()
    if n > 3:                                          # outside the pool: not written
        src[1], dst[2], dst[3] = pool, -1, 1 << 30
    assert A.kv_copy_pages(dev, i32_dev(src), i32_dev(dst)) is dev
    for a, b in zip(src, dst):
        if 0 <= a < pool and 0 <= b < pool:
            cache[:, b] = cache[:, a]
    np.testing.assert_array_equal(dev.cpu().numpy() if fp8 else host_bf16(dev), cache)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    A.kv_copy_pages(dev, e, e)


@TYPES
@pytest.mark.parametrize("batch,vocab", [(1, 20001), (16, 30011)])  # (a chunk a stretch, several)
def test_few_tokens_left(A, batch, vocab, f32):
    """A mask that leaves no, fewer than k, k or some more tokens, by -inf, the type's lowest value
    and a number: the rest counts too, in its order."""
    rng = np.random.default_rng(vocab)
    x, s = draw(rng, batch, 8, vocab, f32)
    s[:, 1] = s[:, 0]
    low = np.finfo(np.float32).min if f32 else np.float32(-3.3895314e38)
    for masked in (-np.inf, low, np.float32(-32768.0)):
        for left in (0, 1, 15, 16, 17, 100, 2000):
            y = np.full_like(x, masked)
            for b in range(batch):
                at = rng.choice(vocab, left, replace=False)
                y[b, :, at] = x[b, :, at]
            y[:, 1] = y[:, 0]                         # equal scores in two beams
            select(A, y, s, 16, f32)
    y = np.full_like(x, -np.inf)                      # what is left differs from beam to beam
    for b in range(batch):
        for w in range(8):
            at = rng.choice(vocab, w * w // 3, replace=False)
            y[b, w, at] = x[b, w, at]
    for k in (1, 8, 64):
        select(A, y, s, k, f32)


@TYPES
def test_best_in_few_lanes(A, f32):
    """The largest numbers in a few columns of 16 bytes that come again and again: most lanes' maxima
    say little of them."""
    rng = np.random.default_rng(8)
    for vocab in (8192, 50001):
        x, s = draw(rng, 1, 4, vocab, f32)
        column = np.arange(vocab) // (4 if f32 else 8) % 64
        x[:, :, column < 10] += 40.0
        x = x if f32 else O.bf16_to_f32(O.f32_to_bf16(x))
        select(A, x, s, 64, f32)
        select(A, x, s, 16, f32)


@TYPES
def test_scores_equal_and_logits_not(A, f32):
    """Beside a logit of 1e38 all others' scores are the same number, -1e38 in fp64 too: equal scores
    go by beam, then by the logits, then by token."""
    rng = np.random.default_rng(9)
    for vocab, width in ((3000, 3), (VOCAB, 8)):
        x = O.bf16_to_f32(O.f32_to_bf16(rng.standard_normal((1, width, vocab)).astype(np.float32)))
        x[0, :, vocab // 3] = O.bf16_to_f32(O.f32_to_bf16(np.array([1e38], np.float32)))
        dev = f32_dev(x[0]) if f32 else bf16_dev(O.f32_to_bf16(x[0]))
        score, beams, tokens = [t.cpu().numpy()[0] for t in
                                A.beam_top_k(dev, f32_dev(np.zeros((1, width), np.float32)), 16)]
        best = np.argsort(-x[0, 0], kind="stable")[:17 - width]       # of the first beam
        np.testing.assert_array_equal(beams, [*range(width), *[0] * (16 - width)])
        np.testing.assert_array_equal(tokens, [*[vocab // 3] * width, *best[1:]])
        assert (score[:width] == 0).all() and (score[width:] == -x[0, 0, vocab // 3]).all()
