"""The 8-bit KV cache on the GPU against the oracle: bit-exact where it writes and reads rows,
and the attention over it within bounds derived from its arithmetic.

The bound of an output: with u = 2^-8 (half a bf16 step) and A = sum p |v| / (sum p + exp(sink)),
|out - exact| <= u |exact| + (e + 2 d) A.  d: the relative error of a probability from its score,
64 products summed in fp32, so at most 64 2^-24 of sum |q k| scale, doubled for the exponent's own
arithmetic.  e: the rounding of the probabilities that enter the matrix product (decode: two bf16
pieces, 2^-16; chunks: up to one bf16 rounding, u) and of the fp32 sums and exponentials (2^-14,
generous)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from gpu_util import bf16_dev, f32_dev, host_bf16, i32_dev, u8_dev  # noqa: E402

pytestmark = pytest.mark.gpu

D, HQ, HKV, PAGE = 64, 64, 8, 16
SCALE = 1.0 / math.sqrt(D)
U = 2.0 ** -8
NAN_ROW = 0x7FC0


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import attn_native
    return attn_native


def bf(x):
    return O.f32_to_bf16(np.asarray(x, dtype=np.float32))


def values(rows, is_v=False):
    return AO.fp8_dequantize(*AO.fp8_quantize(rows, is_v))


def rows_of(rng, n):
    """k or v rows [n, 8, 64] with scales of all sizes and a few special ones."""
    x = rng.standard_normal((n, HKV, D)) * np.exp2(rng.integers(-20, 20, (n, HKV, 1)))
    x = bf(x)
    x[0, 0] = 0
    x[n // 2, 1, 7] = 0x7F80
    x[n // 3, 2, 63] = 0xFFC1
    x[n - 1, 3] = np.where(rng.random(D) < 0.5, 0x7F7F, 0x0001)     # largest and smallest bf16
    x[n - 1, 4] = bf(rng.standard_normal(D) * 2.0 ** -118)
    return x


def untouched(pages):
    return np.full((pages, AO.FP8_PAGE_BYTES), 0xAB, dtype=np.uint8)


@pytest.mark.parametrize("n", [1, 3, 64, 333])
def test_append_bit_exact(A, n):
    from test_gpu_attention import _inv_freq_dev
    rng = np.random.default_rng(n)
    pages = n // PAGE + 5
    qkv = bf(rng.standard_normal((n, (HQ + 2 * HKV) * D)))
    bias = bf(rng.standard_normal((HQ + 2 * HKV) * D) * 0.1)
    pos = rng.integers(0, 131072, n).astype(np.int32)
    slots = rng.choice(pages * PAGE, n, replace=False).astype(np.int32)
    if n > 2:
        qkv[1, HQ * D + 70], qkv[2, (HQ + HKV) * D + 5] = 0x7FC0, 0xFF80   # a bad k, a bad v
        slots[-1] = pages * PAGE + 5                                       # not written
    cache = u8_dev(untouched(pages))
    q = torch.empty((n, HQ, D), dtype=torch.bfloat16, device="cuda")
    inv, conc = _inv_freq_dev()
    A.qkv_rope_append_fp8(bf16_dev(qkv), bf16_dev(bias), i32_dev(pos), i32_dev(slots), inv, conc,
                          cache, q)
    rq, rk, rv = AO.split_qkv(AO.bias_add(qkv, bias))
    np.testing.assert_array_equal(host_bf16(q), AO.rope(rq, pos))
    want = untouched(pages)
    inside = slots < pages * PAGE
    AO.fp8_put(want, slots[inside], AO.rope(rk, pos)[inside], rv[inside])
    np.testing.assert_array_equal(cache.cpu().numpy(), want)


@pytest.mark.parametrize("n", [1, 2, 5, 47, 400])
@pytest.mark.parametrize("order", ["scattered", "in order", "offset"])
def test_quantize_and_read_bit_exact(A, n, order):
    """Rows anywhere, and in the order of a sequence (whole quads of tokens) from its start or
    from inside a quad."""
    rng = np.random.default_rng(100 + n)
    pages = n // PAGE + 4
    k, v = rows_of(rng, n), rows_of(rng, n)
    src = np.zeros((pages, 2, HKV, PAGE, D), dtype=np.uint16)
    if order == "scattered":
        mine = rng.choice(pages * PAGE, n, replace=False)
        slots = rng.choice(pages * PAGE, n, replace=False)
    else:
        ids, t = rng.permutation(pages), np.arange(n) + (3 if order == "offset" else 0)
        mine = slots = ids[t // PAGE] * PAGE + t % PAGE
    src[mine // PAGE, 0, :, mine % PAGE] = k
    src[mine // PAGE, 1, :, mine % PAGE] = v
    cache = u8_dev(untouched(pages))
    A.kv_quantize_fp8(bf16_dev(src), i32_dev(mine), cache, i32_dev(slots))
    want = untouched(pages)
    AO.fp8_put(want, slots, k, v)
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    gk, gv = A.kv_read_fp8(cache, i32_dev(slots))
    for got, rows, is_v in ((gk, k, False), (gv, v, True)):
        np.testing.assert_array_equal(got.double().cpu().numpy(), values(rows, is_v))


@pytest.mark.parametrize("seed", range(4))
def test_quantize_and_read_runs(A, seed):
    """Runs of tokens of all lengths from all places in a quad, upwards and downwards, up to the
    pool's last slot; source slots outside their pool in places, whose rows are not written."""
    rng = np.random.default_rng(300 + seed)
    pages = 40
    free, runs = np.ones(pages * PAGE, dtype=bool), [np.arange(pages * PAGE - 6, pages * PAGE)]
    free[runs[0]] = False
    for _ in range(90):
        a, length = rng.integers(0, pages * PAGE - 12), rng.integers(1, 12)
        run = np.arange(a, a + length)
        if free[run].all():
            free[run] = False
            runs.append(run[::-1] if rng.random() < 0.2 else run)
    slots = np.concatenate([runs[i] for i in rng.permutation(len(runs))])
    n = len(slots)
    k, v = rows_of(rng, n), rows_of(rng, n)
    mine = rng.permutation(pages * PAGE)[:n]
    src = np.zeros((pages, 2, HKV, PAGE, D), dtype=np.uint16)
    src[mine // PAGE, 0, :, mine % PAGE] = k
    src[mine // PAGE, 1, :, mine % PAGE] = v
    bad = rng.random(n) < 0.05
    cache = u8_dev(untouched(pages))
    A.kv_quantize_fp8(bf16_dev(src), i32_dev(np.where(bad, pages * PAGE, mine)), cache,
                      i32_dev(slots))
    want = untouched(pages)
    AO.fp8_put(want, slots[~bad], k[~bad], v[~bad])
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    AO.fp8_put(want, slots, k, v)
    out = rng.random(n) < 0.05
    gk, gv = A.kv_read_fp8(u8_dev(want), i32_dev(np.where(out, -slots - 1, slots)))
    for got, rows, is_v in ((gk, k, False), (gv, v, True)):
        ref = np.where(out[:, None, None], 0.0, values(rows, is_v))
        np.testing.assert_array_equal(got.double().cpu().numpy(), ref)


def test_quantize_and_read_slots_outside(A):
    rng = np.random.default_rng(7)
    src = bf(rng.standard_normal((2, 2, HKV, PAGE, D)))
    mine = np.array([0, 31, 32, -1, 5, 6], dtype=np.int32)
    slots = np.array([2, -1, 3, 4, 48, 5], dtype=np.int32)
    cache = u8_dev(untouched(3))
    A.kv_quantize_fp8(bf16_dev(src), i32_dev(mine), cache, i32_dev(slots))
    want = untouched(3)
    good = [0, 5]
    AO.fp8_put(want, slots[good], src[0, 0][:, mine[good]].transpose(1, 0, 2),
               src[0, 1][:, mine[good]].transpose(1, 0, 2))
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    k, v = A.kv_read_fp8(cache, i32_dev(np.array([2, -1, 48, 5, 2, 1 << 30], dtype=np.int32)))
    want = values(src[0, 1][:, mine[[0, 5]]].transpose(1, 0, 2))
    got = v.double().cpu().numpy()
    np.testing.assert_array_equal(got[[0, 3, 4]], want[[0, 1, 0]])   # a slot may be read twice
    assert not got[[1, 2, 5]].any() and not k[[1, 2, 5]].any().item()
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    assert A.kv_read_fp8(cache, e)[0].shape == (0, HKV, D)
    A.kv_quantize_fp8(bf16_dev(src), e, cache, e)


class Seqs:
    """Sequences of random rows on scattered pages of an 8-bit cache; every byte that no token
    owns is 0xFF (codes and scales that stand for NaN)."""

    def __init__(self, seed, lengths, k=None, v=None, pool=None, spread=1.0):
        rng = np.random.default_rng(seed)
        need = [-(-L // PAGE) for L in lengths]
        pool = pool or sum(need) + 3
        perm = rng.permutation(pool)
        gain = np.exp(0.5 * rng.standard_normal((HKV, D)))
        self.k = k or [bf(rng.standard_normal((L, HKV, D)) * gain) for L in lengths]
        self.v = v or [bf(rng.standard_normal((L, HKV, D))
                          * np.exp(spread * rng.standard_normal((L, 1, 1)))) for L in lengths]
        cache = np.full((pool, AO.FP8_PAGE_BYTES), 0xFF, dtype=np.uint8)
        indptr, ids = [0], []
        for L, kr, vr, npg in zip(lengths, self.k, self.v, need):
            mine = perm[len(ids):len(ids) + npg]
            p = np.arange(L)
            AO.fp8_put(cache, mine[p // PAGE] * PAGE + p % PAGE if L else p, kr, vr)
            ids.extend(mine.tolist())
            indptr.append(len(ids))
        self.kd, self.vd = [values(x) for x in self.k], [values(x, True) for x in self.v]
        self.cache, self.lengths = u8_dev(cache), lengths
        self.page_indptr = i32_dev(np.array(indptr))
        self.page_indices = i32_dev(np.array(ids or [0]))
        self.kv_len = i32_dev(np.array(lengths))

    def tables(self):
        return self.cache, self.page_indptr, self.page_indices, self.kv_len


def within(got, q, k, v, pos, window, sinks, e):
    ref, mag, size = AO.attention_sink(O.bf16_to_f32(q).astype(np.float64), k, v, pos, window,
                                       O.bf16_to_f32(sinks).astype(np.float64), SCALE)
    tol = U * np.abs(ref) + (e + 2.0 ** -14 + 2 * 2.0 ** -17 * size[..., None]) * mag
    g = O.bf16_to_f32(got).astype(np.float64)
    np.testing.assert_array_equal(np.isnan(g), np.isnan(ref))
    ok = np.isnan(ref) | (np.abs(g - ref) <= tol)
    assert ok.all(), (np.argwhere(~ok)[:5], g[~ok][:5], ref[~ok][:5], tol[~ok][:5])


def run_decode(A, seqs, q, sinks, window, span=None, ws=None):
    n = len(seqs.lengths)
    span = span or max(1, max(min(L, window) if window else L for L in seqs.lengths))
    if ws is None:
        ws = A.decode_fp8_workspace(n, span)
    out = torch.full((n, HQ, D), 7.0, dtype=torch.bfloat16, device="cuda")
    A.decode_fp8(bf16_dev(q), *seqs.tables(), span, window, SCALE, bf16_dev(sinks), out, ws)
    return host_bf16(out)


def check_decode(A, seqs, window, seed, scale=2.0):
    rng = np.random.default_rng(seed)
    n = len(seqs.lengths)
    q, sinks = bf(rng.standard_normal((n, HQ, D)) * scale), bf(rng.standard_normal(HQ))
    got = run_decode(A, seqs, q, sinks, window)
    for b, L in enumerate(seqs.lengths):
        within(got[b:b + 1], q[b:b + 1], seqs.kd[b], seqs.vd[b], np.array([L - 1]), window, sinks,
               2.0 ** -16)
    return q, sinks, got


@pytest.mark.parametrize("window", [0, 1, 100, 128])
def test_decode(A, window):
    check_decode(A, Seqs(1, [1, 130, 0, 15, 16, 17, 63, 64, 65, 1000, 4100]), window, 2)


@pytest.mark.parametrize("L", [1, 64, 255, 256, 257, 511, 513, 777, 1025, 5000, 17000])
def test_decode_one_sequence(A, L):
    """One sequence: one split, several, and more keys than 64 splits of four blocks hold."""
    check_decode(A, Seqs(L, [L]), 0, L + 1)


def test_decode_many_sequences(A):
    rng = np.random.default_rng(3)
    check_decode(A, Seqs(4, rng.integers(1, 700, 70).tolist()), 0, 5)
    check_decode(A, Seqs(6, rng.integers(1, 300, 300).tolist()), 128, 7)


def test_decode_sharp_and_far_scores(A):
    """Scores to +-100 and more, the largest anywhere; values of very different sizes."""
    check_decode(A, Seqs(8, [900, 70, 2000], spread=6.0), 0, 9, scale=20.0)


def test_decode_sinks(A):
    """Sinks that take nothing, everything, or more than the keys."""
    seqs = Seqs(10, [300, 0])
    q = bf(np.random.default_rng(11).standard_normal((2, HQ, D)))
    sinks = bf(np.resize([-np.inf, np.inf, 40.0, -40.0, 3e38, -3e38], HQ))
    got = O.bf16_to_f32(run_decode(A, seqs, q, sinks, 0))
    with np.errstate(all="ignore"):
        ref, mag, _ = AO.attention_sink(O.bf16_to_f32(q[:1]).astype(np.float64), seqs.kd[0],
                                        seqs.vd[0], np.array([299]), 0,
                                        np.clip(O.bf16_to_f32(sinks).astype(np.float64), -1e30, 1e30),
                                        SCALE)
    assert (np.abs(got[:1] - ref) <= U * np.abs(ref) + 2.0 ** -12 * mag).all()
    assert not got[1].any()                            # no key: 0, whatever the sink


def test_decode_bound_and_workspace(A):
    """The result follows from the keys and the batch alone: any bound on the span, workspaces
    used before by other batches; the counts are left zero."""
    seqs = Seqs(12, [3000, 200, 1])
    one = Seqs(13, [40000])
    rng = np.random.default_rng(14)
    q, sinks = bf(rng.standard_normal((3, HQ, D))), bf(rng.standard_normal(HQ))
    q1 = bf(rng.standard_normal((1, HQ, D)))
    ws = A.decode_fp8_workspace(64, 1 << 17)
    first = run_decode(A, seqs, q, sinks, 0)
    lone = run_decode(A, one, q1, sinks, 0)
    for span in (3000, 3001, 4096, 1 << 17):
        np.testing.assert_array_equal(run_decode(A, seqs, q, sinks, 0, span, ws), first)
        np.testing.assert_array_equal(run_decode(A, one, q1, sinks, 0, 1 << 17, ws), lone)
        assert int(ws[:2 << 20].count_nonzero()) == 0
    got = O.bf16_to_f32(run_decode(A, seqs, q, sinks, 0, 2999))   # one sequence is too long
    assert np.isnan(got[0]).all()
    np.testing.assert_array_equal(got[1:], O.bf16_to_f32(first[1:]))


def test_decode_bad_rows(A):
    """A token with a NaN in k or an infinity in v: NaN for the heads and queries that see it,
    nothing for those whose window has passed it."""
    seqs0 = Seqs(15, [400, 400, 400])
    k, v = [x.copy() for x in seqs0.k], [x.copy() for x in seqs0.v]
    k[0][100, 3, 5], v[1][100, 4, 9] = NAN_ROW, 0x7F80
    k[2][300, 0, 0], v[2][390, 7, 1] = 0xFF80, NAN_ROW
    seqs = Seqs(15, [400, 400, 400], k=k, v=v)
    assert int((seqs.cache != seqs0.cache).sum()) > 0
    for window in (0, 128):
        _, _, got = check_decode(A, seqs, window, 16)
        bad = np.isnan(O.bf16_to_f32(got)).any(axis=-1).reshape(3, HKV, 8)
        want = np.zeros((3, HKV), dtype=bool)
        want[2, [0, 7]] = True
        want[0, 3] = want[1, 4] = window == 0
        np.testing.assert_array_equal(bad, np.repeat(want[..., None], 8, -1))


def run_prefill(A, seqs, q, qlens, sinks, window, bound, extra=0, longest=None):
    n = sum(qlens)
    indptr = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
    out = torch.full((n + extra, HQ, D), 7.0, dtype=torch.bfloat16, device="cuda")
    qd = torch.zeros((n + extra, HQ, D), dtype=torch.bfloat16, device="cuda")
    qd[:n] = bf16_dev(q)
    A.prefill_fp8(qd, i32_dev(indptr), longest or max(qlens), *seqs.tables(), window, SCALE,
                  bf16_dev(sinks), out, bound)
    got = host_bf16(out)
    assert (got[n:] == 0x40E0).all()                   # rows behind the last sequence stay (7.0)
    return got[:n], indptr


def check_prefill(A, seqs, qlens, window, seed, bound=0, rows=None, scale=2.0, extra=3):
    rng = np.random.default_rng(seed)
    q, sinks = bf(rng.standard_normal((sum(qlens), HQ, D)) * scale), bf(rng.standard_normal(HQ))
    got, indptr = run_prefill(A, seqs, q, qlens, sinks, window, bound, extra)
    for b, (L, n) in enumerate(zip(seqs.lengths, qlens)):
        pick = np.arange(n) if rows is None else np.unique(np.clip(rows, 0, n - 1))
        if not n:
            continue
        at = indptr[b] + pick
        within(got[at], q[at], seqs.kd[b], seqs.vd[b], L - n + pick, window, sinks, U)
    return q, sinks, got


@pytest.mark.parametrize("window", [0, 1, 100, 128])
@pytest.mark.parametrize("qlens,prefix", [
    ([300], [0]), ([1, 64, 0, 65, 200], [0, 5, 40, 100, 37]), ([5, 5, 3, 8, 9], [700, 64, 1, 0, 63]),
    ([2, 1, 4], [0, 0, 130]), ([33, 17, 127], [500, 0, 15])])
def test_prefill(A, window, qlens, prefix):
    lengths = [p + q for p, q in zip(prefix, qlens)]
    seqs = Seqs(20 + len(qlens), lengths)
    for bound in (0, max(lengths)):                    # keys not shared out, and shared out
        check_prefill(A, seqs, qlens, window, 21, bound)


@pytest.mark.parametrize("qlens,prefix,window", [
    ([5], [9000], 0), ([300], [6000], 0), ([64, 64], [3000, 5], 0), ([9], [1500], 0),
    ([16], [2000], 1000), ([700], [0], 0), ([1] * 40, list(range(0, 4000, 100)), 0)])
def test_prefill_shared_keys(A, qlens, prefix, window):
    lengths = [p + q for p, q in zip(prefix, qlens)]
    seqs = Seqs(30, lengths)
    rows = np.array([0, 1, 7, 8, 63, 64, 100, 255, 256, 299, 699])
    check_prefill(A, seqs, qlens, window, 31, max(lengths), rows)
    check_prefill(A, seqs, qlens, window, 31, 4 * max(lengths), rows)   # a bound far above


@pytest.mark.parametrize("qlens,prefix", [
    ([700], [0]), ([1000], [1000]), ([400], [400]), ([130], [2300]),
    ([64, 33, 0, 1], [1500, 40, 9, 0]),
    ([520, 3, 40], [0, 600, 1]), ([30] * 9, list(range(0, 1800, 200)))])
def test_prefill_shared_keys_in_halves(A, qlens, prefix):
    """Tiles whose keys two halves of a workgroup take: of none, one and many blocks, in one share
    and in several, with scores that leave one half all the weight."""
    lengths = [p + q for p, q in zip(prefix, qlens)]
    seqs = Seqs(32, lengths)
    rows = np.array([0, 1, 31, 32, 63, 64, 65, 100, 127, 128, 299, 399, 511, 640, 699, 999])
    for scale in (2.0, 8.0):
        check_prefill(A, seqs, qlens, 0, 33, max(lengths), rows, scale=scale)


def test_prefill_bad_rows_in_halves(A):
    """As test_prefill_bad_rows, with the bad tokens in either half of a tile's keys."""
    L, n = 1500, 700
    seqs0 = Seqs(62, [L])
    k, v = [x.copy() for x in seqs0.k], [x.copy() for x in seqs0.v]
    k[0][100, 2, 5], v[0][1200, 6, 9], k[0][1499, 1, 0] = NAN_ROW, 0xFF80, 0x7F80
    seqs = Seqs(62, [L], k=k, v=v)
    rows = np.array([0, 350, 398, 399, 400, 401, 600, 698, 699])
    _, _, got = check_prefill(A, seqs, [n], 0, 63, L, rows)
    bad = np.isnan(O.bf16_to_f32(got)).any(axis=-1)
    pos = np.arange(L - n, L)
    for h, j in ((2, 100), (6, 1200), (1, 1499)):
        np.testing.assert_array_equal(bad[:, 8 * h], pos >= j)
    assert not bad[:, [0, 24, 32, 40, 56]].any()


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("longest", [1, 2, 3, 4, 5, 6, 12, 13])
def test_prefill_few_tokens(A, longest, window):
    """Drafts of up to `longest` tokens over caches of all lengths, their keys in shares."""
    rng = np.random.default_rng(longest)
    qlens = [longest, 1, 0, *rng.integers(1, longest + 1, 4).tolist()]
    prefix = [2500, 0, 70, 63, 64, 1100, 255]
    seqs = Seqs(500 + longest, [p + n for p, n in zip(prefix, qlens)])
    check_prefill(A, seqs, qlens, window, 501 + longest, bound=2500 + longest)


@pytest.mark.parametrize("window", [0, 128])
def test_prefill_long(A, window):
    """A long prompt at sampled rows: sharp scores, the row maximum anywhere."""
    seqs = Seqs(40, [2100])
    rows = np.array([0, 1, 31, 32, 63, 64, 65, 127, 500, 1023, 1024, 2000, 2098, 2099])
    check_prefill(A, seqs, [2100], window, 41, 2100, rows)
    check_prefill(A, seqs, [2100], window, 42, 2100, rows, scale=12.0)


@pytest.mark.parametrize("window", [0, 128])
def test_prefill_many_tiles(A, window):
    """A ragged batch whose query tiles are two rounds of the chip (the larger tiles)."""
    qlens, prefix = [512, 1, 64, 65, 130, 0, 257, 511], [0, 700, 3, 64, 1, 9, 300, 77]
    seqs = Seqs(45, [p + q for p, q in zip(prefix, qlens)])
    rows = np.array([0, 1, 3, 4, 31, 32, 63, 64, 100, 129, 200, 255, 256, 400, 510, 511])
    check_prefill(A, seqs, qlens, window, 46, 777, rows)


def test_prefill_creeping_maximum(A):
    """Scores that rise block by block, slowly and by large steps, and ones that fall: the
    running reference point of the softmax has to follow."""
    L, n = 1500, 24
    rng = np.random.default_rng(50)
    for step in (0.02, 0.4, 3.0, -0.4, -3.0):
        k = rng.standard_normal((L, HKV, D)) * 0.05
        k[:, :, 0] += step * (np.arange(L)[:, None] // 16 - (0 if step > 0 else L // 16))
        v = bf(rng.standard_normal((L, HKV, D)))
        seqs = Seqs(51, [L], k=[bf(k)], v=[v])
        q = rng.standard_normal((n, HQ, D)) * 0.1
        q[:, :, 0] = 8.0
        for bound in (0, L):
            got, _ = run_prefill(A, seqs, bf(q), [n], bf(np.zeros(HQ)), 0, bound)
            within(got, bf(q), seqs.kd[0], seqs.vd[0], np.arange(L - n, L), 0, bf(np.zeros(HQ)), U)


@pytest.mark.parametrize("window", [0, 40])
def test_prefill_bad_rows(A, window):
    """NaN in a new token's k, infinity in another's v: the rows before them, and those whose
    window has passed them, are not affected."""
    L, n = 260, 200
    seqs0 = Seqs(60, [L, 90])
    k, v = [x.copy() for x in seqs0.k], [x.copy() for x in seqs0.v]
    k[0][150, 2, 5], v[0][100, 6, 9] = NAN_ROW, 0xFF80
    seqs = Seqs(60, [L, 90], k=k, v=v)
    for bound in (0, L):
        _, _, got = check_prefill(A, seqs, [n, 90], window, 61, bound)
        bad = np.isnan(O.bf16_to_f32(got[:n])).any(axis=-1)
        pos = np.arange(L - n, L)
        for h, j in ((2, 150), (6, 100)):
            seen = (pos >= j) & ((pos < j + window) | (window == 0))
            np.testing.assert_array_equal(bad[:, 8 * h], seen)
        assert not bad[:, [0, 8, 24, 40, 56]].any()


def test_prefill_more_queries_than_keys(A):
    """q rows at positions before the sequence's first token see no key: 0."""
    seqs = Seqs(70, [10, 0])
    rng = np.random.default_rng(71)
    q, sinks = bf(rng.standard_normal((40, HQ, D))), bf(rng.standard_normal(HQ))
    got, _ = run_prefill(A, seqs, q, [30, 10], sinks, 0, 0)
    assert not got[:20].any() and not got[30:].any()
    within(got[20:30], q[20:30], seqs.kd[0], seqs.vd[0], np.arange(10), 0, sinks, U)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 20])
def test_window_of_any_size(A, window):
    """As no window, also where a chunk begins before its sequence's first token."""
    seqs = Seqs(75, [10, 300])
    rng = np.random.default_rng(76)
    q, sinks = bf(rng.standard_normal((40, HQ, D))), bf(rng.standard_normal(HQ))
    none, _ = run_prefill(A, seqs, q, [30, 10], sinks, 0, 0)
    got, _ = run_prefill(A, seqs, q, [30, 10], sinks, window, 0)
    within(got[20:30], q[20:30], seqs.kd[0], seqs.vd[0], np.arange(10), 0, sinks, U)
    within(got[30:], q[30:], seqs.kd[1], seqs.vd[1], np.arange(290, 300), 0, sinks, U)
    assert not got[:20].any() and not none[:20].any()
    np.testing.assert_array_equal(run_decode(A, seqs, q[:2], sinks, window, 300),
                                  run_decode(A, seqs, q[:2], sinks, 0, 300))


@pytest.mark.parametrize("n", [5, 40])
def test_prefill_rows_behind(A, n):
    """A few tokens at the head of a long buffer, their keys shared out over workgroups."""
    check_prefill(A, Seqs(77, [2100, 900]), [n, 3], 0, 78, bound=2100, extra=4000)


def test_pages_past_32_bits(A):
    """Pages beyond the fourth GiB of a layer's cache, by every entry point."""
    pool = (4 << 30) // AO.FP8_PAGE_BYTES + 1200
    L = 300
    small = Seqs(80, [L])
    ids = pool - 1 - np.arange(19) * 3
    cache = torch.empty((pool, AO.FP8_PAGE_BYTES), dtype=torch.uint8, device="cuda")
    t = np.arange(L)
    slots = i32_dev(ids[t // PAGE] * PAGE + t % PAGE)
    src = np.zeros((19, 2, HKV, PAGE, D), dtype=np.uint16)
    src[t // PAGE, 0, :, t % PAGE], src[t // PAGE, 1, :, t % PAGE] = small.k[0], small.v[0]
    A.kv_quantize_fp8(bf16_dev(src), i32_dev(t), cache, slots)
    k, v = A.kv_read_fp8(cache, slots)
    np.testing.assert_array_equal(k.double().cpu().numpy(), small.kd[0])
    np.testing.assert_array_equal(v.double().cpu().numpy(), small.vd[0])
    small.cache, small.page_indices = cache, i32_dev(ids)
    check_decode(A, small, 0, 81)
    check_prefill(A, small, [50], 0, 82, L)


def test_bad_page_tables_read_other_pages(A):
    """Ids outside the pool and a list that is too short: other keys, no fault, and the other
    sequences as they are."""
    seqs = Seqs(90, [200, 300])
    rng = np.random.default_rng(91)
    q, sinks = bf(rng.standard_normal((2, HQ, D))), bf(rng.standard_normal(HQ))
    good = run_decode(A, seqs, q, sinks, 0)
    seqs.page_indices[3], seqs.page_indices[5] = 1 << 30, -7
    np.testing.assert_array_equal(run_decode(A, seqs, q, sinks, 0)[1], good[1])
    seqs.page_indptr[0] = seqs.page_indptr[1]          # no pages at all
    np.testing.assert_array_equal(run_decode(A, seqs, q, sinks, 0)[1], good[1])
    run_prefill(A, seqs, bf(rng.standard_normal((40, HQ, D))), [20, 20], sinks, 0, 300)


def test_streams_and_graph(A):
    """The same step eager, on another stream, and captured: append, both attentions and the
    read, replayed over changed inputs with eager work in between."""
    rng = np.random.default_rng(95)
    lengths, n = [700, 90], 6
    seqs = Seqs(96, lengths)
    sinks = bf16_dev(bf(rng.standard_normal(HQ)))
    src = bf16_dev(bf(rng.standard_normal((1, 2, HKV, PAGE, D))))
    new = i32_dev(np.arange(2))
    ends = seqs.page_indices.cpu().numpy()
    last = [ends[-(-700 // PAGE) - 1] * PAGE + 699 % PAGE, ends[-1] * PAGE + 89 % PAGE]
    slots = i32_dev(np.array(last))
    q = bf16_dev(bf(rng.standard_normal((2, HQ, D))))
    qc = bf16_dev(bf(rng.standard_normal((2 * n, HQ, D))))
    qi = i32_dev(np.array([0, n, 2 * n]))
    ws = A.decode_fp8_workspace(2, 700)

    def step():
        out, oc = torch.empty_like(q), torch.empty_like(qc)
        A.kv_quantize_fp8(src, new, seqs.cache, slots)
        A.decode_fp8(q, *seqs.tables(), 700, 0, SCALE, sinks, out, ws)
        A.prefill_fp8(qc, qi, n, *seqs.tables(), 0, SCALE, sinks, oc, 700)
        return (out, oc, *A.kv_read_fp8(seqs.cache, slots))

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        src.copy_(bf16_dev(bf(rng.standard_normal(tuple(src.shape)))))
        q.mul_(-1.0)
        want = [t.clone() for t in step()]
        seqs.cache[:, 0] ^= 0                          # eager work
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), i
    assert int(ws[:2 << 20].count_nonzero()) == 0


# -- through the model -----------------------------------------------------------------------

def _cache(batch, tokens, pages, layers=2):
    from model.kv_cache import PagedKVCache
    return PagedKVCache(num_layers=layers, num_pages=pages, max_batch=batch, max_tokens=tokens,
                        dtype=torch.float8_e4m3fn)


def _close_rows(rows, want):
    """Cached rows (bf16 bits) against the values quantised: within a half step (2^-4 of the
    value, or 2^-17 of the row's largest) and what the projection's own roundings may move (two
    bf16 ulps of the row's largest, from the rotation's sum)."""
    got = O.bf16_to_f32(rows).astype(np.float64)
    w = O.bf16_to_f32(want).astype(np.float64)
    top = np.abs(w).max(axis=-1, keepdims=True)
    assert (np.abs(got - w) <= np.abs(w) * 2.0 ** -4 + top * (2.0 ** -17 + 2 * U)).all()


@pytest.mark.parametrize("layer_idx", [0, 1])  # sliding window 128, full attention
def test_attention_block(A, layer_idx):
    """AttentionBlock over an 8-bit cache: a prompt of 150 (library QKV, the RoPE append), single
    tokens, a chunk of 5 and one of 60 (fused QKV, staged rows), each against the oracle's
    block over the rows that the cache holds."""
    from test_gpu_attention import _block, close
    p = AO.make_attn_params(51 + layer_idx)
    blk = _block(A, p, layer_idx)
    cache = _cache(2, 256, 64)
    cache.add_sequence(0)
    cache.enable_sliding_window(0, 128)
    window = 128 if layer_idx == 0 else 0
    x = O.make_input(52, 220)
    a = 0
    sinks = O.bf16_to_f32(p.sinks).astype(np.float64)
    for n in (150, 1, 1, 5, 60, 1):
        b = a + n
        cache.begin_forward([0], [n])
        got = host_bf16(blk(bf16_dev(x[a:b]).view(1, n, 2880), cache).view(n, 2880))
        cache.end_forward()
        q, k, v = AO.split_qkv(AO.linear(O.rms_norm(x[a:b], p.norm_w, 1e-5), p.qkv_w, p.qkv_b))
        pos = np.arange(a, b)
        kc, vc = (host_bf16(t) for t in cache.read(0, layer_idx))
        _close_rows(kc[a:], AO.rope(k, pos))
        _close_rows(vc[a:], v)
        o, _, _ = AO.attention_sink(O.bf16_to_f32(AO.rope(q, pos)).astype(np.float64),
                                    O.bf16_to_f32(kc).astype(np.float64),
                                    O.bf16_to_f32(vc).astype(np.float64), pos, window, sinks, SCALE)
        y = AO.linear(bf(o).reshape(n, HQ * D), p.out_w, p.out_b)
        close(got, O.f32_to_bf16(O.bf16_to_f32(x[a:b]) + O.bf16_to_f32(y)))
        a = b


@pytest.mark.parametrize("n", [2, 16, 17, 64, 65])
def test_attention_block_decode_batch(A, n):
    """Decode batches on both sides of the lines between the projections."""
    from test_gpu_attention import _block, close
    p = AO.make_attn_params(57)
    blk = _block(A, p, 1)
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 70, n)
    cache = _cache(n, 80 * n, 6 * n)
    bf16 = __import__("model.kv_cache", fromlist=["PagedKVCache"]).PagedKVCache(
        2, 6 * n, n, 80 * n)
    bf16.data.copy_(bf16_dev(bf(rng.standard_normal(tuple(bf16.data.shape)))))
    for i in range(n):
        bf16.add_sequence(i)
        bf16.enable_sliding_window(i, 128)
        if lengths[i]:
            bf16.begin_forward([i], [lengths[i]])
        cache.quantize_from(i, bf16, i)
        if lengths[i]:                                 # moved whole, in both layers
            for layer in (0, 1):
                for got, rows, is_v in zip(cache.read(i, layer), bf16.read(i, layer),
                                           (False, True)):
                    np.testing.assert_array_equal(got.double().cpu().numpy(),
                                                  values(host_bf16(rows), is_v))
    x = O.make_input(58, n)
    cache.begin_forward(list(range(n)), [1] * n)
    got = host_bf16(blk(bf16_dev(x).view(n, 1, 2880), cache).view(n, 2880))
    q, _, _ = AO.split_qkv(AO.linear(O.rms_norm(x, p.norm_w, 1e-5), p.qkv_w, p.qkv_b))
    q = O.bf16_to_f32(AO.rope(q, lengths)).astype(np.float64)
    o = []
    for i in range(n):
        kc, vc = (O.bf16_to_f32(host_bf16(t)).astype(np.float64) for t in cache.read(i, 1))
        o.append(AO.attention_sink(q[i:i + 1], kc, vc, lengths[i:i + 1], 0,
                                   O.bf16_to_f32(p.sinks).astype(np.float64), SCALE)[0])
    y = AO.linear(bf(np.concatenate(o)).reshape(n, HQ * D), p.out_w, p.out_b)
    close(got, O.f32_to_bf16(O.bf16_to_f32(x) + O.bf16_to_f32(y)))


def test_engine_graph_equals_eager(A):
    """Engine with an 8-bit cache: a prompt, eager steps, the same steps replayed from the
    captured graph, then an extend after a rollback and again the graph."""
    from engine import Engine
    from model.config import GPTOssConfig
    cfg = GPTOssConfig(num_hidden_layers=2, num_experts=32, vocab_size=4096,
                       context_window_size=1024, prefill_chunk_size=512)
    torch.manual_seed(5)
    eng = Engine(config=cfg, max_total_seq_len=1024, kv_dtype=torch.float8_e4m3fn)
    for name, w in eng.model.named_parameters():
        if w.dtype == torch.uint8:
            w.copy_(torch.randint(*((114, 118) if "scales" in name else (0, 256)), w.shape,
                                  dtype=torch.uint8, device="cuda"))
        elif "norm" not in name:
            w.copy_(torch.randn(w.shape, device="cuda") * (1.0 if "embedding" in name else 0.02))
    assert eng.paged_kv_cache.fp8
    seq = eng.begin_sequence()
    prompt = np.random.default_rng(6).integers(0, 4096, 140).astype(np.int32)
    tok0 = eng.sample_device(eng.prefill(prompt, seq)).clone()
    eng._token.copy_(tok0)

    def eager(steps):
        out = []
        for _ in range(steps):
            lg = eng.decode(eng._token, seq)
            assert torch.isfinite(lg).all()
            out.append((lg.view(-1).clone(), int(eng.sample_device(lg).item())))
        return out

    def graphed(steps):
        out = []
        for _ in range(steps):
            t = eng.decode_sample(seq)
            out.append((eng.graph_logits.view(-1).clone(), int(t.item())))
        return out

    want = eager(5)
    eng.popn(seq, 5)
    eng._token.copy_(tok0)
    eng.capture_decode(seq)
    for (a, s), (b, t) in zip(want, graphed(5)):
        assert torch.equal(a, b) and s == t
    eng.popn(seq, 3)
    eng.sample_device(eng.extend(prompt[:100], seq))
    tok1 = eng._token.clone()
    want = eager(3)
    eng.popn(seq, 3)
    eng._token.copy_(tok1)
    for (a, s), (b, t) in zip(want, graphed(3)):
        assert torch.equal(a, b) and s == t
    assert eng.get_kv_total_seq_len() == 140 + 2 + 100 + 3


def test_tensors_of_any_class(A):
    """Arguments of a caller's own class of tensor, as the bf16 cache's wrappers take them."""
    class Named(torch.Tensor):
        pass

    rng = np.random.default_rng(130)
    seqs = Seqs(131, [40])
    q, sinks = bf16_dev(bf(rng.standard_normal((1, HQ, D)))), bf16_dev(bf(rng.standard_normal(HQ)))
    ws, out = A.decode_fp8_workspace(1, 40), torch.empty_like(q)
    want = A.decode_fp8(q, *seqs.tables(), 40, 0, SCALE, sinks, out, ws).clone()
    args = [t.as_subclass(Named) for t in (q, *seqs.tables())]
    out.zero_()
    A.decode_fp8(*args, 40, 0, SCALE, sinks.as_subclass(Named), out.as_subclass(Named), ws)
    assert torch.equal(out, want)
    slots = i32_dev(np.arange(5))
    for a, b in zip(A.kv_read_fp8(args[1], slots.as_subclass(Named)),
                    A.kv_read_fp8(seqs.cache, slots)):
        np.testing.assert_array_equal(host_bf16(a), host_bf16(b))


@pytest.mark.parametrize("longest,batch,window,threads,tokens", [
    (600, 60000, 0, 1024, 64), (600, 60000, 128, 512, 32), (7, 600000, 0, 256, 2)])
def test_prefill_more_tiles_than_a_launch(A, longest, batch, window, threads, tokens):
    """Tiles of the longest sequence for so many sequences (nearly all of them empty here) that
    they go in several launches: sequences at the ends and on both sides of the border."""
    border = ((1 << 32) - 1) // (threads * HKV * -(-longest // tokens))
    assert border + 1 < batch
    at = np.array([0, border - 1, border, border + 1, batch - 1])
    qlens = np.minimum([70, 5, 33, 64, 1], longest)
    lengths = qlens + [0, 40, 300, 0, 200]
    small = Seqs(140, lengths.tolist())
    q_len, kv_len, pages = (np.zeros(batch, dtype=np.int32) for _ in range(3))
    q_len[at], kv_len[at], pages[at] = qlens, lengths, -(-lengths // PAGE)
    q_indptr, page_indptr = (np.concatenate([[0], np.cumsum(x)]) for x in (q_len, pages))
    rng = np.random.default_rng(141)
    n = int(q_indptr[-1])
    q, sinks = bf(rng.standard_normal((n, HQ, D)) * 2.0), bf(rng.standard_normal(HQ))
    out = torch.full((n + 2, HQ, D), 7.0, dtype=torch.bfloat16, device="cuda")
    qd = torch.zeros((n + 2, HQ, D), dtype=torch.bfloat16, device="cuda")
    qd[:n] = bf16_dev(q)
    A.prefill_fp8(qd, i32_dev(q_indptr), longest, small.cache, i32_dev(page_indptr),
                  small.page_indices, i32_dev(kv_len), window, SCALE, bf16_dev(sinks), out,
                  int(lengths.max()))
    got = host_bf16(out)
    assert (got[n:] == 0x40E0).all()
    for i, b in enumerate(at):
        rows = slice(q_indptr[b], q_indptr[b + 1])
        within(got[rows], q[rows], small.kd[i], small.vd[i],
               np.arange(lengths[i] - qlens[i], lengths[i]), window, sinks, U)


@pytest.mark.parametrize("longest", [1, 2, 3, 4, 5, 8, 12, 16, 20])
def test_prefill_few_tokens_as_exact_as_decode(A, longest):
    """Drafts of up to `longest` tokens keep their probabilities to decode's two bf16 pieces
    (2^-16), alone and in shares: flat scores over few keys, whose roundings do not average out,
    and sharp ones."""
    qlens = [longest, 1, longest, max(1, longest - 1), longest]
    lengths = [n + p for n, p in zip(qlens, [0, 2, 5, 40, 1300])]
    seqs = Seqs(600 + longest, lengths)
    indptr = np.concatenate([[0], np.cumsum(qlens)])
    rng = np.random.default_rng(601)
    for scale, bound in ((0.25, 0), (0.25, max(lengths)), (4.0, max(lengths))):
        q = bf(rng.standard_normal((sum(qlens), HQ, D)) * scale)
        sinks = bf(rng.standard_normal(HQ))
        got, _ = run_prefill(A, seqs, q, qlens, sinks, 0, bound)
        for b, (L, n) in enumerate(zip(lengths, qlens)):
            rows = slice(indptr[b], indptr[b + 1])
            within(got[rows], q[rows], seqs.kd[b], seqs.vd[b], np.arange(L - n, L), 0, sinks,
                   2.0 ** -16)


class LongSeqs(Seqs):
    """Sequences of any length on a pool of `pool` pages of random rows, each page of a sequence
    any page of the pool: a page read in another's place shows."""

    def __init__(self, seed, lengths, pool=300):
        super().__init__(seed, [pool * PAGE])
        rng = np.random.default_rng(seed + 1)
        order = self.page_indices.cpu().numpy()        # order[i]: where tokens 16 i .. lie
        lists = [rng.integers(0, pool, -(-L // PAGE)) for L in lengths]
        rows = [(p[:, None] * PAGE + np.arange(PAGE)).ravel()[:L] for p, L in zip(lists, lengths)]
        self.kd, self.vd = [self.kd[0][r] for r in rows], [self.vd[0][r] for r in rows]
        self.lengths = lengths
        self.page_indptr = i32_dev(np.concatenate([[0], np.cumsum([len(p) for p in lists])]))
        self.page_indices = i32_dev(order[np.concatenate(lists)])
        self.kv_len = i32_dev(np.array(lengths))


@pytest.mark.parametrize("lengths", [[33000], [40000], [70000], [140000, 90]])
def test_decode_long(A, lengths):
    """Against the oracle: one sequence in 33 to 64 splits, and splits of more than 64 blocks,
    whose waves fetch a second set of page ids (two sequences: at most 32 splits)."""
    seqs = LongSeqs(700, lengths)
    check_decode(A, seqs, 0, 701)
    check_decode(A, seqs, 0, 702, scale=4.0)


def parts(A, rows, batch, longest, most_kv, window):
    """Rows of the parts that a chunk call's shares leave for the merge: shares x the tokens of
    its tiles."""
    size = A._lib.attn_prefill_fp8_workspace_bytes(rows, batch, longest, most_kv, window)
    assert size % (HQ * (D + 2) * 4) == 0
    return size // (HQ * (D + 2) * 4)


@pytest.mark.parametrize("qlens,prefix,bound,window", [
    ([2], [9000], 0, 0), ([4], [9000], 0, 0), ([12, 1], [9000, 70], 0, 0),   # tiles of 2 and 4
    ([40], [9000], 0, 0), ([40, 3], [9000, 100], 0, 8000),                   # of 32, whole
    ([30] + [1] * 31, [9000] + [50] * 31, 9030, 0),                          # two halves
    ([4200], [0], 4200, 0), ([40] + [33] * 63, [9000] + [5] * 63, 9040, 0)])  # of 64
def test_prefill_more_blocks_than_page_ids_at_hand(A, qlens, prefix, bound, window):
    """More than 64 blocks of keys for one workgroup, or half of one: its waves fetch a second
    and third set of page ids."""
    lengths = [p + q for p, q in zip(prefix, qlens)]
    assert parts(A, sum(qlens), len(qlens), max(qlens), bound, window) == 0      # one share
    rows = np.array([0, 1, 2, 3, 11, 29, 31, 32, 39, 2000, 4095, 4096, 4097, 4170, 4199])
    seqs = LongSeqs(710, lengths)
    check_prefill(A, seqs, qlens, window, 711, bound, rows)
    check_prefill(A, seqs, qlens, window, 712, bound, rows, scale=4.0)


@pytest.mark.parametrize("qlen,prefix,window,shares", [
    (550, 2500, 0, 3), (380, 3000, 0, 5), (550, 6000, 4000, 3), (300, 6000, 2000, 3)])
def test_prefill_shared_keys_in_odd_shares(A, qlen, prefix, window, shares):
    """Tiles of 32 tokens in an odd number of shares, each a workgroup's (the first three: as many
    as fit the chip, 512 workgroups) or two halves' (the last), with and without a window."""
    L, tiles = qlen + prefix, -(-qlen // 32)
    assert parts(A, qlen, 1, qlen, L, window) == shares * 32 * tiles
    assert shares == 512 // (8 * tiles) // (2 if qlen == 300 else 1)
    rows = np.array([0, 1, 31, 32, 33, 160, qlen // 2, qlen - 33, qlen - 32, qlen - 31, qlen - 1])
    seqs = LongSeqs(720, [L])
    for scale in (2.0, 8.0):
        check_prefill(A, seqs, [qlen], window, 721, L, rows, scale=scale)


def test_prefill_larger_tiles_sharp_scores(A):
    """Tiles of 64 tokens (a batch of two rounds of the chip): scores of +-100 and more, and ones
    that rise or fall slowly and by large steps along the keys."""
    qlens, prefix = [512, 64, 1, 130, 3, 33, 400, 100], [100, 0, 700, 9, 64, 31, 300, 77]
    lengths = [p + q for p, q in zip(prefix, qlens)]
    rows = np.array([0, 1, 3, 31, 32, 63, 64, 129, 255, 256, 399, 511])
    check_prefill(A, Seqs(730, lengths), qlens, 0, 731, 700, rows, scale=12.0)
    rng = np.random.default_rng(732)
    for step in (0.02, 3.0, -3.0):
        k = []
        for L in lengths:
            x = rng.standard_normal((L, HKV, D)) * 0.05
            x[:, :, 0] += step * (np.arange(L)[:, None] // 16 - (0 if step > 0 else L // 16))
            k.append(bf(x))
        seqs = Seqs(733, lengths, k=k)
        q = rng.standard_normal((sum(qlens), HQ, D)) * 0.1
        q[:, :, 0] = 8.0
        q, sinks = bf(q), bf(np.zeros(HQ))
        got, indptr = run_prefill(A, seqs, q, qlens, sinks, 0, 700)
        for b, (L, n) in enumerate(zip(lengths, qlens)):
            pick = np.unique(np.clip(rows, 0, n - 1))
            at = indptr[b] + pick
            within(got[at], q[at], seqs.kd[b], seqs.vd[b], L - n + pick, 0, sinks, U)


def test_prefill_larger_tiles_bad_rows(A):
    """Tiles of 64 tokens: a NaN in k, infinities in v and k reach the queries that see them, in
    their kv head, and no others; what lies past the sequences' ends reaches none."""
    qlens, prefix = [512, 64, 1, 130, 3, 33, 400, 100], [100, 0, 700, 9, 64, 31, 300, 77]
    lengths = [p + q for p, q in zip(prefix, qlens)]
    seqs0 = Seqs(740, lengths)
    k, v = [x.copy() for x in seqs0.k], [x.copy() for x in seqs0.v]
    k[0][150, 2, 5], v[0][500, 6, 9], k[0][611, 1, 0] = NAN_ROW, 0xFF80, 0x7F80
    seqs = Seqs(740, lengths, k=k, v=v)
    rows = np.array([0, 49, 50, 51, 399, 400, 401, 510, 511])
    _, _, got = check_prefill(A, seqs, qlens, 0, 741, 700, rows)
    bad = np.isnan(O.bf16_to_f32(got)).any(axis=-1)
    pos = np.arange(100, 612)
    for h, j in ((2, 150), (6, 500), (1, 611)):
        np.testing.assert_array_equal(bad[:512, 8 * h:8 * h + 8],
                                      np.repeat((pos >= j)[:, None], 8, 1))
    assert not bad[512:].any() and not bad[:, [0, 24, 32, 40, 56]].any()


def test_captured_writes(A):
    """A step that appends, quantises, attends and reads, on another stream and captured: before
    each run the rows that it writes are replaced by others, so that only its own writes give the
    outputs and the cache that the eager step left."""
    from test_gpu_attention import _inv_freq_dev
    rng = np.random.default_rng(750)
    seqs = Seqs(751, [700, 90])
    cache, ids = seqs.cache, seqs.page_indices.cpu().numpy()
    ends = [int(x) for x in seqs.page_indptr[1:].cpu().numpy()]

    def slot(b, pos):
        return ids[(0 if b == 0 else ends[0]) + pos // PAGE] * PAGE + pos % PAGE

    appended = i32_dev(np.array([slot(0, 698), slot(0, 699), slot(1, 89)]))
    moved = i32_dev(np.array([slot(0, 690), slot(0, 691), slot(1, 80)]))
    both = torch.cat([appended, moved])

    def draw(*shape):
        return bf16_dev(bf(rng.standard_normal(shape)))

    qkv, bias, src = draw(3, (HQ + 2 * HKV) * D), draw((HQ + 2 * HKV) * D), draw(1, 2, HKV, PAGE, D)
    pos, three, six = (i32_dev(np.array(x)) for x in ([698, 699, 89], [0, 1, 2], range(6)))
    inv, conc = _inv_freq_dev()
    q, qc, sinks, n = draw(2, HQ, D), draw(8, HQ, D), draw(HQ), 4
    qi = i32_dev(np.array([0, n, 2 * n]))
    ws = A.decode_fp8_workspace(2, 700)

    def step():
        qn = torch.empty((3, HQ, D), dtype=torch.bfloat16, device="cuda")
        out, oc = torch.empty_like(q), torch.empty_like(qc)
        A.qkv_rope_append_fp8(qkv, bias, pos, appended, inv, conc, cache, qn)
        A.kv_quantize_fp8(src, three, cache, moved)
        A.decode_fp8(q, *seqs.tables(), 700, 0, SCALE, sinks, out, ws)
        A.prefill_fp8(qc, qi, n, *seqs.tables(), 0, SCALE, sinks, oc, 700)
        return (qn, out, oc, *A.kv_read_fp8(cache, both))

    def expect():
        """What the step gives and leaves; then other rows in the places that it writes."""
        want = [t.clone() for t in step()], cache.clone()
        A.kv_quantize_fp8(draw(1, 2, HKV, PAGE, D), six, cache, both)
        assert not torch.equal(cache, want[1])
        return want

    def same(got, want):
        for a, b in zip(got, want[0]):
            assert torch.equal(a, b)
        assert torch.equal(cache, want[1])

    want = expect()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        qkv.copy_(draw(*qkv.shape))
        src.copy_(draw(*src.shape))
        q.mul_(-1.0)
        want = expect()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(held, want)
    assert int(ws[:2 << 20].count_nonzero()) == 0
