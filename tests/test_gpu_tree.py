"""Trees of drafted tokens on the GPU: attention over both caches against the oracle, and the walk
and the moves after verification, bit for bit.

The bound of an output is that of the 8-bit cache's chunks (test_gpu_fp8_cache.py): with u = 2^-8
(half a bf16 step) and A = sum p |v| / (sum p + exp(sink)), |out - exact| <= u |exact| + (e + 2 d)
A.  d: the relative error of a probability from its score, 64 products summed in fp32, so at most
64 2^-24 of sum |q k| scale, doubled for the exponent's own arithmetic.  e: one rounding of the
probabilities to bf16 (u) and the fp32 sums and exponentials (2^-14, generous)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from gpu_util import bf16_dev, host_bf16, i32_dev, u8_dev  # noqa: E402

pytestmark = pytest.mark.gpu

D, HQ, HKV, PAGE = 64, 64, 8, 16
SCALE = 1.0 / math.sqrt(D)
U = 2.0 ** -8
BOTH = pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import attn_native
    return attn_native


def bf(x):
    return O.f32_to_bf16(np.asarray(x, dtype=np.float32))


def f64(bits):
    return O.bf16_to_f32(bits).astype(np.float64)


def random_tree(rng, m, depth=5):
    """Parents in any order that has them before their children."""
    level, parents = [0][:m], [-1][:m]
    for i in range(1, m):
        at = rng.choice([j for j in range(i) if level[j] < depth] or [0])
        parents.append(int(at))
        level.append(level[at] + 1)
    return parents


def tree_bits(parents):
    """[m, m] bool: node i sees node j; and the nodes' depths."""
    m = len(parents)
    see = np.zeros((m, m), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see, see.sum(axis=1) - 1


class Case:
    """Sequences of cached tokens and nodes on scattered pages; every place that no token owns holds
    a NaN.  see[b] [m, m] and pos[b] [m] may be any."""

    def __init__(self, seed, fp8, cached, nodes, see=None, pos=None, k=None, v=None, pool=None,
                 depth=5, spread=1.0, scale=2.0):
        rng = np.random.default_rng(seed)
        self.fp8, self.cached, self.nodes = fp8, cached, nodes
        lengths = [c + m for c, m in zip(cached, nodes)]
        if see is None:
            see, pos = zip(*(tree_bits(random_tree(rng, m, depth)) for m in nodes)) if nodes else ((), ())
            pos = [c + p for c, p in zip(cached, pos)]
        self.see, self.pos = list(see), list(pos)
        need = [-(-L // PAGE) for L in lengths]
        self.pool = pool or sum(need) + 3
        perm = rng.permutation(self.pool)
        gain = np.exp(0.5 * rng.standard_normal((HKV, D)))
        self.k = k or [bf(rng.standard_normal((L, HKV, D)) * gain) for L in lengths]
        self.v = v or [bf(rng.standard_normal((L, HKV, D))
                          * np.exp(spread * rng.standard_normal((L, 1, 1)))) for L in lengths]
        if fp8:
            cache = np.full((self.pool, AO.FP8_PAGE_BYTES), 0xFF, dtype=np.uint8)
        else:
            cache = np.full((self.pool, 2, HKV, PAGE, D), 0x7FC0, dtype=np.uint16)
        indptr, ids = [0], []
        for L, kr, vr, n in zip(lengths, self.k, self.v, need):
            mine = perm[len(ids):len(ids) + n]
            p = np.arange(L)
            slots = mine[p // PAGE] * PAGE + p % PAGE if L else p
            if fp8:
                AO.fp8_put(cache, slots, kr, vr)
            else:
                cache[slots // PAGE, 0, :, slots % PAGE] = kr
                cache[slots // PAGE, 1, :, slots % PAGE] = vr
            ids.extend(mine.tolist())
            indptr.append(len(ids))
        if fp8:
            self.kd = [AO.fp8_dequantize(*AO.fp8_quantize(x, False)) for x in self.k]
            self.vd = [AO.fp8_dequantize(*AO.fp8_quantize(x, True)) for x in self.v]
        else:
            self.kd, self.vd = [f64(x) for x in self.k], [f64(x) for x in self.v]
        self.cache = u8_dev(cache) if fp8 else bf16_dev(cache)
        self.page_indptr = i32_dev(np.array(indptr))
        self.page_indices = i32_dev(np.array(ids or [0]))
        self.kv_len = i32_dev(np.array(lengths))
        self.starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.lengths, self.rng = lengths, rng
        n = int(self.starts[-1])
        self.q = bf(rng.standard_normal((n, HQ, D)) * scale)
        self.sinks = bf(rng.standard_normal(HQ))

    def mask(self, words=None, junk=False):
        longest = max(self.nodes)
        words = words or -(-longest // 32)
        out = np.zeros((int(self.starts[-1]), 32 * words), dtype=bool)
        if junk:                                       # bits past q_len
            out[:] = self.rng.random(out.shape) < 0.5
        for b, m in enumerate(self.nodes):
            out[self.starts[b]:self.starts[b + 1], :m] = self.see[b]
        return i32_dev(np.packbits(out, axis=1, bitorder="little").view(np.int32))

    def run(self, A, window=0, bound=True, extra=2, words=None, junk=False, longest=None):
        n = int(self.starts[-1])
        out = torch.full((n + extra, HQ, D), 7.0, dtype=torch.bfloat16, device="cuda")
        q = torch.zeros_like(out)
        q[:n] = bf16_dev(self.q)
        mask = torch.cat([self.mask(words, junk),
                          torch.full((extra, words or -(-max(self.nodes) // 32)), -1,
                                     dtype=torch.int32, device="cuda")])
        pos = torch.cat([i32_dev(np.concatenate(self.pos)),
                         torch.zeros(extra, dtype=torch.int32, device="cuda")])
        fn = A.tree_fp8 if self.fp8 else A.tree
        fn(q, i32_dev(self.starts), longest or max(self.nodes), mask, pos, self.cache,
           self.page_indptr, self.page_indices, self.kv_len, window, SCALE, bf16_dev(self.sinks),
           out, max(self.lengths) if bound else 0)
        got = host_bf16(out)
        assert (got[n:] == 0x40E0).all()               # rows behind the last sequence stay (7.0)
        return got[:n]

    def seen(self, b, window):
        c, m = self.cached[b], self.nodes[b]
        pos = np.maximum(np.asarray(self.pos[b]), c)
        where = np.concatenate([np.arange(c), pos])
        seen = np.concatenate([np.ones((m, c), dtype=bool), self.see[b]], axis=1)
        return seen & (where[None, :] > pos[:, None] - window) if window else seen

    def check(self, got, window=0, rows=None):
        sinks = f64(self.sinks)
        for b, m in enumerate(self.nodes):
            pick = np.arange(m) if rows is None else np.unique(np.clip(rows, 0, m - 1))
            if not m:
                continue
            at = self.starts[b] + pick
            ref, mag, size = AO.attention_seen(f64(self.q[at]), self.kd[b], self.vd[b],
                                               self.seen(b, window)[pick], sinks, SCALE)
            tol = U * np.abs(ref) + (U + 2.0 ** -14 + 2 * 2.0 ** -17 * size[..., None]) * mag
            g = f64(got[at])
            bad = ~np.isfinite(ref)
            assert not np.isfinite(g[bad]).any()
            ok = bad | (np.abs(g - ref) <= tol)
            assert ok.all(), (b, np.argwhere(~ok)[:5], g[~ok][:5], ref[~ok][:5], tol[~ok][:5])


@BOTH
@pytest.mark.parametrize("window", [0, 1, 3, 100, 128])
def test_tree(A, fp8, window):
    """A ragged batch: sequences without cached tokens, without nodes, ends inside and at the ends of
    pages and blocks."""
    c = Case(1, fp8, [0, 1, 15, 16, 17, 63, 64, 130, 40, 700], [1, 5, 8, 2, 33, 64, 7, 12, 0, 20])
    for bound in (False, True):
        c.check(c.run(A, window, bound), window)


@BOTH
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 26, 32, 33, 63, 64, 65, 129])
def test_tree_sizes(A, fp8, m):
    """One tree of m nodes, its keys in one share and in several."""
    c = Case(m, fp8, [1030], [m], depth=9)
    rows = np.array([0, 1, 2, 3, 4, 7, 8, 15, 16, 31, 32, 33, 62, 63, 64, 100, 128])
    for bound in (False, True):
        c.check(c.run(A, 0, bound), 0, rows)


@BOTH
@pytest.mark.parametrize("b", [2, 9, 40, 70])
def test_tree_batches(A, fp8, b):
    rng = np.random.default_rng(b)
    c = Case(b, fp8, rng.integers(0, 400, b).tolist(), rng.integers(1, 14, b).tolist())
    c.check(c.run(A))
    c.check(c.run(A, 50), 50)


@BOTH
@pytest.mark.parametrize("cached,m", [(17000, 3), (9000, 26), (5000, 64)])
def test_tree_long(A, fp8, cached, m):
    c = Case(cached, fp8, [cached, 90], [m, 2])
    rows = np.array([0, 1, m // 2, m - 1])
    c.check(c.run(A), 0, rows)
    c.check(c.run(A, 4000), 4000, rows)


@BOTH
def test_any_mask(A, fp8):
    """Masks that are no tree's, rows that see no node, rows that see nothing at all; bits past the
    tree's end and a mask of more words than it needs; positions in any order."""
    rng = np.random.default_rng(3)
    cached, nodes = [0, 70, 0, 200], [40, 40, 7, 65]
    see = [rng.random((m, m)) < 0.3 for m in nodes]
    for s in see:
        s[1] = False
        s[:, 2] = False
    see[2][:] = False
    pos = [c + rng.integers(0, 30, m) for c, m in zip(cached, nodes)]
    pos[1][:5] = 0                                     # before the cached tokens' end
    c = Case(4, fp8, cached, nodes, see, pos)
    for window in (0, 4, 90):
        got = c.run(A, window, junk=True, words=5, longest=150)
        c.check(got, window)
        assert not got[1].any() and not got[80:87].any()


@BOTH
def test_hidden_rows(A, fp8):
    """NaN and infinities in k and v of nodes and cached tokens reach the rows that see them, in
    their kv head (of a bf16 cache in the dimensions of v that have them), and no others."""
    rng = np.random.default_rng(5)
    cached, nodes = [200, 33, 0], [30, 40, 5]
    see = [np.eye(m, dtype=bool) for m in nodes]       # every node on its own
    for s in see:
        s[:, 0] = True
    pos = [c + np.minimum(np.arange(m), 1) for c, m in zip(cached, nodes)]
    k = [bf(rng.standard_normal((c + m, HKV, D))) for c, m in zip(cached, nodes)]
    v = [bf(rng.standard_normal((c + m, HKV, D))) for c, m in zip(cached, nodes)]
    k[0][210, 1, 3], v[0][212, 2, 5], v[0][215, 2, 6] = 0x7FC0, 0x7F80, 0x7FC1
    k[1][40, 0, 0], v[1][70, 7, 63], v[2][3, 4, 4] = 0xFF80, 0xFF80, 0x7FFF
    v[0][50, 5, 9] = 0x7FC0                            # in a window of 160 of the first, or not
    c = Case(6, fp8, cached, nodes, see, pos, k=k, v=v)
    for window in (160, 100):
        got = c.run(A, window)
        c.check(got, window)
        bad = ~np.isfinite(f64(got)).all(axis=-1).reshape(-1, HKV, 8)
        want = np.zeros((75, HKV), dtype=bool)
        want[10, 1] = want[12, 2] = want[15, 2] = want[30 + 7, 0] = want[30 + 37, 7] = True
        want[70 + 3, 4] = True
        want[:30, 5] = window == 160
        want = np.repeat(want[..., None], 8, -1)
        if not fp8:    # a score of -inf has the probability exp(-inf) = 0: only +inf shows
            want[30 + 7, 0] = f64(c.q[30 + 7, :8, 0]) < 0
        np.testing.assert_array_equal(bad, want)


@BOTH
def test_sharp_scores(A, fp8):
    """Scores to +-100 and more, and ones that rise or fall along the keys."""
    c = Case(7, fp8, [900, 70, 2000], [5, 17, 33], spread=6.0, scale=20.0)
    c.check(c.run(A))
    rng = np.random.default_rng(8)
    for step in (0.02, 3.0, -3.0):
        cached, nodes = [600, 1500], [9, 40]
        k = []
        for L in (609, 1540):
            x = rng.standard_normal((L, HKV, D)) * 0.05
            x[:, :, 0] += step * (np.arange(L)[:, None] // 16 - (0 if step > 0 else L // 16))
            k.append(bf(x))
        c = Case(9, fp8, cached, nodes, k=k)
        q = rng.standard_normal(c.q.shape) * 0.1
        q[:, :, 0] = 8.0
        c.q = bf(q)
        c.check(c.run(A))


@BOTH
def test_sinks(A, fp8):
    """Sinks that take nothing, everything, or more than the keys; a node that sees nothing."""
    see, pos = tree_bits([-1, 0, 0, 1])
    none = np.zeros((2, 2), dtype=bool)
    c = Case(10, fp8, [300, 0], [4, 2], [see, none], [300 + pos, np.zeros(2, dtype=int)])
    c.sinks = bf(np.resize([-np.inf, np.inf, 40.0, -40.0, 3e38, -3e38], HQ))
    got = f64(c.run(A))
    with np.errstate(all="ignore"):
        ref, mag, size = AO.attention_seen(f64(c.q[:4]), c.kd[0], c.vd[0], c.seen(0, 0),
                                           np.clip(f64(c.sinks), -1e30, 1e30), SCALE)
    tol = U * np.abs(ref) + (U + 2.0 ** -14 + 2 * 2.0 ** -17 * size[..., None]) * mag
    assert (np.abs(got[:4] - ref) <= tol).all()
    assert not got[4:].any()


@BOTH
def test_pages_past_32_bits(A, fp8):
    """A sequence on the last pages of a pool of more than 4 GB (and 2^31 elements)."""
    pool = (1 << 32) // (AO.FP8_PAGE_BYTES if fp8 else 32768) + 4000
    c = Case(11, fp8, [100], [12])
    big = torch.zeros((pool, *c.cache.shape[1:]), dtype=c.cache.dtype, device="cuda")
    n = c.cache.shape[0]
    big[pool - n:] = c.cache
    c.cache, c.page_indices = big, c.page_indices + (pool - n)
    c.check(c.run(A))


@BOTH
def test_bad_page_tables_read_other_pages(A, fp8):
    """Ids outside the pool, lists that are too short or empty: other keys, no fault, and the other
    sequences as they should be."""
    c = Case(12, fp8, [200, 150, 90], [6, 20, 3])
    good = c.run(A)
    ids = c.page_indices.clone()
    first = int(c.page_indptr[1])
    ids[:first] = torch.tensor([-5, 1 << 30, c.pool, -(1 << 31)], dtype=torch.int32,
                               device="cuda").repeat(-(-first // 4))[:first]
    c.page_indices = ids
    np.testing.assert_array_equal(c.run(A)[6:], good[6:])
    c.page_indptr = i32_dev(np.array([0, 0, int(c.page_indptr[1]) * 0 + 3, int(c.page_indptr[2])]))
    assert c.run(A).shape == good.shape


def test_streams_and_graph(A):
    """On another stream, captured, and replayed with other inputs between: the eager results; two
    captured calls whose replays follow one another in either order."""
    for fp8 in (False, True):
        small, large = Case(13, fp8, [300, 40], [5, 3]), Case(14, fp8, [4000], [40])
        calls = []
        for c in (small, large):
            n = int(c.starts[-1])
            fn = A.tree_fp8 if fp8 else A.tree
            q, out = bf16_dev(c.q), torch.empty((n, HQ, D), dtype=torch.bfloat16, device="cuda")
            args = (i32_dev(c.starts), max(c.nodes), c.mask(), i32_dev(np.concatenate(c.pos)),
                    c.cache, c.page_indptr, c.page_indices, c.kv_len, 0, SCALE, bf16_dev(c.sinks))
            calls.append((q, out, lambda f=fn, q=q, a=args, o=out, c=c: f(q, *a, o, max(c.lengths))))
        side = torch.cuda.Stream()
        graphs = []
        for q, out, call in calls:
            want = call().clone()
            out.zero_()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call()
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(out, want)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
            graphs.append(graph)
        for order in ((0, 1), (1, 0), (0, 0), (1, 1)):
            for q, out, _ in calls:
                q.mul_(-0.5).add_(0.25)
            want = [call().clone() for _, _, call in calls]
            for _, out, _ in calls:
                out.zero_()
            torch.cuda.synchronize()
            for i in order:
                graphs[i].replay()
            torch.cuda.synchronize()
            for i in set(order):
                assert torch.equal(calls[i][1], want[i])


# -- the walk and the moves ------------------------------------------------------------------

def layers_of(rng, fp8, layers, pool):
    """Random bytes: a move takes whatever is there."""
    shape = (layers, pool, AO.FP8_PAGE_BYTES) if fp8 else (layers, pool, 2, HKV, PAGE, D)
    return rng.integers(0, 256 if fp8 else 65536, shape, dtype=np.uint8 if fp8 else np.uint16)


def move_row(cache, fp8, src, dst):
    """Slot src to slot dst in every layer."""
    (sp, st), (dp, dt) = divmod(int(src), PAGE), divmod(int(dst), PAGE)
    if not fp8:
        cache[:, dp, :, :, dt] = cache[:, sp, :, :, st].copy()
        return
    d = np.arange(D)
    for h in range(HKV):
        at = h * 1024
        k = [at + t * D + d for t in (st, dt)]
        v = [AO.FP8_V + at + t // 4 * 256 + d % 16 * 16 + d // 16 * 4 + t % 4 for t in (st, dt)]
        s = [AO.FP8_SCALES + h * 32 + np.array([t, 16 + t]) for t in (st, dt)]
        for a, b in (k, v, s):
            cache[:, dp, b] = cache[:, sp, a].copy()


def commit_case(A, seed, fp8, cached, trees, layers=2, agree=0.9, tokens=30, longest=None, tail=3,
                last=False):
    """Trees with tokens of a small vocabulary (siblings of the same token among them) and a model
    that agrees with some child (or the last) most of the time."""
    rng = np.random.default_rng(seed)
    token = [rng.integers(0, tokens, len(t)) for t in trees]
    chosen = []
    for t, tk in zip(trees, token):
        kids = [[j for j in range(len(t)) if t[j] == i] for i in range(len(t))]
        chosen.append([tk[k[-1] if last else rng.choice(k)] if k and rng.random() < agree
                       else int(rng.integers(0, tokens)) for k in kids])
    lengths = [c + len(t) for c, t in zip(cached, trees)]
    need = [-(-L // PAGE) for L in lengths]
    pool = sum(need) + 2
    ids = rng.permutation(pool)[:sum(need)]
    indptr = np.concatenate([[0], np.cumsum(need)])
    starts = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
    cache = layers_of(rng, fp8, layers, pool)
    dev = u8_dev(cache) if fp8 else bf16_dev(cache)
    pad = np.zeros(tail, dtype=np.int32)
    flat = [i32_dev(np.concatenate([*x, pad])) for x in (token, trees, chosen)]
    path, count, after = A.tree_commit(
        dev, i32_dev(indptr), i32_dev(ids if len(ids) else np.zeros(1)), i32_dev(np.array(lengths)),
        i32_dev(starts), longest or max(len(t) for t in trees), *flat)
    want_path = np.full(int(starts[-1]) + tail, -1)
    for b, t in enumerate(trees):
        way = AO.tree_walk(token[b], t, chosen[b])
        want_path[starts[b]:starts[b] + len(way)] = way
        assert int(count[b]) == len(way)
        assert int(after[b]) == (chosen[b][way[-1]] if way else -1)
        mine = ids[indptr[b]:indptr[b + 1]]
        for i, node in enumerate(way):
            s, d = cached[b] + node, cached[b] + i
            if s != d:
                move_row(cache, fp8, mine[s // PAGE] * PAGE + s % PAGE,
                         mine[d // PAGE] * PAGE + d % PAGE)
    np.testing.assert_array_equal(path.cpu().numpy(), want_path)
    got = dev.cpu().numpy() if fp8 else host_bf16(dev)
    np.testing.assert_array_equal(got, cache)
    return [int(x) for x in count]


@BOTH
@pytest.mark.parametrize("seed", range(4))
def test_commit(A, fp8, seed):
    """Ragged trees in depth order and in any order, moves that overlap, pages of all kinds."""
    rng = np.random.default_rng(40 + seed)
    nodes = [1, 2, 5, 8, 26, 64, 70, 3, 0, 17]
    trees = [random_tree(rng, m, depth=12) if m else [] for m in nodes]
    got = commit_case(A, 50 + seed, fp8, rng.integers(0, 70, len(nodes)).tolist(), trees, layers=3)
    assert max(got) > 2


@BOTH
def test_commit_chains_and_combs(A, fp8):
    """A chain that is accepted whole (nothing moves), a path whose every node moves over places
    that later nodes of it leave, siblings of one token, and the largest tree."""
    chain = [-1] + list(range(39))
    comb = [-1] + [x for i in range(0, 40, 2) for x in (i, i)]     # a leaf and a stem node in turn
    same = [-1, 0, 0, 0, 1, 2, 3]
    large = [-1] + [max(0, i - 2) for i in range(1, 1024)]
    got = commit_case(A, 60, fp8, [7, 3, 0, 30], [chain, comb, same, large], agree=1.0, tokens=100000,
                      last=True)
    assert got[0] == 40 and got[1] > 10 and got[3] > 300
    commit_case(A, 61, fp8, [7, 3, 0, 30], [chain, comb, same, large], agree=1.0, tokens=1)
    commit_case(A, 62, fp8, [20], [same], agree=0.0, tokens=100000, layers=36, longest=1024)


@BOTH
def test_commit_many(A, fp8):
    rng = np.random.default_rng(63)
    trees = [random_tree(rng, int(m), 7) for m in rng.integers(1, 27, 70)]
    commit_case(A, 64, fp8, rng.integers(0, 50, 70).tolist(), trees, layers=5, tail=0)


def test_commit_graph(A):
    """Captured with its outputs: replayed on rows and choices that change between."""
    for fp8 in (False, True):
        rng = np.random.default_rng(65)
        trees = [random_tree(rng, m, 6) for m in (9, 26)]
        n = 35
        parents, tokens = i32_dev(np.concatenate(trees)), i32_dev(rng.integers(0, 3, n))
        chosen = i32_dev(rng.integers(0, 3, n))
        shape = (4, 5, AO.FP8_PAGE_BYTES) if fp8 else (4, 5, 2, HKV, PAGE, D)
        cache = torch.randint(0, 250, shape, device="cuda").to(torch.uint8 if fp8
                                                               else torch.bfloat16)
        tables = (i32_dev(np.array([0, 2, 5])), i32_dev(np.array([3, 0, 4, 1, 2])),
                  i32_dev(np.array([20, 40])), i32_dev(np.array([0, 9, 35])), 26)

        def call():
            return A.tree_commit(cache, *tables, tokens, parents, chosen)

        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        for _ in range(4):
            chosen.copy_(torch.randint(0, 3, (n,), device="cuda", dtype=torch.int32))
            before = torch.randint(0, 250, shape, device="cuda").to(cache.dtype)
            cache.copy_(before)
            want = [t.clone() for t in call()] + [cache.clone()]
            cache.copy_(before)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip((*held, cache), want):
                assert torch.equal(a, b)


@BOTH
@pytest.mark.parametrize("cached,nodes", [([100], [1024]), ([0, 1000], [513, 40])])
def test_large_trees(A, fp8, cached, nodes):
    """Masks of up to 32 words; a chain's deepest node sees a thousand others."""
    see, pos = zip(*(tree_bits(list(range(-1, m - 1)) if b == 0 else
                               random_tree(np.random.default_rng(m), m))
                     for b, m in enumerate(nodes)))
    c = Case(11, fp8, cached, nodes, see, [n + p for n, p in zip(cached, pos)])
    rows = np.array([0, 1, 31, 32, 39, 63, 64, 200, 511, 512, 800, 1022, 1023])
    for window in (0, 128):
        c.check(c.run(A, window), window, rows)


@BOTH
def test_many_tiles(A, fp8):
    """More tiles than are shared out, of sequences of several tiles each."""
    rng = np.random.default_rng(12)
    nodes = rng.integers(1, 130, 48).tolist()
    nodes[3], nodes[7] = 129, 0
    c = Case(12, fp8, rng.integers(0, 60, 48).tolist(), nodes)
    rows = np.array([0, 1, 30, 31, 32, 64, 95, 96, 128])
    c.check(c.run(A), 0, rows)
    c.check(c.run(A, 20), 20, rows)


@BOTH
def test_commit_replayed_on_other_rows(A, fp8):
    """Each replay, with eager calls between, moves the rows that are there then."""
    rng = np.random.default_rng(66)
    trees = [random_tree(rng, m, 6) for m in (9, 26)]
    n, shape = 35, (4, 5, AO.FP8_PAGE_BYTES) if fp8 else (4, 5, 2, HKV, PAGE, D)
    parents, tokens = i32_dev(np.concatenate(trees)), i32_dev(rng.integers(0, 3, n))
    chosen = i32_dev(np.zeros(n))
    cache = torch.zeros(shape, dtype=torch.uint8 if fp8 else torch.bfloat16, device="cuda")
    tables = (i32_dev(np.array([0, 2, 5])), i32_dev(np.array([3, 0, 4, 1, 2])),
              i32_dev(np.array([20, 40])), i32_dev(np.array([0, 9, 35])), 26)

    def call():
        return A.tree_commit(cache, *tables, tokens, parents, chosen)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    moved = 0
    for _ in range(6):
        before = torch.randint(0, 250, shape, device="cuda").to(cache.dtype)
        chosen.copy_(torch.randint(0, 3, (n,), device="cuda", dtype=torch.int32))
        cache.copy_(before)
        want = [t.clone() for t in call()]
        rows = cache.clone()
        moved += not torch.equal(rows, before)
        cache.copy_(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and torch.equal(cache, rows)
    assert moved


@BOTH
def test_moves_past_32_bits(A, fp8):
    """Rows and pages of the last layer of caches of more than 4 GB (and 2^31 elements)."""
    page = (AO.FP8_PAGE_BYTES,) if fp8 else (2, HKV, PAGE, D)
    pool = (1 << 31) // (AO.FP8_PAGE_BYTES if fp8 else 32768) + 3000
    cache = torch.empty((3, pool, *page), dtype=torch.uint8 if fp8 else torch.bfloat16,
                        device="cuda")
    ids = [pool - 1, pool - 5, 7, pool - 2]
    small = torch.randint(0, 250, (3, 4, *page), device="cuda").to(cache.dtype)
    cache[:, ids] = small
    i32 = lambda x: i32_dev(np.array(x))  # noqa: E731
    args = (i32([23]), i32([0, 5]), 5, i32([1, 2, 3, 4, 5]), i32([-1, 0, 0, 2, 3]),
            i32([3, 0, 4, 5, 9]))
    for data, pages in ((cache, ids), (small, [0, 1, 2, 3])):
        path, count, after = A.tree_commit(data, i32([0, 2]), i32(pages[:2]), *args)
        assert path.tolist() == [0, 2, 3, 4, -1] and (int(count), int(after)) == (4, 9)
        A.kv_copy_pages(data, i32([pages[1], pages[2]]), i32([pages[3], pages[0]]))
    assert torch.equal(cache[:, ids], small)


@BOTH
@pytest.mark.parametrize("window", [0, 3, 100])
def test_shared_out(A, fp8, window):
    """A bound far above the lengths: the keys of every tile go to as many workgroups as there are,
    whose shares begin and end anywhere; sequences without nodes or keys, of one and of several
    tiles."""
    rng = np.random.default_rng(13)
    for seed, (cached, nodes) in enumerate((
            ([0, 1, 15, 16, 17, 63, 64, 130, 40, 700], [1, 5, 8, 2, 33, 64, 7, 12, 0, 20]),
            ([0, 2000, 3, 0, 900], [0, 4, 0, 1, 3]),
            (rng.integers(0, 600, 64).tolist(), rng.integers(0, 9, 64).tolist()),
            (rng.integers(0, 300, 30).tolist(), rng.integers(9, 17, 30).tolist()),
            ([1500, 40], [70, 100]), ([5], [1]))):
        c = Case(100 + seed, fp8, cached, nodes)
        n, lengths = int(c.starts[-1]), list(c.lengths)
        c.lengths = [*lengths, 100000]                 # (what run takes its bound from)
        got = c.run(A, window)
        c.lengths = lengths
        assert got.shape[0] == n
        c.check(got, window)
