"""Trees and beams through the model: the attention block over a tree against the oracle's chains,
and the engine's tree step and beam search, replayed from the logits that it saw and the cache that
it left."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from gpu_util import bf16_dev, host_bf16  # noqa: E402

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
CACHES = pytest.mark.parametrize("kv_dtype", [torch.bfloat16, FP8], ids=["bf16", "fp8"])


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import attn_native
    return attn_native


@CACHES
@pytest.mark.parametrize("layer_idx", [0, 1])           # sliding window 128, full attention
def test_attention_block_tree(A, layer_idx, kv_dtype):
    """Trees through the attention block: q, k and v as the oracle projects and rotates them at the
    nodes' positions, and the output as its attention over the rows that the cache holds gives it,
    every node seeing its ancestors."""
    from model.kv_cache import PagedKVCache
    from test_gpu_attention import _block, close
    p = AO.make_attn_params(60 + layer_idx)
    blk, window = _block(A, p, layer_idx), 128 if layer_idx == 0 else 0
    cache = PagedKVCache(2, 60, 2, 256, device="cuda", dtype=kv_dtype)
    prefix = [150, 20]
    for trees in ([[-1, 0, 0, 1, 1, 2, 3, 3, 5], [-1, 0, 1, 1]],
                  [[-1] + [i // 3 for i in range(49)], [-1] + list(range(19))]):   # library QKV
        n = sum(len(t) for t in trees)
        x0, x1 = O.make_input(62, sum(prefix)), O.make_input(63, n)
        with torch.no_grad():
            cache.clear()
            for s in range(2):
                cache.add_sequence(s)
                cache.enable_sliding_window(s, 128)
            cache.begin_forward([0, 1], prefix)
            blk(bf16_dev(x0).view(1, -1, 2880), cache)
            cache.end_forward()
            t = cache.begin_tree([0, 1], trees)
            pos = t.positions.cpu().numpy()
            got = host_bf16(blk(bf16_dev(x1).view(1, -1, 2880), cache).view(-1, 2880))
            cache.end_forward()
        q, k, v = AO.split_qkv(AO.linear(O.rms_norm(x1, p.norm_w, 1e-5), p.qkv_w, p.qkv_b))
        q, k = AO.rope(q, pos), AO.rope(k, pos)
        sinks, o, at = O.bf16_to_f32(p.sinks).astype(np.float64), [], 0
        for s, (c, tree) in enumerate(zip(prefix, trees)):
            m = len(tree)
            rows = slice(at, at + m)
            depth = np.zeros(m, dtype=int)
            see = np.eye(m, dtype=bool)
            for i in range(1, m):
                depth[i], see[i] = depth[tree[i]] + 1, see[tree[i]] | see[i]
            np.testing.assert_array_equal(pos[rows], c + depth)
            kc, vc = (O.bf16_to_f32(host_bf16(x)).astype(np.float64) for x in cache.read(s, layer_idx))
            for mine, want in ((kc[c:], k[rows]), (vc[c:], v[rows])):
                w = O.bf16_to_f32(want).astype(np.float64)
                top = np.abs(w).max(axis=-1, keepdims=True)
                # half a step of the 8-bit codes, and two bf16 ulps of the row's largest for the
                # projection's own roundings
                half = np.abs(w) * 2.0 ** -4 + top * 2.0 ** -17 if cache.fp8 else 0.0
                assert (np.abs(mine - w) <= half + top * 2.0 ** -7).all()
            where = np.concatenate([np.arange(c), pos[rows]])
            seen = np.concatenate([np.ones((m, c), dtype=bool), see], axis=1)
            if window:
                seen &= where[None, :] > pos[rows][:, None] - window
            o.append(AO.attention_seen(O.bf16_to_f32(q[rows]).astype(np.float64), kc, vc, seen,
                                       sinks)[0])
            at += m
        o = O.f32_to_bf16(np.concatenate(o).reshape(n, -1).astype(np.float32))
        y = AO.linear(o, p.out_w, p.out_b)
        close(got, O.f32_to_bf16(O.bf16_to_f32(x1) + O.bf16_to_f32(y)))


def small_engine(kv_dtype, seed, max_batch=1):
    from engine import Engine
    from model.config import GPTOssConfig
    cfg = GPTOssConfig(num_hidden_layers=2, num_experts=32, vocab_size=4096,
                       context_window_size=1024, prefill_chunk_size=512)
    torch.manual_seed(seed)
    eng = Engine(config=cfg, max_total_seq_len=1024, kv_dtype=kv_dtype, max_batch=max_batch)
    for name, w in eng.model.named_parameters():
        if w.dtype == torch.uint8:
            w.copy_(torch.randint(*((114, 118) if "scales" in name else (0, 256)), w.shape,
                                  dtype=torch.uint8, device="cuda"))
        elif "norm" not in name:
            w.copy_(torch.randn(w.shape, device="cuda") * (1.0 if "embedding" in name else 0.02))
    return eng


def snapshot(cache, sid):
    return [tuple(host_bf16(t) for t in cache.read(sid, i)) for i in range(2)]


def same(a, b):
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x[0], y[0])
        np.testing.assert_array_equal(x[1], y[1])


@CACHES
def test_decode_tree(A, kv_dtype):
    """Steps over trees: the tokens follow from the logits of the nodes by the sampler and the walk;
    the cache holds the rows that it held and those that the path's nodes wrote, in order; and a
    plain decode goes on from there."""
    eng = small_engine(kv_dtype, 70)
    cache, p = eng.paged_kv_cache, eng.sample_parameters
    rng = np.random.default_rng(71)
    seq = eng.begin_sequence()
    token = eng.sample(eng.prefill(rng.integers(0, 4096, 140).astype(np.int32), seq))
    seen = {}
    logits_of, end = eng.model.decode_logits_bf16, cache.end_forward

    def record(embed, c):
        out = logits_of(embed, c)
        seen["logits"] = out.float().cpu().numpy()
        seen["rows"] = snapshot(c, seq)
        return out

    eng.model.decode_logits_bf16 = record
    length, accepted, guess = 140, 0, {}
    for step in range(12):
        # the tokens that an earlier pass over the same place took, where there was one, as drafts
        # among others
        tree, tokens = [-1, 0, 0, 1, 1, 2, 2, 3], [token] + rng.integers(0, 4096, 7).tolist()
        for node in (2, 5):
            if (step % 2, node) in guess and step % 2:
                tokens[node] = guess[(step % 2, node)]
        before = snapshot(cache, seq)
        root = token
        new = eng.decode_tree(tokens, tree, seq)
        chosen = [AO.sample_top_p_from_logits(x, p["temperature"], p["top_p"], p["random_seed"])
                  for x in seen["logits"]]
        way = AO.tree_walk(tokens, tree, chosen)
        assert new == [tokens[i] for i in way[1:]] + [chosen[way[-1]]]
        assert int(eng._token.item()) == new[-1]
        assert cache.seq_len(seq) == length + len(way)
        after = snapshot(cache, seq)
        same([(k[:length], v[:length]) for k, v in after], before)
        same([(k[length:], v[length:]) for k, v in after],
             [(k[length:][way], v[length:][way]) for k, v in seen["rows"]])
        accepted += len(way) - 1
        if step % 2 == 0:    # again from the same place, now with what was chosen as a draft
            eng.popn(seq, len(way))
            token, guess = root, {(1, 2): chosen[0], (1, 5): chosen[2]}
        else:
            token, length = new[-1], length + len(way)
    assert accepted >= 3
    eng.model.decode_logits_bf16 = logits_of
    lg = eng.decode(np.array([token], dtype=np.int32), seq)
    assert torch.isfinite(lg).all() and eng.get_kv_total_seq_len() == length + 1


@CACHES
def test_decode_tree_refusals(A, kv_dtype):
    eng = small_engine(kv_dtype, 72)
    seq = eng.begin_sequence()
    eng.prefill(np.arange(20, dtype=np.int32), seq)
    for tokens, parents in (([1, 2], [-1]), ([1], [0]), ([1, 2], [-1, 1]), ([], [])):
        with pytest.raises(ValueError):
            eng.decode_tree(tokens, parents, seq)
    assert eng.get_kv_total_seq_len() == 20 and eng.paged_kv_cache.tables is None
    assert len(eng.decode_tree([3], [-1], seq)) == 1 and eng.get_kv_total_seq_len() == 21


@CACHES
@pytest.mark.parametrize("width,stops", [(1, 0), (4, 0), (3, 2)])
def test_beam_search(A, kv_dtype, width, stops):
    """Every step's choice follows from the logits that the step saw, and every beam's rows are those
    that its own line of tokens wrote, whatever pages it shared on the way."""
    eng = small_engine(kv_dtype, 73, max_batch=width)
    cache = eng.paged_kv_cache
    other = eng.begin_sequence()                       # a sequence that is none of its business
    eng.prefill(np.arange(37, dtype=np.int32), other)
    held, free = snapshot(cache, other), len(cache.free)
    steps = []
    select, begin, end = A.beam_top_k, cache.begin_forward, cache.end_forward
    rows, batch = {}, []

    def spy(logits, scores, k):
        steps.append((logits.float().cpu().numpy(), scores.cpu().numpy(), k))
        return select(logits, scores, k)

    def began(ids, counts, *rest):
        t = begin(ids, counts, *rest)
        batch[:] = list(zip(ids, counts))
        for sid, n in batch:                           # what was there before is its line's
            if sid in rows:
                same([(k[:-n], v[:-n]) for k, v in snapshot(cache, sid)], rows[sid])
        return t

    def ended_():
        for sid, _ in batch:
            rows[sid] = snapshot(cache, sid)
        end()

    branch = cache.branch

    def branched(ids, parents, new=None):
        old = [rows[s] for s in ids]
        branch(ids, parents, new)
        for s in ids:
            del rows[s]
        for s, q in zip(new, parents):
            rows[s] = old[q]

    A.beam_top_k, cache.begin_forward, cache.end_forward, cache.branch = spy, began, ended_, branched
    stop = []
    try:
        if stops:                                       # tokens that beams do meet
            first = eng.beam_search(np.arange(100, 150, dtype=np.int32), width, 5)
            stop = [first[0][0][2], first[-1][0][3]]
            steps.clear()
        got = eng.beam_search(np.arange(100, 150, dtype=np.int32), width, 20, stop)
    finally:
        A.beam_top_k, cache.begin_forward, cache.end_forward, cache.branch = select, begin, end, branch
    beams, finished = [([], np.float32(0))], []
    for x, s, k in steps:
        # (the selection's bound on a score: test_gpu_beams.py)
        for (_, v), score in zip(beams, s[0], strict=True):
            assert abs(v - score) <= 2.0 ** -24 * abs(v) + 2.0 ** -20
        beams, live = [(b[0], v) for b, v in zip(beams, s[0])], []
        for v, b, t in zip(*AO.beam_top_k(x, s[0], k)):
            if len(live) == width:
                break
            (finished if t in stop else live).append((beams[b][0] + [int(t)], np.float32(v)))
        beams = live
    want = sorted(finished + beams, key=lambda b: b[1], reverse=True)[:width]
    assert [b[0] for b in got] == [b[0] for b in want]
    assert np.allclose([b[1] for b in got], [b[1] for b in want], rtol=2.0 ** -24, atol=2.0 ** -20)
    assert len(steps) == 20 or len(finished) >= width
    if stops:
        assert finished
    assert len(cache.free) == free and list(cache.seqs) == [other]
    same(snapshot(cache, other), held)
    with pytest.raises(ValueError):
        eng.beam_search([1, 2], width + 1, 3)
    assert len(cache.free) == free
