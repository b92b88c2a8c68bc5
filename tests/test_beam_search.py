"""Engine.beam_search on the CPU over a small table model (the next token's probabilities follow
from the last token), against every continuation there is."""
import itertools
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402


def table_engine(monkeypatch, table, width):
    """An engine whose model's logits are rows of `table` [vocab, vocab]; the selection is the
    oracle's."""
    import engine as E
    from model.kv_cache import PagedKVCache
    table = torch.as_tensor(np.asarray(table, dtype=np.float32))

    def top_k(logits, scores, k):
        s, b, t = AO.beam_top_k(logits.numpy(), scores[0].numpy(), k)
        return [torch.as_tensor(np.asarray(x))[None] for x in (s.astype(np.float32), b, t)]

    monkeypatch.setattr(E.A, "beam_top_k", top_k)
    eng = object.__new__(E.Engine)
    eng.device = torch.device("cpu")
    eng.config = types.SimpleNamespace(vocab_size=len(table), sliding_window_size=0)
    eng.paged_kv_cache = PagedKVCache(1, 40, width, 64, kv_heads=1, head_dim=8, device="cpu",
                                      dtype=torch.float32)
    eng.steps = 0

    def logits(embed, cache):
        eng.steps += 1
        return table[embed.long()]

    eng.model = types.SimpleNamespace(embed=lambda ids: ids, decode_logits_bf16=logits,
                                      prefill=lambda embed, cache: logits(embed[-1:], cache))
    return eng


def best_of_all(table, start, n, stops, penalty, width):
    """The best `width` of all continuations that end with a stop token or have n tokens."""
    p = np.asarray(table, dtype=np.float64)
    p = p - np.log(np.exp(p).sum(axis=1, keepdims=True))
    out = []
    for length in range(1, n + 1):
        for c in itertools.product(range(len(p)), repeat=length):
            if any(t in stops for t in c[:-1]) or (length < n and c[-1] not in stops):
                continue
            s = sum(p[a, b] for a, b in zip((start, *c), c))
            out.append((list(c), s))
    return sorted(out, key=lambda b: b[1] / len(b[0]) ** penalty, reverse=True)[:width]


def test_unfinished_beams_are_no_results(monkeypatch):
    """Token 3 ends a continuation (.3), token 0 goes on (.6): of two beams the first to end are not
    the last word, and no prefix that neither ended nor has all its tokens is an answer."""
    table = np.log(np.tile([.6, .05, .05, .3], (4, 1)))
    for penalty in (0.0, 1.0):
        eng = table_engine(monkeypatch, table, 2)
        got = eng.beam_search([1], 2, 20, [3], penalty)
        for tokens, score in got:
            assert tokens[-1] == 3 or len(tokens) == 20, tokens
            assert abs(score - sum(table[0, t] for t in tokens)) < 1e-4
        if penalty == 0.0:
            assert [t for t, _ in got] == [[3], [0, 3]] and eng.steps < 6
        else:                                  # -0.511 a token, whatever follows
            assert got[0][0] == [0] * 20 and eng.steps == 20


@pytest.mark.parametrize("penalty", [0.0, 0.5, 1.0, 2.0, -0.5])
@pytest.mark.parametrize("seed", range(6))
def test_against_all_continuations(monkeypatch, seed, penalty):
    """With as many beams as there are prefixes the search is exact: it may stop early only where
    nothing can come that is better."""
    rng = np.random.default_rng(seed)
    table = rng.standard_normal((3, 3)) * 1.5
    n, width = 4, 16                            # 2 tokens go on: at most 2^4 live beams
    eng = table_engine(monkeypatch, table, width)
    got = eng.beam_search([1], width, n, [2], penalty)
    want = best_of_all(table, 1, n, {2}, penalty, width)
    # (continuations of the same steps in another order are equally good: compared by their worth)
    every = {tuple(t): s for t, s in best_of_all(table, 1, n, {2}, penalty, None)}
    assert len({tuple(t) for t, _ in got}) == len(got) == len(want)
    np.testing.assert_allclose([s for _, s in got], [every[tuple(t)] for t, _ in got],
                               rtol=1e-5, atol=1e-5)
    np.testing.assert_allclose([s / len(t) ** penalty for t, s in got],
                               [s / len(t) ** penalty for t, s in want], rtol=1e-5, atol=1e-5)
    assert not eng.paged_kv_cache.seqs and len(eng.paged_kv_cache.free) == 40


@pytest.mark.parametrize("penalty", [0.0, 0.7, -0.5])
def test_later_and_better(monkeypatch, penalty):
    """Narrow searches over sharp tables: the result is the best of the lines that the search
    follows to their ends, stopping early or not."""
    rng = np.random.default_rng(9)
    for _ in range(20):
        table = rng.standard_normal((6, 6)) * 3
        width, n, stops = 2, 9, {4, 5}
        got = table_engine(monkeypatch, table, width).beam_search([0], width, n, stops, penalty)
        p = table.astype(np.float32).astype(np.float64)
        p = p - np.log(np.exp(p).sum(axis=1, keepdims=True))
        live, ended = [([], 0.0)], []           # the same search without any early end
        for _ in range(n):
            all_ = sorted((([*c, t], s + p[([0] + c)[-1], t]) for c, s in live for t in range(6)),
                          key=lambda b: -b[1])
            live, k = [], width * 3
            for c, s in all_[:k]:
                if len(live) == width:
                    break
                (ended if c[-1] in stops else live).append((c, s))
        want = sorted(ended + live, key=lambda b: b[1] / len(b[0]) ** penalty, reverse=True)[:width]
        assert [t for t, _ in got] == [t for t, _ in want]


def test_nothing_left(monkeypatch):
    """Rows without a continuation end the search with what has ended."""
    table = np.full((3, 3), -np.inf)
    table[0, 2] = table[0, 1] = 0.0             # 1: no token follows
    eng = table_engine(monkeypatch, table, 2)
    assert [t for t, _ in eng.beam_search([0], 2, 5, [2])] == [[2]]
    assert eng.beam_search([1], 2, 5) == []
