"""Sequences that share pages list them once each, so a forward's page lists may be longer than the
pool: the tables have to hold them, or the forward is refused before anything changes."""
import pytest

torch = pytest.importorskip("torch")

from model.kv_cache import PagedKVCache  # noqa: E402


def make(pages, batch, tokens, **kw):
    return PagedKVCache(num_layers=1, num_pages=pages, max_batch=batch, max_tokens=tokens,
                        kv_heads=1, head_dim=8, device="cpu", dtype=torch.float32, **kw)


def branched(prompt, beams, pages, tokens=None, **kw):
    c = make(pages, beams, tokens or max(prompt, 64), **kw)
    c.add_sequence(0)
    for at in range(0, prompt, c.max_tokens):
        c.begin_forward([0], [min(c.max_tokens, prompt - at)])
        c.end_forward()
    c.branch([0], [0] * beams, list(range(beams)))
    return c


def check(c, ids, counts, depths, t):
    """Every table against the sequences themselves."""
    at, rows = [0], 0
    for i, (sid, a) in enumerate(zip(ids, counts)):
        s = c.seqs[sid]
        start = s.length - a
        assert t.page_indices[at[-1]:at[-1] + len(s.pages)].tolist() == s.pages
        at.append(at[-1] + len(s.pages))
        assert t.kv_len[i] == s.length
        assert t.positions[rows:rows + a].tolist() == [start + d for d in depths[i]]
        assert t.slots[rows:rows + a].tolist() == [s.pages[p // 16] * 16 + p % 16
                                                   for p in range(start, s.length)]
        rows += a
    assert t.page_indptr.tolist() == at and t.page_indices.numel() == at[-1]
    assert t.q_indptr.tolist() == [sum(counts[:i]) for i in range(len(counts) + 1)]
    assert t.num_tokens == rows == t.positions.numel() == t.slots.numel()


@pytest.mark.parametrize("prompt,beams,pages", [(160, 4, 24), (250, 8, 32), (165, 4, 24)])
@pytest.mark.parametrize("kind", ["step", "tree", "chunk"])
def test_lists_longer_than_the_pool(prompt, beams, pages, kind):
    c = branched(prompt, beams, pages)
    c.data.copy_(torch.arange(pages).view(1, -1, 1, 1, 1, 1).expand(c.data.shape))
    before = {s: list(c.seqs[s].pages) for s in range(beams)}
    ids = list(range(beams))
    if kind == "tree":
        tree = [-1, 0, 0, 1, 2]
        counts, depths = [5] * beams, [[0, 1, 1, 2, 2]] * beams
        t = c.begin_tree(ids, [tree] * beams)
    else:
        counts = [1 if kind == "step" else 3 + i % 3 for i in ids]
        depths = [range(a) for a in counts]
        t = c.begin_forward(ids, counts)
    assert t.page_indices.numel() > pages
    check(c, ids, counts, depths, t)
    for sid in ids:                       # a copied page holds what the shared one did
        for new, old in zip(c.seqs[sid].pages, before[sid]):
            assert (c.data[0, new] == (c.data[0, old] if new != old else float(old))).all()
            assert (c.data[0, new] == float(old)).all()
    assert prompt % 16 == 0 or len({c.seqs[s].pages[prompt // 16] for s in ids}) == beams


def test_lists_that_do_not_fit_are_refused_whole():
    """A cache whose tables have room for 50 entries: a forward that lists more changes nothing."""
    c = branched(160, 4, 24, max_listed=50)
    state = {s: (q.length, list(q.pages)) for s, q in c.seqs.items()}
    free, refs = list(c.free), list(c._refs)
    t = c.begin_forward([0, 1, 2, 3], [1] * 4)                 # 44
    check(c, [0, 1, 2, 3], [1] * 4, [[0]] * 4, t)
    c.end_forward()
    for s in range(4):
        c.popn(s, 1)
    assert {s: (q.length, list(q.pages)) for s, q in c.seqs.items()} == state
    for call in (lambda: c.begin_forward([0, 1, 2, 3], [40] * 4 if c.max_tokens >= 160 else [16] * 4),
                 lambda: c.begin_tree([0, 1, 2, 3], [[-1] + [0] * 39] * 4)):
        with pytest.raises(MemoryError, match="max_listed"):
            call()
        assert {s: (q.length, list(q.pages)) for s, q in c.seqs.items()} == state
        assert sorted(c.free) == sorted(free) and c._refs == refs
    assert make(24, 4, 64, max_listed=1)._page_indices.numel() == 24   # never less than the pool


def test_room_of_the_tables():
    assert make(24, 4, 64)._page_indices.numel() == 96
    assert make(24, 1, 64)._page_indices.numel() == 24


def test_trees_whose_upload_fails_change_nothing(monkeypatch):
    c = branched(20, 2, 24)

    def fails(_):
        raise MemoryError("no memory")

    with monkeypatch.context() as m:
        m.setattr(torch, "from_numpy", fails)
        with pytest.raises(MemoryError):
            c.begin_tree([0, 1], [[-1, 0], [-1]])
    assert c.seq_len(0) == c.seq_len(1) == 20 and c.tables is None
    assert c.begin_tree([0, 1], [[-1, 0], [-1]]).parents.tolist() == [-1, 0, -1]
