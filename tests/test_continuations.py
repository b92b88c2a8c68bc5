"""Trees of drafted tokens and beams on the CPU: the entry points' refusals (no launch, no GPU
needed) and the oracle's own rules."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attn_oracle as AO  # noqa: E402
from test_abi import header_codes  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    import attn_native  # noqa: F401  (registers the signatures)
    import moe_native
    return moe_native.lib()


P, ODD = ctypes.c_void_p(16), ctypes.c_void_p(18)      # never dereferenced: validation fails first


def refused(fn, good, changes):
    codes = header_codes()
    for at, value, code in changes:
        args = list(good)
        args[at] = value
        assert fn(*args) == codes[code], (at, value, code)


@pytest.mark.parametrize("name", ["attn_tree", "attn_tree_fp8"])
def test_tree_refusals(lib, name):
    fn = getattr(lib, name)
    #        q rows qi batch maxq mask words pos cache pages ptr ids len maxkv window scale sinks out ws
    good = [P, 8, P, 1, 8, P, 1, P, P, 4, P, P, P, 50, 0, 0.125, P, P, P, 1 << 40, None]
    refused(fn, good, [
        (1, -1, "MOE_ERR_SHAPE"), (1, (1 << 24) + 1, "MOE_ERR_SHAPE"), (3, -1, "MOE_ERR_SHAPE"),
        (3, 65536, "MOE_ERR_SHAPE"), (4, -1, "MOE_ERR_SHAPE"), (4, 1025, "MOE_ERR_SHAPE"),
        (4, 33, "MOE_ERR_SHAPE"), (6, 0, "MOE_ERR_SHAPE"), (6, 33, "MOE_ERR_SHAPE"),
        (9, 0, "MOE_ERR_SHAPE"), (9, 1 << 27, "MOE_ERR_SHAPE"), (13, -1, "MOE_ERR_SHAPE"),
        (15, 0.0, "MOE_ERR_UNSUPPORTED"), (15, float("nan"), "MOE_ERR_UNSUPPORTED"),
        (15, float("inf"), "MOE_ERR_UNSUPPORTED"), (15, -1.0, "MOE_ERR_UNSUPPORTED"),
        *((i, None, "MOE_ERR_NULL") for i in (0, 2, 5, 7, 8, 10, 11, 12, 16, 17)),
        *((i, ODD, "MOE_ERR_ALIGN") for i in (0, 2, 5, 7, 8, 10, 11, 12, 17)),
        (16, ctypes.c_void_p(17), "MOE_ERR_ALIGN"),
        (1, 0, "MOE_OK"), (3, 0, "MOE_OK"), (4, 0, "MOE_OK")])
    need = lib.attn_tree_workspace_bytes(1, 8, 100000, 0)
    if need:
        long = list(good)
        long[13] = 100000
        refused(fn, long, [(18, None, "MOE_ERR_NULL"), (18, ODD, "MOE_ERR_ALIGN"),
                           (19, need - 1, "MOE_ERR_WORKSPACE")])


def test_tree_workspace_bytes(lib):
    """A pure function, small for any arguments."""
    for batch in (-1, 0, 1, 3, 64, 65535, (1 << 62) + 3):
        for longest in (-1, 0, 1, 5, 64, 1024, 1 << 40):
            for most in (-1, 0, 1, 777, 131072, (1 << 31) - 1, (1 << 62) + 1):
                for window in (-1, 0, 1, 128, (1 << 31) - 1):
                    got = lib.attn_tree_workspace_bytes(batch, longest, most, window)
                    assert got == lib.attn_tree_workspace_bytes(batch, longest, most, window)
                    assert 0 <= got <= 1 << 28, (batch, longest, most, window)


@pytest.mark.parametrize("name", ["attn_tree_commit", "attn_tree_commit_fp8"])
def test_commit_refusals(lib, name):
    #    cache layers pages ptr ids len qi batch rows maxq tokens parents chosen path count next
    good = [P, 2, 4, P, P, P, P, 1, 8, 8, P, P, P, P, P, P, None]
    refused(getattr(lib, name), good, [
        (1, 0, "MOE_ERR_SHAPE"), (1, 65536, "MOE_ERR_SHAPE"), (2, 0, "MOE_ERR_SHAPE"),
        (7, -1, "MOE_ERR_SHAPE"), (7, 65536, "MOE_ERR_SHAPE"), (8, -1, "MOE_ERR_SHAPE"),
        (8, (1 << 24) + 1, "MOE_ERR_SHAPE"), (9, -1, "MOE_ERR_SHAPE"), (9, 1025, "MOE_ERR_SHAPE"),
        *((i, None, "MOE_ERR_NULL") for i in (0, 3, 4, 5, 6, 10, 11, 12, 13, 14, 15)),
        *((i, ODD, "MOE_ERR_ALIGN") for i in (0, 3, 4, 5, 6, 10, 11, 12, 13, 14, 15)),
        (7, 0, "MOE_OK")])


def test_copy_refusals(lib):
    good = [P, 2, 4, 16640, P, P, 3, None]
    refused(lib.attn_kv_copy_pages, good, [
        (1, 0, "MOE_ERR_SHAPE"), (1, 65536, "MOE_ERR_SHAPE"), (2, 0, "MOE_ERR_SHAPE"),
        (2, 1 << 27, "MOE_ERR_SHAPE"), (3, 0, "MOE_ERR_SHAPE"), (3, 24, "MOE_ERR_SHAPE"),
        (3, 1 << 21, "MOE_ERR_SHAPE"), (6, -1, "MOE_ERR_SHAPE"),
        *((i, None, "MOE_ERR_NULL") for i in (0, 4, 5)),
        *((i, ODD, "MOE_ERR_ALIGN") for i in (0, 4, 5)), (6, 0, "MOE_OK")])


def test_beam_refusals(lib):
    #   logits f32 batch width vocab scores k out beams tokens ws bytes
    good = [P, 0, 2, 4, 1000, P, 8, P, P, P, P, 1 << 40, None]
    need = lib.attn_beam_workspace_bytes(2, 4, 1000, 8)
    assert need > 0
    refused(lib.attn_beam_top_k, good, [
        (2, -1, "MOE_ERR_SHAPE"), (2, 65536, "MOE_ERR_SHAPE"), (3, 0, "MOE_ERR_SHAPE"),
        (3, 65, "MOE_ERR_UNSUPPORTED"), (4, 0, "MOE_ERR_SHAPE"), (4, 1 << 30, "MOE_ERR_SHAPE"),
        (4, 1, "MOE_ERR_SHAPE"), (6, 0, "MOE_ERR_SHAPE"), (6, 65, "MOE_ERR_UNSUPPORTED"),
        *((i, None, "MOE_ERR_NULL") for i in (0, 5, 7, 8, 9, 10)),
        *((i, ODD, "MOE_ERR_ALIGN") for i in (0, 5, 7, 8, 9, 10)),
        (11, need - 1, "MOE_ERR_WORKSPACE"), (2, 0, "MOE_OK")])
    assert lib.attn_beam_workspace_bytes(0, 4, 1000, 8) == 0
    assert lib.attn_beam_workspace_bytes(2, 4, 1, 8) == 0


def test_wrappers_refuse_host_tensors():
    import attn_native as A
    i = torch.zeros(2, dtype=torch.int32)
    bf = torch.zeros((4, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        A.beam_top_k(bf, torch.zeros((1, 4)), 2)
    with pytest.raises(TypeError):
        A.beam_top_k(bf.double(), torch.zeros((1, 4)), 2)
    with pytest.raises(TypeError):
        A.beam_top_k([1.0], torch.zeros((1, 4)), 2)
    with pytest.raises(ValueError, match="GPU"):
        A.kv_copy_pages(torch.zeros((1, 4, 2, 8, 16, 64), dtype=torch.bfloat16), i, i)
    with pytest.raises(TypeError):
        A.kv_copy_pages(torch.zeros((1, 4, 2, 8, 16, 64)), i, i)
    with pytest.raises(ValueError, match="GPU"):
        A.tree_commit(torch.zeros((1, 4, 16640), dtype=torch.uint8), i, i, i, i, 1, i, i, i)
    q = torch.zeros((1, 64, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        A.tree(q, i, 1, i.view(2, 1), i, torch.zeros((4, 2, 8, 16, 64), dtype=torch.bfloat16), i, i,
               i, 0, 0.125, q, q)
    with pytest.raises(ValueError, match="GPU"):
        A.tree_fp8(q, i, 1, i.view(2, 1), i, torch.zeros((4, 16640), dtype=torch.uint8), i, i, i, 0,
                   0.125, q, q)


def test_oracle_walk():
    #        0
    #      1   2     (the same token), 3 under 1, 4 under 2
    parents, tokens = [-1, 0, 0, 1, 2], [9, 5, 5, 7, 8]
    assert AO.tree_walk(tokens, parents, [5, 8, 8, 0, 0]) == [0, 1]       # the lowest child
    assert AO.tree_walk(tokens, parents, [5, 7, 8, 0, 0]) == [0, 1, 3]
    assert AO.tree_walk(tokens, parents, [6, 7, 8, 0, 0]) == [0]
    assert AO.tree_walk([], [], []) == []


def test_oracle_beams():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.8, 0.1]]))
    s, b, t = AO.beam_top_k(x, np.array([0.0, -1.0]), 6)
    np.testing.assert_allclose(s, np.sort(np.concatenate([x[0], x[1] - 1]))[::-1])
    assert (b.tolist(), t.tolist()) == ([0, 1, 0, 0, 1, 1], [0, 1, 1, 2, 0, 2])


def test_oracle_attention_seen_is_the_causal_one():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 64, 64)), *rng.standard_normal((2, 9, 8, 64))
    sinks = rng.standard_normal(64)
    seen = np.arange(9)[None, :] <= np.array([6, 7, 8])[:, None]
    for window in (0, 4):
        mask = seen & (np.arange(9)[None, :] > np.array([6, 7, 8])[:, None] - window) if window else seen
        for a, b in zip(AO.attention_seen(q, k, v, mask, sinks),
                        AO.attention_sink(q, k, v, np.array([6, 7, 8]), window, sinks)):
            np.testing.assert_allclose(a, b, rtol=1e-12)


# -- the cache's host side ---------------------------------------------------------------------

def make(pages=12, batch=4, tokens=64):
    from model.kv_cache import PagedKVCache
    return PagedKVCache(num_layers=2, num_pages=pages, max_batch=batch, max_tokens=tokens,
                        device="cpu", dtype=torch.float32)


def write(c, t, values):
    """Row i of a forward's tokens gets values[i] in k and -values[i] in v, in every layer."""
    for i, slot in enumerate(t.slots.tolist()):
        c.data[:, slot // 16, 0, :, slot % 16] = float(values[i])
        c.data[:, slot // 16, 1, :, slot % 16] = -float(values[i])
    c.end_forward()


def rows(c, sid):
    out = []
    for layer in range(2):
        k, v = c.read(sid, layer)
        assert torch.equal(k, -v) and (k == k[:, :1, :1]).all()
        out.append(k[:, 0, 0].tolist())
    assert out[0] == out[1]
    return out[0]


def test_branches_share_pages_until_they_write():
    c = make()
    c.add_sequence(0)
    c.enable_sliding_window(0, 128)
    write(c, c.begin_forward([0], [20]), range(20))
    c.branch([0], [0, 0, 0], [5, 6, 0])
    assert len(c.free) == 10 and c.total_sequence_length() == 60
    assert c.seqs[5].pages == c.seqs[6].pages == c.seqs[0].pages
    t = c.begin_forward([5, 6, 0], [1, 1, 1])       # two of three copy the part-filled page
    assert len(c.free) == 8 and t.windows == (128,) * 3
    write(c, t, [100, 101, 102])
    for sid, last in ((5, 100), (6, 101), (0, 102)):
        assert rows(c, sid) == list(range(20)) + [last]
    # beams 6 and 0 end, 5 goes on twice
    c.branch([5, 6, 0], [0, 0, 1], [5, 6, 0])
    assert len(c.free) == 9
    write(c, c.begin_forward([5, 6, 0], [1, 1, 13]), [200, 201] + list(range(300, 313)))
    assert rows(c, 5) == list(range(20)) + [100, 200]
    assert rows(c, 6) == list(range(20)) + [100, 201]
    assert rows(c, 0) == list(range(20)) + [101] + list(range(300, 313))
    for sid in (5, 0, 6):
        c.remove_sequence(sid)
    assert sorted(c.free) == list(range(12)) and not any(c._refs)


def test_branch_at_a_page_end_and_popn_into_shared_pages():
    c = make()
    c.add_sequence(0)
    write(c, c.begin_forward([0], [32]), range(32))
    c.branch([0], [0, 0], [0, 1])
    write(c, c.begin_forward([0, 1], [1, 1]), [50, 51])     # pages of their own: nothing to copy
    assert len(c.free) == 8
    c.popn(1, 13)                                            # into the shared second page
    assert len(c.free) == 9
    write(c, c.begin_forward([1], [2]), [60, 61])            # which is copied first
    assert len(c.free) == 8
    assert rows(c, 1) == list(range(20)) + [60, 61]
    assert rows(c, 0) == list(range(32)) + [50]
    c.popn(0, 33)
    write(c, c.begin_forward([0], [1]), [7])
    assert rows(c, 0) == [7] and rows(c, 1) == list(range(20)) + [60, 61]
    c.clear()
    assert sorted(c.free) == list(range(12)) and not any(c._refs)


def test_branch_refusals():
    c = make(pages=3)
    c.add_sequence(0)
    c.add_sequence(1)
    write(c, c.begin_forward([0], [17]), range(17))
    for args in (([0], [0, 0]), ([0], [1]), ([0], [-1]), ([0, 0], [0]), ([7], [0]),
                 ([0], [0, 0], [2, 2]), ([0], [0, 0], [0, 1]), ([0], [0, 0], [2])):
        with pytest.raises(ValueError):
            c.branch(*args)
    assert c.seqs[0].length == 17 and sorted(c.seqs) == [0, 1] and len(c.free) == 1
    c.branch([0], [0, 0, 0], [0, 2, 3])
    with pytest.raises(MemoryError):                 # two copies needed, one page free
        c.begin_forward([0, 2, 3], [1, 1, 1])
    assert c.seqs[0].pages == c.seqs[2].pages == c.seqs[3].pages and len(c.free) == 1
    c.branch([0, 2, 3], [], [])                      # no branch: all of them end
    assert sorted(c.seqs) == [1] and len(c.free) == 3


def test_begin_tree_tables():
    c = make()
    c.add_sequence(0)
    c.add_sequence(1)
    write(c, c.begin_forward([0, 1], [20, 3]), range(23))
    wide = [-1] + [0] * 39
    t = c.begin_tree([0, 1], [[-1, 0, 0, 1, 3], wide])
    assert not t.is_decode and t.max_q_len == 40 and t.kv_len.tolist() == [25, 43]
    assert t.positions.tolist() == [20, 21, 21, 22, 23] + [3] + [4] * 39
    assert t.parents.tolist() == [-1, 0, 0, 1, 3] + wide
    ids = c.seqs[0].pages
    assert t.slots[:5].tolist() == [ids[1] * 16 + 4 + i for i in range(5)]
    m = t.tree_mask.numpy().view(np.uint32)
    assert m.shape == (45, 2)
    assert m[:5, 0].tolist() == [1, 3, 5, 11, 27] and not m[:5, 1].any()
    assert m[5 + 31].tolist() == [1 | 1 << 31, 0] and m[5 + 32].tolist() == [1, 1]
    c.end_forward()
    c.popn(0, 3)
    assert c.seq_len(0) == 22
    for bad in ([], [0], [-1, 1], [-1, -1], [-1, 0, 5], [-1] + [0] * 1024):
        with pytest.raises(ValueError):
            c.begin_tree([0], [bad])
    assert c.seq_len(0) == 22 and c.tables is None
    assert not c.begin_tree([0], [[-1]]).is_decode


def test_trees_of_as_many_different_sequences():
    c = make()
    c.add_sequence(0)
    c.add_sequence(1)
    for ids, trees in (([0, 0], [[-1], [-1]]), ([0, 1], [[-1]]), ([0], [[-1], [-1]])):
        with pytest.raises(ValueError):
            c.begin_tree(ids, trees)
    assert c.seq_len(0) == c.seq_len(1) == 0 and len(c.free) == 12


def test_last_holder_of_a_page_needs_no_copy():
    c = make(pages=2)
    c.add_sequence(0)
    write(c, c.begin_forward([0], [5]), range(5))
    c.branch([0], [0, 0], [0, 1])
    write(c, c.begin_forward([0, 1], [1, 1]), [10, 11])      # one copy, the one page there is
    assert not c.free and rows(c, 0) == [*range(5), 10] and rows(c, 1) == [*range(5), 11]
    c.clear()
    c.add_sequence(0)
    write(c, c.begin_forward([0], [5]), range(5))
    c.branch([0], [0, 0, 0], [0, 1, 2])
    with pytest.raises(MemoryError):                         # sequence 2 keeps it: two copies
        c.begin_forward([0, 1], [1, 1])
    write(c, c.begin_forward([1], [1]), [20])
    assert not c.free and rows(c, 1) == [*range(5), 20] and rows(c, 0) == rows(c, 2) == [*range(5)]
