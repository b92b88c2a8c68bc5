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
