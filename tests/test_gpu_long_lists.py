"""Beams over a prompt that fills half of the pool: their page lists are longer than the pool."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_engine_continuations import A, CACHES, small_engine  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@CACHES
def test_beams_and_trees_over_half_a_pool(A, kv_dtype):  # noqa: F811
    """The same as in a cache with a pool for four such prompts; a forward of a tree a beam too, whose
    tokens take the long tables behind the lists."""
    eng = small_engine(kv_dtype, 90, max_batch=4)
    prompt = np.random.default_rng(90).integers(0, 4096, 500).astype(np.int32)
    tree = [-1, 0, 0, 1, 2]
    tokens = np.random.default_rng(91).integers(0, 4096, 20).astype(np.int32)
    out = []
    for pages in (eng.paged_kv_cache.num_pages, 400):
        eng.paged_kv_cache = eng.model.create_paged_kv_cache(4, 16 * (pages - 4), 512, 16, "cuda",
                                                             dtype=kv_dtype)
        cache = eng.paged_kv_cache
        assert cache.num_pages == pages and (4 * 32 > pages) == (pages < 400)
        beams = eng.beam_search(prompt, 4, 6)
        one = eng.begin_sequence()
        eng.prefill(prompt, one)
        cache.branch([one], [0] * 4, [one, 1001, 1002, 1003])
        with torch.no_grad():
            t = cache.begin_tree([one, 1001, 1002, 1003], [tree] * 4)
            assert t.page_indices.numel() == 128
            logits = eng.model.decode_logits_bf16(eng.model.embed(eng._ids(tokens)), cache)
            cache.end_forward()
        cache.clear()
        out.append((beams, logits.float().cpu().numpy()))
    assert out[0][0] == out[1][0]
    np.testing.assert_array_equal(out[0][1], out[1][1])
    # (the trees hold other tokens each, so an error in one beam's pages would show)
    assert len({x.tobytes() for x in out[0][1]}) == 20
