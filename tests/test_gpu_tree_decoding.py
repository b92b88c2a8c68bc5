"""Engine.decode_tree against decode and sample one token at a time."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_engine_continuations import A, CACHES, small_engine  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@CACHES
@pytest.mark.parametrize("seed", [80, 81, 82])
def test_the_tokens_of_decoding_one_by_one(A, kv_dtype, seed):  # noqa: F811
    """With the largest logit as the sample (temperature 0) a tree whose nodes are the right tokens
    and others gives what single steps give, as far as these are certain: the kernels of a tree and
    of a step round differently, eight bf16 roundings of the residual's size in two layers, so the
    logits may differ by about 8 2^-8 of their spread and a lead of 2^-3 of it decides."""
    eng = small_engine(kv_dtype, seed)
    eng.sample_parameters["temperature"] = 0.0
    rng = np.random.default_rng(seed)
    prompt = rng.integers(0, 4096, 140).astype(np.int32)
    one = eng.begin_sequence()
    line, certain = [eng.sample(eng.prefill(prompt, one))], [True]
    for _ in range(24):
        x = eng.decode(np.array([line[-1]], dtype=np.int32), one).flatten()
        top = x.topk(2).values
        line.append(eng.sample(x.view(1, 1, -1)))
        certain.append(bool(top[0] - top[1] > x.std() / 8))
    two = eng.begin_sequence()
    assert eng.sample(eng.prefill(prompt, two)) == line[0]
    at = 0                                   # line[at] is the root
    steps = []
    while at < 20 and len(steps) < 30:
        # the right token among wrong ones at three depths: nodes 2, 4, 7
        tree = [-1, 0, 0, 2, 2, 1, 4, 4, 3]
        tokens = [line[at]] + rng.integers(0, 4096, 8).tolist()
        for depth, node in enumerate((2, 4, 7)):
            tokens[node] = line[at + 1 + depth]
        before = eng.paged_kv_cache.seq_len(two)
        new = eng.decode_tree(tokens, tree, two)
        assert eng.paged_kv_cache.seq_len(two) == before + len(new)
        good = 0
        while good < len(new) and new[good] == line[at + 1 + good]:
            good += 1
        steps.append(good)
        if good < len(new) or len(new) < 4:  # not the same, or not as far as the drafts go
            assert not certain[at + 1 + good], (at, new, line[at + 1:at + 5])
            if good < len(new):
                break                        # (another line from here on)
        at += len(new)
    assert sum(steps) >= 4
