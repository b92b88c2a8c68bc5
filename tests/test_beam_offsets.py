"""Logits whose first row begins anywhere: a later request's rows of an odd vocabulary."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_abi import header_codes  # noqa: E402


def test_four_bytes_are_enough():
    """Words are no misalignment for the entry point (another refusal comes first: no launch)."""
    import attn_native  # noqa: F401
    import moe_native
    lib, codes, p = moe_native.lib(), header_codes(), ctypes.c_void_p(16)
    for f32 in (0, 1):
        for at, want in ((20, "MOE_ERR_WORKSPACE"), (24, "MOE_ERR_WORKSPACE"), (17, "MOE_ERR_ALIGN"),
                         (18, "MOE_ERR_ALIGN")):
            assert lib.attn_beam_top_k(ctypes.c_void_p(at), f32, 2, 4, 1001, p, 8, p, p, p, p, 1,
                                       None) == codes[want], (at, f32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 5, 1001, 30011])
def test_rows_from_any_element_on(dtype, vocab):
    import attn_native as A
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((6, vocab), generator=g, device="cuda").to(dtype)
    scores = torch.tensor([[0.0, -0.5, -0.25], [-0.1, 0.0, -3.0]], device="cuda")
    k = min(6, 3 * vocab)
    want = A.beam_top_k(x, scores, k)
    for off in range(1, 10):
        held = torch.full((6 * vocab + 16,), 50.0, dtype=dtype, device="cuda")
        held[off:off + 6 * vocab] = x.flatten()
        view = held[off:off + 6 * vocab].view(6, vocab)
        for a, b in zip(A.beam_top_k(view, scores, k), want):
            np.testing.assert_array_equal(a.cpu().numpy(), b.cpu().numpy())
    late = A.beam_top_k(x[3:], scores[1:], k)             # the second request's rows alone
    for a, b in zip(late, want):
        np.testing.assert_array_equal(a[0, :k].cpu().numpy(), b[1].cpu().numpy())
