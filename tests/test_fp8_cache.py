"""The 8-bit KV cache on the CPU: the oracle's format against torch's e4m3, the host side of
PagedKVCache, and the refusals of the entry points (no launch, no GPU needed)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from model.kv_cache import FP8_PAGE_BYTES, PagedKVCache  # noqa: E402
from oracle import attn_oracle as AO  # noqa: E402
from oracle import moe_oracle as O  # noqa: E402
from test_abi import header_codes  # noqa: E402

FP8 = torch.float8_e4m3fn


def test_codes_are_torchs_e4m3():
    every = torch.arange(256, dtype=torch.uint8).view(FP8).float().numpy()
    np.testing.assert_array_equal(AO.e4m3_values(), every.astype(np.float64))


def test_quantizer_rounds_to_nearest_even():
    """Every bf16 fraction, ties included, below a row maximum in each of a few binades."""
    for top in (0x4300, 0x3F80, 0x0600, 0x7E80):      # 128, 1, tiny, the last binade but one
        x = (np.arange(top - 0x780, top).clip(0).astype(np.uint16)).reshape(-1, 64)
        x[:, 0] = top | 0x7F                           # the row's largest magnitude
        x[:, 1::2] |= 0x8000
        codes, s = AO.fp8_quantize(x, False)
        want_s = max((top >> 7) - 7, 10)
        assert (s == want_s).all()
        scaled = torch.from_numpy(O.bf16_to_f32(x).astype(np.float64) * 2.0 ** (127 - want_s))
        np.testing.assert_array_equal(codes, scaled.float().to(FP8).view(torch.uint8).numpy())
        back = AO.fp8_dequantize(codes, s)
        v = O.bf16_to_f32(x).astype(np.float64)
        largest = np.abs(v).max(axis=-1, keepdims=True)
        # half a step: 2^-4 of a normal code's value, 2^-10 scale of a subnormal's: 2^-17 of the
        # row's largest, 128 scale or more, but 2^-127 where the scale stops at 2^-117
        bound = np.maximum(np.maximum(np.abs(v) * 2.0 ** -4, largest * 2.0 ** -17), 2.0 ** -127)
        assert (np.abs(back - v) <= bound).all()


def test_quantizer_last_binade():
    """Magnitudes from 2^127 on: 248 2^120 and more become 240 2^120 (off by less than 2^-4)
    and not 2^128."""
    x = np.arange(0x7F00, 0x7F80).astype(np.uint16).reshape(2, 64)
    codes, s = AO.fp8_quantize(x, True)
    v, back = O.bf16_to_f32(x).astype(np.float64), AO.fp8_dequantize(codes, s)
    assert (s == 247).all() and back.max() == 240 * 2.0 ** 120
    assert (np.abs(back - v) <= v * 2.0 ** -4).all()


def test_quantizer_special_rows():
    x = np.zeros((4, 64), dtype=np.uint16)
    x[1, 3], x[2, 63] = 0x7F80, 0xFFC1                # inf, NaN
    x[3, 5] = 1                                       # the smallest subnormal: to 0
    for is_v, code in ((False, 0x7F), (True, 0)):
        codes, s = AO.fp8_quantize(x, is_v)
        assert s.tolist() == [10, 255, 255, 10]
        assert (codes[1:3] == code).all() and (codes[[0, 3]] == 0).all()
        assert np.isnan(AO.fp8_dequantize(codes, s)[1:3]).all()


def test_host_cache():
    c = PagedKVCache(num_layers=3, num_pages=8, max_batch=2, max_tokens=64, device="cpu", dtype=FP8)
    assert c.fp8 and c.data.shape == (3, 8, FP8_PAGE_BYTES) and c.data.dtype == torch.uint8
    assert c.staging.shape == (4, 2, 8, 16, 64) and c.staging_slots.tolist() == list(range(64))
    c.add_sequence(0)
    t = c.begin_forward([0], [20])
    assert c.slots_of(0).tolist() == t.slots.tolist()
    assert c.slots_of(0, 3, 5).tolist() == t.slots[3:5].tolist()
    with pytest.raises(ValueError):
        c.slots_of(0, 3, 21)
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 1, 16, kv_heads=4, device="cpu", dtype=FP8)
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 1, 16, device="cpu", dtype=torch.float8_e5m2)
    assert PagedKVCache(1, 2, 1, 16, device="cpu", dtype=torch.float32).data.dtype == torch.float32
    b = PagedKVCache(num_layers=3, num_pages=8, max_batch=2, max_tokens=64, device="cpu")
    assert not b.fp8
    with pytest.raises(ValueError):
        b.quantize_from(1, b, 0)                       # into a bf16 cache
    with pytest.raises(ValueError):
        c.quantize_from(1, c, 0)                       # from an 8-bit one
    b.add_sequence(5)
    b.begin_forward([5], [64])
    b.seqs[5].length = 16 * 7                          # more than the 6 pages left
    with pytest.raises(MemoryError):
        c.quantize_from(1, b, 5)
    assert 1 not in c.seqs and len(c.free) == 6


@pytest.mark.parametrize("source", [dict(dtype=torch.float32), dict(dtype=torch.float16),
                                    dict(kv_heads=4), dict(head_dim=32), dict()])
def test_refused_move_leaves_the_cache(source):
    """A sequence that quantize_from does not take (or whose rows a launch does not: here, on the
    CPU, the last) is not in the cache afterwards, and its pages are free."""
    c = PagedKVCache(num_layers=2, num_pages=8, max_batch=2, max_tokens=64, device="cpu", dtype=FP8)
    b = PagedKVCache(num_layers=2, num_pages=8, max_batch=2, max_tokens=64, device="cpu", **source)
    b.add_sequence(5)
    b.begin_forward([5], [20])
    free = list(c.free)
    with pytest.raises(ValueError):
        c.quantize_from(1, b, 5)
    assert 1 not in c.seqs and c.free == free and b.seq_len(5) == 20


def test_bf16_cache_reads_its_rows():
    c = PagedKVCache(num_layers=1, num_pages=4, max_batch=1, max_tokens=64, device="cpu")
    c.data.copy_(torch.randn(c.data.shape))
    c.add_sequence(0)
    c.begin_forward([0], [40])
    k, v = c.read(0, 0, 10, 40)
    pages = c.seqs[0].pages
    for i, p in enumerate(range(10, 40)):
        assert torch.equal(k[i], c.data[0, pages[p // 16], 0, :, p % 16])
        assert torch.equal(v[i], c.data[0, pages[p // 16], 1, :, p % 16])


def test_refusals():
    import attn_native as A
    import moe_native
    lib, codes = moe_native.lib(), header_codes()
    P = ctypes.c_void_p
    p, odd = P(0x1000), P(0x1008)       # never dereferenced: validation fails first
    ok, null, shape, align, unsupported, space = (
        codes["MOE_OK"], codes["MOE_ERR_NULL"], codes["MOE_ERR_SHAPE"], codes["MOE_ERR_ALIGN"],
        codes["MOE_ERR_UNSUPPORTED"], codes["MOE_ERR_WORKSPACE"])
    most = 1 << 27                       # pages whose slots no longer fit 31 bits
    # append
    ap = lib.attn_qkv_rope_append_fp8
    assert ap(p, p, 1, p, p, p, 1.0, p, 0, p, None) == shape
    assert ap(p, p, 1, p, p, p, 1.0, p, most, p, None) == shape
    assert ap(p, p, -1, p, p, p, 1.0, p, 4, p, None) == shape
    assert ap(p, p, 1, p, None, p, 1.0, p, 4, p, None) == null
    assert ap(p, p, 1, p, p, p, 1.0, odd, 4, p, None) == align
    assert ap(p, p, 0, p, p, p, 1.0, p, 4, p, None) == ok
    # quantise, read
    qz, rd = lib.attn_kv_quantize_fp8, lib.attn_kv_read_fp8
    assert qz(p, 0, p, 1, p, 4, p, None) == shape and qz(p, 4, p, 1, p, most, p, None) == shape
    assert qz(p, most, p, 1, p, 4, p, None) == shape and qz(p, 4, p, -1, p, 4, p, None) == shape
    assert qz(p, 4, None, 1, p, 4, p, None) == null and qz(odd, 4, p, 1, p, 4, p, None) == align
    assert qz(None, 4, None, 0, None, 4, None, None) == ok
    assert rd(p, 4, p, (1 << 24) + 1, p, p, None) == shape and rd(p, most, p, 1, p, p, None) == shape
    assert rd(p, 4, p, 1, p, None, None) == null and rd(p, 4, p, 1, odd, p, None) == align
    assert rd(None, 4, None, 0, None, None, None) == ok
    # decode
    size = lib.attn_decode_fp8_workspace_bytes
    assert size(0, 100) == 0 and size(1, 0) == 0 and size(65536, 100) == 0
    need = size(2, 1000)
    assert need >= (2 << 20) + 2 * 64 * 3 * 66 * 4      # 3 splits of 4 blocks at least

    def dec(q=p, batch=2, cache=p, pages=8, span=1000, scale=0.125, out=p, ws=p, bytes_=need):
        return lib.attn_decode_fp8(q, batch, cache, pages, p, p, p, span, 0, scale, p, out, ws,
                                   bytes_, None)
    assert dec(bytes_=need - 1) == space and dec(pages=0) == shape and dec(pages=most) == shape
    assert dec(batch=65536) == shape and dec(span=0) == shape and dec(batch=0, q=None) == ok
    assert dec(scale=0.0) == unsupported and dec(scale=float("nan")) == unsupported
    assert dec(scale=float("inf")) == unsupported and dec(scale=-1.0) == unsupported
    assert dec(q=None) == null and dec(ws=None) == null and dec(out=odd) == align
    # chunks
    size = lib.attn_prefill_fp8_workspace_bytes
    assert size(5, 1, 5, 4000, 0) > 0 and size(5, 1, 5, 0, 0) == 0 and size(5, 1, 5, 100, 0) == 0
    assert size(4096, 1, 4096, 4096, 0) == 0            # tiles enough
    for batch in (-1, 0, (1 << 60) + 1, (1 << 62) + 3, (1 << 63) - 1):
        assert size(300, batch, 300, 6300, 0) == 0, batch
    need = size(5, 1, 5, 4000, 0)
    assert size(1 << 20, 1, 5, 4000, 0) == need         # rows behind the sequences cost nothing
    assert size(5, 1, 5, (1 << 63) - 1, 0) == size(5, 1, 5, 1 << 31, 0) < 1 << 28
    for batch in (1, 3, 40, 512):                       # a call's parts are bounded
        for longest in (1, 2, 4, 7, 12, 24, 30, 33, 100, 300, 2000):
            for window in (0, 128):
                assert size(9, batch, longest, 1 << 20, window) <= 64 << 20, (batch, longest)

    def pre(q=p, rows=5, batch=1, longest=5, pages=8, most_kv=4000, scale=0.125, out=p, ws=p,
            bytes_=need):
        return lib.attn_prefill_fp8(q, rows, p, batch, longest, p, pages, p, p, p, most_kv, 0,
                                    scale, p, out, ws, bytes_, None)
    assert pre(bytes_=need - 1) == space and pre(ws=None) == null and pre(ws=odd) == align
    assert pre(pages=0) == shape and pre(rows=-1) == shape and pre(longest=-1) == shape
    assert pre(batch=-1) == shape and pre(batch=1 << 30) == shape and pre(longest=1 << 25) == shape
    assert pre(scale=0.0) == unsupported and pre(q=None) == null and pre(out=odd) == align
    assert pre(rows=0, q=None) == ok and pre(batch=0, q=None) == ok and pre(longest=0) == ok
    # the wrappers: types, shapes and devices before any of that
    cpu = torch.zeros((4, FP8_PAGE_BYTES), dtype=torch.uint8)
    slots = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        A.kv_read_fp8(cpu, slots)
    with pytest.raises(TypeError):
        A.kv_read_fp8(cpu.view(torch.int8), slots)
    assert A.FP8_PAGE_BYTES == FP8_PAGE_BYTES == AO.FP8_PAGE_BYTES


def test_chunks_of_many_sequences():
    """The sizes that attn_prefill takes: up to 2^24 tiles of 64 tokens (checked before the
    pointers, so a call without them says which check it came to)."""
    import attn_native  # noqa: F401  (the entry points' signatures)
    import moe_native
    lib, codes = moe_native.lib(), header_codes()
    p = ctypes.c_void_p(0x1000)

    def pre(batch, longest, window=0):
        return lib.attn_prefill_fp8(None, 1 << 20, p, batch, longest, p, 8, p, p, p, 1 << 20,
                                    window, 0.125, p, p, None, 0, None)
    for window in (0, 128):
        for batch, longest in ((2048, 16384), (65535, 16384), (1, 1 << 24), (63, 1 << 24),
                               (600000, 7), ((1 << 24) - 1, 1)):
            assert pre(batch, longest, window) == codes["MOE_ERR_NULL"], (batch, longest)
        for batch, longest in ((65536, 16384), (64, 1 << 24), (1 << 24, 1)):
            assert pre(batch, longest, window) == codes["MOE_ERR_SHAPE"], (batch, longest)


class Named(torch.Tensor):
    """A tensor of a caller's own class."""


def test_tensors_of_any_class():
    import attn_native as A
    t = torch.zeros((3, 8), dtype=torch.bfloat16)
    for x in (t, torch.nn.Parameter(t, requires_grad=False), t.as_subclass(Named)):
        A._need(x, "x", torch.bfloat16, (3, 8), -1)        # -1: the index of a CPU tensor
        with pytest.raises(ValueError, match="GPU"):
            A._need(x, "x", torch.bfloat16, (3, 8), 0)


def test_arguments_that_are_no_tensors(monkeypatch):
    """None, an array or a single value where a tensor of rows belongs: a TypeError or a
    ValueError that names it, before any launch."""
    import attn_native as A
    monkeypatch.setattr(A, "_need_fp8", lambda cache: (4, -1, None))   # as if on this device
    cache = torch.zeros((4, FP8_PAGE_BYTES), dtype=torch.uint8)
    i32, bf16 = torch.zeros(3, dtype=torch.int32), torch.bfloat16
    q, sinks = torch.zeros((2, 64, 64), dtype=bf16), torch.zeros(64, dtype=bf16)
    src = torch.zeros((1, 2, 8, 16, 64), dtype=bf16)
    for bad in (None, np.zeros((2, 64, 64), dtype=np.float32), 5, torch.zeros((), dtype=bf16),
                torch.zeros((), dtype=torch.int32)):
        for name, call in (
                ("qkv", lambda: A.qkv_rope_append_fp8(bad, None, i32, i32, None, 1.0, cache, q)),
                ("src", lambda: A.kv_quantize_fp8(bad, i32, cache, i32)),
                ("src_slots", lambda: A.kv_quantize_fp8(src, bad, cache, i32)),
                ("slots", lambda: A.kv_read_fp8(cache, bad)),
                ("q", lambda: A.decode_fp8(bad, cache, i32, i32, i32[:2], 9, 0, 0.1, sinks, q,
                                           None)),
                ("page_indices", lambda: A.decode_fp8(
                    q, cache, i32, bad if getattr(bad, "dtype", None) != torch.int32 else "0",
                    i32[:2], 9, 0, 0.1, sinks, q, None)),
                ("workspace", lambda: A.decode_fp8(q, cache, i32, i32, i32[:2], 9, 0, 0.1, sinks,
                                                   q, bad)),
                ("q_indptr", lambda: A.prefill_fp8(q, bad, 1, cache, i32, i32, i32[:2], 0, 0.1,
                                                   sinks, q))):
            with pytest.raises((TypeError, ValueError), match=f"^{name}: "):
                call()


def test_staging_holds_the_fused_projections():
    """A step that takes the fused QKV projection finds a staging row for each of its tokens."""
    import attn_native as A
    c = PagedKVCache(1, 2, 1, 16, device="cpu", dtype=FP8)
    assert c.staging_slots.numel() == c.staging.shape[0] * A.PAGE >= A.ROWS_QKV_MAX_TOKENS
    assert A.ROWS_QKV_MAX_TOKENS >= A.GEMV_MAX_TOKENS
