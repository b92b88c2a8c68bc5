"""Workloads of the 8-bit paged KV cache and of the attention that reads it.

Five kinds:

  append    the bias, RoPE and cache append after the QKV projection of a prompt's chunk, with k
            and v quantised as they are written; what was written is read back
  quantise  rows of a bf16 cache into an 8-bit one: a decode step's new rows, or a whole
            sequence that moves; what was written is read back
  read      a sequence's rows back as bf16 values
  decode    attention of one new token for each of a ragged batch of sequences
  chunk     causal attention of each sequence's new tokens over its cached ones: drafted tokens
            under verification, the next turn of a chat, a prompt

The cache's format.  A row is the 64 values of one token, head and k or v.  It has one scale byte
s and 64 e4m3 codes: a code c stands for c 2^(s - 127), s = max(e - 7, 10) for e the biased
exponent of the row's largest magnitude, and codes round to nearest even (at s = 247, the last, they
stop at 240).  A row with an infinity
or a NaN has s = 255 and stands for NaN (its codes: NaN in k, 0 in v).  A page of 16 tokens is 16640
bytes: the codes of k [head][token][dim], those of v [head][token / 4][dim % 16][dim / 16][token % 4]
(four tokens of a dimension in a word), then the scales [head][k, v][token].

Attention: out = sum_j p_j v_j / (sum_j p_j + exp(sink)), p_j = exp(q . k_j / 8), over the keys up
to the query's position, and within the window where there is one.

Keys get a fixed gain per head and dimension (a few of them large, as trained keys have), values one
per token; queries are twice N(0, 1), so the softmax is neither flat nor a single key.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
FP8 = torch.float8_e4m3fn
QH, KVH, DIM, PAGE = 64, 8, 64, 16
GROUP = QH // KVH
QKV = (QH + 2 * KVH) * DIM
CODES = KVH * PAGE * DIM                    # code bytes of a page's keys, or of its values
PAGE_BYTES = 2 * CODES + 2 * KVH * PAGE
ROW = 2 * KVH * (DIM + 1)                   # bytes of a token in the cache
SCALE = 1.0 / math.sqrt(DIM)
WINDOW = 128
CONTEXT = 40960


def _native():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "gpt-oss-tvm_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import attn_native
    return attn_native


# -- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # an ordinary chat prompt
        {"name": "append_prompt333", "kind": "append", "tokens": 333, "prefix": 0},
        # a full prefill chunk in the middle of a long document
        {"name": "append_chunk8192", "kind": "append", "tokens": 8192, "prefix": 16384},
        # the new rows of a decode step of 48 sequences
        {"name": "quantise_decode48", "kind": "quantise", "tokens": 48},
        # an idle sequence of the longest context moves to the 8-bit cache
        {"name": "quantise_context40960", "kind": "quantise", "tokens": CONTEXT},
        # a chat's cache on its way to another cache or to host memory
        {"name": "read_sequence1000", "kind": "read", "tokens": 1000},
        # the same at the longest context
        {"name": "read_context40960", "kind": "read", "tokens": CONTEXT},
        # one chat at a time: every full layer of every token of a single user's answer
        {"name": "decode1_context777", "kind": "decode", "sequences": 1, "context": 777,
         "window": False},
        # a full layer of a decode batch with chats of all lengths
        {"name": "decode64_context4096", "kind": "decode", "sequences": 64, "context": 4096,
         "window": False},
        # two users, each with a book in the context
        {"name": "decode2_context131072", "kind": "decode", "sequences": 2, "context": 131072,
         "window": False},
        # a few drafted tokens of each sequence of a batch under verification
        {"name": "chunk5_16x4000", "kind": "chunk", "sequences": 16, "tokens": 5, "prefix": 4000,
         "window": False},
        # the next turn of a chat: a short text over what is cached
        {"name": "chunk300_over6000", "kind": "chunk", "sequences": 1, "tokens": 300,
         "prefix": 6000, "window": False},
        # a long prompt
        {"name": "chunk4096", "kind": "chunk", "sequences": 1, "tokens": 4096, "prefix": 0,
         "window": False},
    ]


def _spread(rng, lo, hi):
    """An integer of lo..hi, uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["append", "quantise", "read", "decode", "decode", "chunk", "chunk", "chunk"])
    if kind == "append":
        return {"kind": kind, "tokens": _spread(rng, 1, 8192), "prefix": rng.randint(0, 32768)}
    if kind in ("quantise", "read"):
        return {"kind": kind, "tokens": _spread(rng, 1, CONTEXT)}
    if kind == "decode":
        sequences = _spread(rng, 1, 96)
        # no more keys than the longest listed context's two
        context = _spread(rng, 1, min(131072, 2 * 131072 // sequences))
        return {"kind": kind, "sequences": sequences, "context": context,
                "window": rng.random() < 0.3}
    sequences = rng.choice([1, 1, 2, 3, 8, 16, 40])
    tokens = _spread(rng, 1, 4096 if sequences == 1 else 2048 // sequences)
    # no more query-key pairs than the listed prompt has
    most = max(0, min(16384, 4096 * 2048 // (tokens * sequences) - tokens // 2))
    return {"kind": kind, "sequences": sequences, "tokens": tokens,
            "prefix": rng.choice([0, rng.randint(0, most), _spread(rng, 1, most + 1) - 1]),
            "window": rng.random() < 0.3}


# -- inputs, from the seed alone ------------------------------------------------------------

def _gen(seed, *parts):
    g = torch.Generator(device=DEV)
    value = 1469598103934665603
    for p in (seed, *parts):
        value = ((value ^ (int(p) + 7)) * 1099511628211) % (1 << 63)
    g.manual_seed(value)
    return g


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def _lengths(case):
    """(cached, new) tokens of each sequence, the same for every seed: one of full length, the
    others between a quarter (cached) or a half (new) of it and all of it."""
    kind, b = case["kind"], case.get("sequences", 1)
    rng = random.Random("%s %d" % (kind, b))
    out = []
    for i in range(b):
        part, piece = (1.0, 1.0) if i == 0 else (rng.uniform(0.25, 1.0), rng.uniform(0.5, 1.0))
        if kind == "decode":  # the new token included
            out.append((max(1, round(case["context"] * part)) - 1, 1))
        elif kind == "chunk":
            out.append((round(case["prefix"] * part), max(1, round(case["tokens"] * piece))))
        else:
            out.append((0, case["tokens"]))
    return out


def _pool(lengths):
    return sum(-(-(c + n) // PAGE) for c, n in lengths) + 5


def _inputs(case, seed):
    """The tensors in hand before a call, the sequences' pages scattered over the pool."""
    kind, g = case["kind"], _gen(seed, 1)
    lengths = _lengths(case)
    pool = _pool(lengths)
    ids = torch.randperm(pool, generator=g, device=DEV)
    x = {"pool": pool, "lengths": lengths}
    if kind in ("append", "quantise", "read"):
        n = case["tokens"]
        t = torch.arange(n, device=DEV)
        x["slots"] = (ids[t // PAGE] * PAGE + t % PAGE).int()
        gain = torch.exp(_normal(g, (KVH, DIM), 0.5))
        if kind == "append":
            qkv = _normal(g, (n, QKV))
            qkv[:, QH * DIM:(QH + KVH) * DIM] *= gain.flatten()
            x["qkv"] = qkv.to(BF)
            x["bias"] = _normal(g, (QKV,), 0.1).to(BF)
            x["positions"] = (t + case["prefix"]).int()
            x["inv_freq"] = (150000.0 ** (-torch.arange(DIM // 2, device=DEV).double()
                                          / (DIM // 2))).float()
        else:
            rows = _normal(g, (pool, 2, KVH, PAGE, DIM))
            rows[:, 0] *= gain[:, None, :]
            rows[:, 1] *= torch.exp(_normal(g, (pool, 1, PAGE, 1), 0.5))
            x["rows"] = rows.to(BF)
            # where they lie in the bf16 cache
            mine = torch.randperm(pool, generator=g, device=DEV)
            x["from"] = (mine[t // PAGE] * PAGE + t % PAGE).int()
        return x
    indptr, used = [0], 0
    for c, m in lengths:
        used += -(-(c + m) // PAGE)
        indptr.append(used)
    n = sum(m for _, m in lengths)
    x["q"] = _normal(g, (n, QH, DIM), 2.0).to(BF)
    x["sinks"] = _normal(g, (QH,)).to(BF)
    x["cache"] = torch.empty((pool, PAGE_BYTES), dtype=torch.uint8, device=DEV)
    gain = torch.exp(_normal(g, (KVH, 1, DIM), 0.5))
    for part in x["cache"].split(4096):      # every row of every page, those behind the ends too
        p = part.shape[0]
        k = _normal(g, (p, KVH, PAGE, DIM)) * gain
        v = _normal(g, (p, KVH, PAGE, DIM)) * torch.exp(_normal(g, (p, 1, PAGE, 1), 0.5))
        _put(part, torch.arange(p * PAGE, device=DEV), k.to(BF).transpose(1, 2).flatten(0, 1),
             v.to(BF).transpose(1, 2).flatten(0, 1))
    x["page_indptr"] = torch.tensor(indptr, dtype=torch.int32, device=DEV)
    x["page_indices"] = ids[:used].int()
    x["kv_len"] = torch.tensor([c + m for c, m in lengths], dtype=torch.int32, device=DEV)
    starts = [0]
    for _, m in lengths:
        starts.append(starts[-1] + m)
    x["q_indptr"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    return x


def prepare(case, seed):
    kind = case["kind"]
    with torch.no_grad():
        x = _inputs(case, seed)
        x["kind"] = kind
        if kind == "append":
            x["q"] = torch.empty((case["tokens"], QH, DIM), dtype=BF, device=DEV)
        if kind in ("append", "quantise", "read"):
            x["cache"] = torch.zeros((x["pool"], PAGE_BYTES), dtype=torch.uint8, device=DEV)
        if kind == "read":
            k, v = _rows_of(x["rows"], x["from"])
            _put(x["cache"], x["slots"].long(), k, v)
            del x["rows"], x["from"]
        if kind in ("decode", "chunk"):
            x["window"] = WINDOW if case["window"] else 0
            x["max_q"] = max(m for _, m in x["lengths"])
            x["max_kv"] = max(c + m for c, m in x["lengths"])
            x["out"] = torch.empty_like(x["q"])
        if own:
            x["native"] = _native()
            if kind == "decode":
                x["span"] = min(x["max_kv"], x["window"] or x["max_kv"])
                x["workspace"] = x["native"].decode_fp8_workspace(len(x["lengths"]), x["span"],
                                                                  DEV)
        return x


# -- one pass ------------------------------------------------------------------------------

def run(x):
    with torch.no_grad():
        return _run_own(x) if own else _run_plain(x)


def _run_own(x):
    a, kind = x["native"], x["kind"]
    if kind == "append":
        a.qkv_rope_append_fp8(x["qkv"], x["bias"], x["positions"], x["slots"], x["inv_freq"],
                              _CONCENTRATION, x["cache"], x["q"])
        return (x["q"], *a.kv_read_fp8(x["cache"], x["slots"]))
    if kind == "quantise":
        a.kv_quantize_fp8(x["rows"], x["from"], x["cache"], x["slots"])
        return a.kv_read_fp8(x["cache"], x["slots"])
    if kind == "read":
        return a.kv_read_fp8(x["cache"], x["slots"])
    tables = (x["cache"], x["page_indptr"], x["page_indices"], x["kv_len"])
    if kind == "decode":
        return a.decode_fp8(x["q"], *tables, x["span"], x["window"], SCALE, x["sinks"], x["out"],
                            x["workspace"])
    return a.prefill_fp8(x["q"], x["q_indptr"], x["max_q"], *tables, x["window"], SCALE,
                         x["sinks"], x["out"], x["max_kv"])


# -- the plain forms ---------------------------------------------------------------------------

_CONCENTRATION = float(np.float32(0.1 * math.log(32.0) + 1.0))


def _quantise(x, code_of_bad):
    """[..., 64] bf16 -> (codes [..., 64] and scale bytes [...], uint8)."""
    x = x.float()
    amax = x.abs().amax(-1)
    exponent = (amax.view(torch.int32) >> 23) & 255
    bad = exponent == 255
    s = torch.where(bad, 255, (exponent - 7).clamp(min=10))
    inverse = ((254 - s.clamp(max=247)) << 23).view(F32)       # 2^(127 - s)
    most = torch.where(s == 247, 240.0, 256.0)[..., None]
    x = torch.minimum(torch.maximum(x * inverse[..., None], -most), most)
    codes = torch.where(bad[..., None], code_of_bad, x).to(FP8)
    return codes.view(torch.uint8), s.to(torch.uint8)


def _parts(cache):
    """Views of the pages: codes of k and of v, scales."""
    return (cache[:, :CODES].unflatten(1, (KVH, PAGE, DIM)),
            cache[:, CODES:2 * CODES].unflatten(1, (KVH, PAGE // 4, DIM // 4, 4, 4)),
            cache[:, 2 * CODES:].unflatten(1, (KVH, 2, PAGE)))


def _put(cache, slots, k, v):
    """k, v [n, 8, 64] bf16 -> the rows at slots [n]."""
    kc, vc, sc = _parts(cache)
    page, at = slots // PAGE, slots % PAGE
    kc[page, :, at], sc[page, :, 0, at] = _quantise(k, math.nan)
    codes, sc[page, :, 1, at] = _quantise(v, 0.0)
    vc[page, :, at // 4, :, :, at % 4] = codes.unflatten(-1, (4, DIM // 4)).transpose(-1, -2)


def _get(cache, slots):
    """The rows at slots [n], k and v [n, 8, 64] fp32."""
    kc, vc, sc = _parts(cache)
    page, at = slots // PAGE, slots % PAGE
    out = []
    v = vc[page, :, at // 4, :, :, at % 4].transpose(-1, -2).flatten(-2)
    for codes, s in ((kc[page, :, at], sc[page, :, 0, at]), (v, sc[page, :, 1, at])):
        factor = torch.where(s == 255, math.nan, (s.int() << 23).view(F32))
        out.append(codes.view(FP8).float() * factor[..., None])
    return out


def _rows_of(rows, slots):
    """k, v [n, 8, 64] of a bf16 cache [pages, 2, 8, 16, 64]."""
    page, at = slots.long() // PAGE, slots.long() % PAGE
    return rows[page, 0, :, at], rows[page, 1, :, at]


def _rope(x, positions, inv_freq):
    """x [n, heads, 64] fp32: cos and sin rounded to bf16 and scaled, products and sums in fp32."""
    angle = (positions.float()[:, None] * inv_freq).double()
    cos, sin = ((f.float().to(BF).float() * _CONCENTRATION)[:, None, :]
                for f in (torch.cos(angle), torch.sin(angle)))
    a, b = x[..., :DIM // 2], x[..., DIM // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).to(BF)


def _attend(q, k, v, first, window, sinks):
    """q [n, 64, 64] at positions first.., k, v [m, 8, 64], fp32: a few heads at a time."""
    n, m = q.shape[0], k.shape[0]
    at = torch.arange(first, first + n, device=DEV)[:, None]
    key = torch.arange(m, device=DEV)[None, :]
    hidden = (key > at) | (key <= at - window) if window else key > at
    q = q.view(n, KVH, GROUP, DIM).permute(1, 2, 0, 3)             # [8, 8, n, 64]
    k, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    sinks = sinks.view(KVH, GROUP, 1, 1)
    step = max(1, min(KVH, (1 << 27) // max(1, GROUP * n * m)))
    outs = []
    for h in range(0, KVH, step):
        s = torch.matmul(q[h:h + step].reshape(-1, GROUP * n, DIM), k[h:h + step]) * SCALE
        s = s.view(-1, GROUP, n, m).masked_fill(hidden, -math.inf)
        top = torch.maximum(s.amax(-1, keepdim=True), sinks[h:h + step])
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True) + torch.exp(sinks[h:h + step] - top)
        o = torch.matmul(p.view(-1, GROUP * n, m), v[h:h + step]).view(-1, GROUP, n, DIM)
        outs.append(o / total)
    return torch.cat(outs).permute(2, 0, 1, 3).reshape(n, QH, DIM)


def _run_plain(x):
    kind, cache = x["kind"], x["cache"]
    if kind == "append":
        y = (x["qkv"].float() + x["bias"].float()).to(BF).float().view(-1, QH + 2 * KVH, DIM)
        qk = _rope(y[:, :QH + KVH], x["positions"], x["inv_freq"])
        slots = x["slots"].long()
        _put(cache, slots, qk[:, QH:], y[:, QH + KVH:].to(BF))
        k, v = _get(cache, slots)
        return qk[:, :QH].contiguous(), k.to(BF), v.to(BF)
    if kind in ("quantise", "read"):
        slots = x["slots"].long()
        if kind == "quantise":
            _put(cache, slots, *_rows_of(x["rows"], x["from"]))
        k, v = _get(cache, slots)
        return k.to(BF), v.to(BF)
    out, row, page = [], 0, 0
    sinks = x["sinks"].float()
    for cached, new in x["lengths"]:
        total = cached + new
        pages = x["page_indices"][page:page - (-total // PAGE)].long()
        low = max(0, cached - x["window"] + 1) if x["window"] else 0   # the first key in sight
        t = torch.arange(low, total, device=DEV)
        k, v = _get(cache, pages[t // PAGE] * PAGE + t % PAGE)
        out.append(_attend(x["q"][row:row + new].float(), k, v, cached - low, x["window"], sinks))
        row, page = row + new, page - (-total // PAGE)
    return torch.cat(out).to(BF)


# -- what a pass cannot do without -------------------------------------------------------------

def _attended(cached, new, window):
    """(query-key pairs, keys read) of one head and one sequence."""
    w = window or (cached + new)
    pairs = sum(min(p + 1, w) for p in range(cached, cached + new))
    return pairs, min(cached + new, w + new - 1)


def work(case):
    kind, n = case["kind"], case.get("tokens", 0)
    values = 2 * KVH * DIM
    if kind == "append":
        return {"bytes": n * (QKV * 2 + QH * DIM * 2 + ROW + values * 2 + 8) + QKV * 2,
                "flops": n * (QKV + 3 * (QH + KVH) * DIM + 2 * values)}
    if kind == "quantise":
        return {"bytes": n * (values * 2 + ROW + values * 2 + 8), "flops": n * 3 * values}
    if kind == "read":
        return {"bytes": n * (ROW + values * 2 + 4), "flops": n * values}
    lengths = _lengths(case)
    each = [_attended(c, m, WINDOW if case["window"] else 0) for c, m in lengths]
    return {"bytes": sum(k for _, k in each) * ROW + sum(m for _, m in lengths) * QH * DIM * 4,
            "flops": sum(p for p, _ in each) * QH * 4.0 * DIM}


# -- the same in 64 bits, apart from the forms above ---------------------------------------------
# The roundings that belong to the definition (the bias's sum, the tables of cos and sin, the
# rotation's products and sums, k and v to bf16 and then to their codes) are made where it makes
# them, in numpy.

def _bf16(a):
    """float32 array -> rounded to bf16, as float32."""
    u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def _stored(a):
    """What the cache holds of rows a [..., 64]: multiples of the code's step, ties to even."""
    a = np.asarray(a, dtype=np.float64)
    top = np.abs(a).max(-1, keepdims=True)
    _, e = np.frexp(top)                          # top = f 2^e, f in [0.5, 1)
    unit = np.exp2(np.maximum(np.where(top > 0, e - 1 - 7, -200), -117).astype(np.float64))
    c = np.where(top >= 2.0 ** 127, np.clip(a / unit, -240.0, 240.0), a / unit)
    _, e = np.frexp(c)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)   # e4m3: 3 fraction bits, exponents from -6
    return np.rint(c / step) * step * unit


def _host(t):
    return t.float().cpu().numpy()


def _to_bf(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float64)).to(DEV)


def _decoded(cache, pages, low, total):
    """k, v [total - low, 8, 64] float64, from the codes' bits."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    value = np.where(e == 0, f / 8.0 * 2.0 ** -6, (1 + f / 8.0) * np.exp2(e - 7.0))
    value = np.where((c & 127) == 127, np.nan, np.where(c & 128, -value, value))
    table = torch.from_numpy(value).to(DEV)
    mine = cache[pages]
    p = mine.shape[0]
    scale = torch.exp2(mine[:, 2 * CODES:].view(p, KVH, 2, PAGE).double() - 127.0)
    k = table[mine[:, :CODES].int()].view(p, KVH, PAGE, DIM) * scale[:, :, 0, :, None]
    v = table[mine[:, CODES:2 * CODES].int()].view(p, KVH, PAGE // 4, DIM // 4, 4, 4)
    v = v.permute(0, 1, 2, 5, 4, 3).reshape(p, KVH, PAGE, DIM) * scale[:, :, 1, :, None]
    k = k.permute(0, 2, 1, 3).reshape(p * PAGE, KVH, DIM)
    v = v.permute(0, 2, 1, 3).reshape(p * PAGE, KVH, DIM)
    return k[low:total], v[low:total]


def exact(case, seed):
    kind = case["kind"]
    with torch.no_grad():
        x = _inputs(case, seed)
        if kind == "append":
            y = _bf16(_host(x["qkv"]) + _host(x["bias"])).reshape(-1, QH + 2 * KVH, DIM)
            angle = (_host(x["positions"]).astype(np.float32)[:, None]
                     * _host(x["inv_freq"])).astype(np.float64)
            conc = np.float32(_CONCENTRATION)
            cos, sin = ((_bf16(f.astype(np.float32)) * conc)[:, None, :]
                        for f in (np.cos(angle), np.sin(angle)))
            half = DIM // 2
            qk = y[:, :QH + KVH]
            turned = np.empty_like(qk)
            turned[..., :half] = qk[..., :half] * cos - qk[..., half:] * sin
            turned[..., half:] = qk[..., :half] * sin + qk[..., half:] * cos
            turned = _bf16(turned)
            return (_to_bf(turned[:, :QH]), _to_bf(_stored(turned[:, QH:])),
                    _to_bf(_stored(y[:, QH + KVH:])))
        if kind in ("quantise", "read"):
            k, v = _rows_of(x["rows"], x["from"])
            return _to_bf(_stored(_host(k))), _to_bf(_stored(_host(v)))
        window = WINDOW if case["window"] else 0
        out, row, page = [], 0, 0
        for cached, new in x["lengths"]:
            total = cached + new
            count = (total + PAGE - 1) // PAGE
            first = max(0, cached + 1 - window) // PAGE * PAGE if window else 0
            pages = x["page_indices"][page + first // PAGE:page + count].long()
            k, v = _decoded(x["cache"], pages, 0, total - first)
            q = x["q"][row:row + new].double()
            pos = torch.arange(cached, total, device=DEV)
            at = torch.arange(first, total, device=DEV)
            seen = at[None, :] <= pos[:, None]
            if window:
                seen &= at[None, :] > pos[:, None] - window
            heads = []
            for h in range(QH):
                s = q[:, h] @ k[:, h // GROUP].t() / 8.0
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                lse = torch.logsumexp(s, dim=1, keepdim=True)
                o = torch.exp(s - lse) @ v[:, h // GROUP]
                heads.append(o * torch.sigmoid(lse - x["sinks"][h].double()))
            out.append(torch.stack(heads, dim=1))
            row, page = row + new, page + count
        return torch.cat(out)
