"""Workloads of decoding several continuations at once: trees of drafted tokens, and beams.

Four kinds:

  tree    attention of each sequence's tree of drafted tokens over its paged cache
  commit  after verification: the walk from each tree's root along the tokens that the model chose,
          and the accepted tokens' keys and values moved behind the cached ones, in every layer
  beams   the best k continuations of each request over its beams and the vocabulary
  pages   the last, partly filled pages of beams that have the same parent copied, in every layer

A tree.  Node 0 is the last token that was sampled, whose keys and values are not cached yet; every
other node has its parent before it.  A sequence of c cached tokens holds its node i at index c + i
of its pages; the node's position is c plus its depth.  Bit j of row i of the mask (bit j % 32 of
word j / 32): node i sees node j, itself and its ancestors.  Every node sees the cached tokens, and
where there is a window only keys of positions above its own minus the window.

Attention: out = sum_j p_j v_j / (sum_j p_j + exp(sink)), p_j = exp(q . k_j / 8), over the keys seen.

The walk.  From node 0 on: the child of the node at hand whose token is the one that the model chose
after it (the first of them), until there is none; `next` is what the model chose after the last.
Accepted node i of the path moves to index c + i.

Beams.  The score of (beam b, token t) is scores[b] + log_softmax(logits[b])[t]; a row without a
maximum (NaN, +inf, nothing but -inf) has -inf everywhere.  Equal scores: the lowest beam, then the
lowest token.

The caches: bf16 [pages, 2 (k, v), 8, 16, 64], or the 8-bit one of 16640 bytes a page: e4m3 codes of
the keys [head][token][dim], of the values [head][token / 4][dim % 16][dim / 16][token % 4], then
scale bytes [head][k, v][token]; a code c stands for c 2^(s - 127).

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
CODES = KVH * PAGE * DIM                    # code bytes of a page's keys, or of its values
PAGE_BYTES = 2 * CODES + 2 * KVH * PAGE
BF_PAGE_BYTES = 2 * KVH * PAGE * DIM * 2
SCALE = 1.0 / math.sqrt(DIM)
WINDOW = 128
VOCAB = 201088
SHARED = 512                                # tokens of a prompt that sequences share


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
        # one chat at a time, a draft of a few tokens from the text itself: a chain
        {"name": "tree1x5_over777", "kind": "tree", "cache": "bf16", "sequences": 1, "nodes": 5,
         "context": 777, "window": False},
        # a batch of chats, each with a small tree from a draft head
        {"name": "tree16x8_over4000", "kind": "tree", "cache": "bf16", "sequences": 16, "nodes": 8,
         "context": 4000, "window": False},
        # the same batch size and larger trees in a layer with a sliding window
        {"name": "tree32x16_window", "kind": "tree", "cache": "bf16", "sequences": 32, "nodes": 16,
         "context": 4000, "window": True},
        # one user, a large tree over a long document, 8-bit cache
        {"name": "tree1x64_over16000_fp8", "kind": "tree", "cache": "fp8", "sequences": 1,
         "nodes": 64, "context": 16000, "window": False},
        # two users, each with a book in the context, 8-bit cache
        {"name": "tree2x26_over131072_fp8", "kind": "tree", "cache": "fp8", "sequences": 2,
         "nodes": 26, "context": 131072, "window": False},
        # one user's tree through all layers of the smaller model
        {"name": "commit1x8", "kind": "commit", "cache": "bf16", "sequences": 1, "nodes": 8,
         "layers": 24},
        # a full batch through all layers of the larger one, 8-bit cache
        {"name": "commit64x26_fp8", "kind": "commit", "cache": "fp8", "sequences": 64, "nodes": 26,
         "layers": 36},
        # one request of four beams; twice as many candidates, as some may end
        {"name": "beams1x4", "kind": "beams", "type": "bf16", "requests": 1, "beams": 4, "k": 8,
         "vocab": VOCAB},
        # logits as the model's decode returns them
        {"name": "beams4x5_f32", "kind": "beams", "type": "f32", "requests": 4, "beams": 5,
         "k": 10, "vocab": VOCAB},
        # a batch of requests
        {"name": "beams16x8", "kind": "beams", "type": "bf16", "requests": 16, "beams": 8, "k": 16,
         "vocab": VOCAB},
        # three of four beams descend from one: two copies in every layer
        {"name": "pages2", "kind": "pages", "cache": "bf16", "pages": 2, "layers": 24},
        # sixteen requests of eight beams
        {"name": "pages80_fp8", "kind": "pages", "cache": "fp8", "pages": 80, "layers": 36},
    ]


def _spread(rng, lo, hi):
    """An integer of lo..hi, uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "commit", "beams", "beams", "pages"])
    cache = rng.choice(["bf16", "fp8"])
    if kind == "tree":
        sequences = rng.choice([1, 1, 2, 3, 8, 16, 32, 64])
        nodes = _spread(rng, 1, 64 if sequences <= 8 else 26)
        # no more keys, and no more query-key pairs, than the longest listed context has
        most = min(131072, 2 * 131072 // sequences, 2 * 26 * 131072 // (sequences * nodes))
        return {"kind": kind, "cache": cache, "sequences": sequences, "nodes": nodes,
                "context": rng.choice([0, _spread(rng, 1, most), _spread(rng, 1, most)]),
                "window": rng.random() < 0.3}
    if kind == "commit":
        return {"kind": kind, "cache": cache, "sequences": _spread(rng, 1, 64),
                "nodes": _spread(rng, 1, 26), "layers": rng.choice([24, 36])}
    if kind == "beams":
        requests = _spread(rng, 1, 16)
        beams = _spread(rng, 1, 8)
        return {"kind": kind, "type": rng.choice(["bf16", "f32"] if requests * beams <= 64
                                                 else ["bf16"]),
                "requests": requests, "beams": beams, "k": rng.choice([1, 2]) * beams,
                "vocab": rng.choice([VOCAB, _spread(rng, 1000, VOCAB)])}
    return {"kind": kind, "cache": cache, "pages": _spread(rng, 1, 80 if cache == "fp8" else 40),
            "layers": rng.choice([24, 36])}


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
    """(cached, nodes) of each sequence, the same for every seed: one of full length, the others
    between a quarter (cached) or a half (nodes) of it and all of it."""
    rng = random.Random("%s %d" % (case["kind"], case["sequences"]))
    out = []
    for i in range(case["sequences"]):
        part, piece = (1.0, 1.0) if i == 0 else (rng.uniform(0.25, 1.0), rng.uniform(0.5, 1.0))
        nodes = max(1, round(case["nodes"] * piece))
        if case["kind"] == "tree":
            out.append((round(case["context"] * part), nodes))
        else:                       # the shared prompt and a few tokens of the sequence's own
            out.append((SHARED + rng.randint(0, 15), nodes))
    return out


def _tree(rng, nodes):
    """Parents of a tree in the order of depth, its levels as wide as a draft head's: a chain up
    to five nodes, then up to six levels."""
    width = 1 if nodes <= 5 else -(-(nodes - 1) // min(6, 1 + nodes // 4))
    parents, last = [-1], [0]
    while len(parents) < nodes:
        here = sorted(rng.choice(last) for _ in range(min(width, nodes - len(parents))))
        last = list(range(len(parents), len(parents) + len(here)))
        parents += here
    return parents


def _ancestors(parents, i):
    """Node i and its ancestors, from the root."""
    path = [i]
    while parents[path[-1]] >= 0:
        path.append(parents[path[-1]])
    return path[::-1]


def _accepted(rng, parents):
    """A node up to which the model agrees with the draft: one whose path either has every node in
    its place already or moves only nodes from behind the places that it fills."""
    for i in rng.sample(range(len(parents)), len(parents)):
        path = _ancestors(parents, i)
        if all(p == at or p >= len(path) for at, p in enumerate(path)):
            return i
    return 0


def _codes(rows, kv):
    """[..., 64] bf16 rows -> (codes, scale bytes) uint8."""
    x = rows.float()
    e = (x.abs().amax(-1).view(torch.int32) >> 23) & 255
    s = (e - 7).clamp(min=10, max=246)
    return (x * torch.exp2(127.0 - s.float())[..., None]).to(FP8).view(torch.uint8), s.to(torch.uint8)


def _fill(g, pages, cache, layers=None):
    """A cache of random rows: [pages, ...], or [layers, pages, ...]."""
    n = pages * (layers or 1)
    shape = (n, 2, KVH, PAGE, DIM) if cache == "bf16" else (n, PAGE_BYTES)
    out = torch.empty(shape, dtype=BF if cache == "bf16" else torch.uint8, device=DEV)
    gain = torch.exp(_normal(g, (KVH, 1, DIM), 0.5))
    for part in out.split(4096):
        p = part.shape[0]
        k = (_normal(g, (p, KVH, PAGE, DIM)) * gain).to(BF)
        v = (_normal(g, (p, KVH, PAGE, DIM)) * torch.exp(_normal(g, (p, 1, PAGE, 1), 0.5))).to(BF)
        if cache == "bf16":
            part[:, 0], part[:, 1] = k, v
            continue
        kc, vc, sc = _parts(part)
        kc[:], sc[:, :, 0] = _codes(k, 0)
        codes, sc[:, :, 1] = _codes(v, 1)
        vc[:] = codes.view(p, KVH, PAGE // 4, 4, 4, DIM // 4).permute(0, 1, 2, 5, 4, 3)
    return out if layers is None else out.unflatten(0, (layers, pages))


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _trees(case, seed, lengths, x):
    """Each sequence's tree, packed one after the other: parents, tokens, what the model chose,
    the mask and the positions."""
    rng = random.Random("%d %d %d" % (seed, case["sequences"], case["nodes"]))
    parents, tokens, chosen, masks, positions, starts = [], [], [], [], [], [0]
    words = -(-max(m for _, m in lengths) // 32)
    for c, m in lengths:
        mine = _tree(rng, m)
        token = [rng.randrange(VOCAB) for _ in mine]
        choice = [rng.randrange(VOCAB) for _ in mine]
        path = _ancestors(mine, _accepted(rng, mine))
        for at, child in zip(path, path[1:]):
            choice[at] = token[child]
        for i in range(m):
            up = _ancestors(mine, i)
            bits = sum(1 << j for j in up)
            masks.append([(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
            positions.append(c + len(up) - 1)
        parents += mine
        tokens += token
        chosen += choice
        starts.append(starts[-1] + m)
    x["parents"], x["tokens"], x["chosen"] = _int(parents), _int(tokens), _int(chosen)
    x["positions"], x["q_indptr"] = _int(positions), _int(starts)
    x["tree_mask"] = torch.from_numpy(np.array(masks, dtype=np.uint32).view(np.int32)).to(DEV)


def _inputs(case, seed):
    """The tensors in hand before a call, the sequences' pages scattered over the pool."""
    kind, g = case["kind"], _gen(seed, 1)
    x = {"kind": kind}
    if kind == "beams":
        n, b, w = case["requests"], case["beams"], case["vocab"]
        logits = _normal(g, (n * b, w), 2.5)
        # a few tokens that the text makes likely, and some that a filter has ruled out
        likely = torch.randint(0, w, (n * b, 12), generator=g, device=DEV)
        logits.scatter_add_(1, likely, torch.rand((n * b, 12), generator=g, device=DEV) * 9.0)
        out = torch.randint(0, w, (n * b, 20), generator=g, device=DEV)
        logits.scatter_(1, out, -math.inf)
        x["logits"] = logits.to(BF if case["type"] == "bf16" else F32)
        x["scores"] = -20.0 * torch.rand((n, b), generator=g, device=DEV).sort(1)[0]
        x["k"] = case["k"]
        return x
    if kind == "pages":
        n = case["pages"]
        x["cache"] = _fill(g, 2 * n + 1, case["cache"], case["layers"])
        ids = torch.randperm(2 * n + 1, generator=g, device=DEV).int()
        # two or three children of a parent
        x["src"] = ids[:n][torch.div(torch.arange(n, device=DEV), 2, rounding_mode="floor")]
        x["dst"] = ids[n:2 * n].contiguous()
        return x
    lengths = _lengths(case)
    x["lengths"] = lengths
    indptr, used = [0], 0
    for c, m in lengths:
        used += -(-(c + m) // PAGE)
        indptr.append(used)
    x["page_indptr"] = _int(indptr)
    x["kv_len"] = _int([c + m for c, m in lengths])
    x["max_q"], x["max_kv"] = max(m for _, m in lengths), max(c + m for c, m in lengths)
    _trees(case, seed, lengths, x)
    if kind == "tree":
        pool = used + 5
        x["page_indices"] = torch.randperm(pool, generator=g, device=DEV)[:used].int()
        x["cache"] = _fill(g, pool, case["cache"])
        n = sum(m for _, m in lengths)
        x["q"] = _normal(g, (n, QH, DIM), 2.0).to(BF)
        x["sinks"] = _normal(g, (QH,)).to(BF)
        return x
    # every sequence begins with the shared prompt's pages
    shared = SHARED // PAGE
    pool = shared + sum(-(-(c + m) // PAGE) - shared for c, m in lengths)
    ids = torch.randperm(pool, generator=g, device=DEV).int()
    parts, at = [], shared
    for c, m in lengths:
        mine = -(-(c + m) // PAGE) - shared
        parts += [ids[:shared], ids[at:at + mine]]
        at += mine
    x["page_indices"] = torch.cat(parts)
    x["cache"] = _fill(g, pool, case["cache"], case["layers"])
    return x


def prepare(case, seed):
    with torch.no_grad():
        x = _inputs(case, seed)
        if x["kind"] == "tree":
            x["window"] = WINDOW if case["window"] else 0
            x["out"] = torch.empty_like(x["q"])
        if x["kind"] in ("tree", "commit"):
            # where each packed row lies: its sequence and its place there
            starts = x["q_indptr"].long()
            n = x["parents"].numel()
            x["row_seq"] = torch.searchsorted(starts[1:].contiguous(), torch.arange(n, device=DEV),
                                              right=True)
            x["row_node"] = torch.arange(n, device=DEV) - starts[x["row_seq"]]
        return x


# -- one pass ------------------------------------------------------------------------------

def run(x):
    with torch.no_grad():
        return _run_own(x) if own else _PLAIN[x["kind"]](x)


def _run_own(x):
    a, kind = _native(), x["kind"]
    if kind == "beams":
        return a.beam_top_k(x["logits"], x["scores"], x["k"])
    if kind == "pages":
        return a.kv_copy_pages(x["cache"], x["src"], x["dst"])
    if kind == "commit":
        return (*a.tree_commit(x["cache"], x["page_indptr"], x["page_indices"], x["kv_len"],
                               x["q_indptr"], x["max_q"], x["tokens"], x["parents"], x["chosen"]),
                x["cache"])
    tree = a.tree if x["cache"].dtype == BF else a.tree_fp8
    return tree(x["q"], x["q_indptr"], x["max_q"], x["tree_mask"], x["positions"], x["cache"],
                x["page_indptr"], x["page_indices"], x["kv_len"], x["window"], SCALE, x["sinks"],
                x["out"], x["max_kv"])


# -- the plain forms ---------------------------------------------------------------------------

def _parts(cache):
    """Views of an 8-bit cache's pages: codes of k and of v, scales."""
    return (cache[..., :CODES].unflatten(-1, (KVH, PAGE, DIM)),
            cache[..., CODES:2 * CODES].unflatten(-1, (KVH, PAGE // 4, DIM // 4, 4, 4)),
            cache[..., 2 * CODES:].unflatten(-1, (KVH, 2, PAGE)))


def _rows(cache, page, at):
    """k, v [..., 8, 64] fp32 of the rows at pages and places [...]."""
    if cache.dtype == BF:
        return cache[page, 0, :, at].float(), cache[page, 1, :, at].float()
    kc, vc, sc = _parts(cache)
    s = torch.exp2(sc[page, :, :, at].float() - 127.0)
    v = vc[page, :, at // 4, :, :, at % 4].transpose(-1, -2).flatten(-2)
    return (kc[page, :, at].view(FP8).float() * s[..., 0, None],
            v.contiguous().view(FP8).float() * s[..., 1, None])


def _seen_nodes(x):
    """[sequences, nodes, nodes] bool: node i sees node j."""
    b, m = x["kv_len"].numel(), x["max_q"]
    j = torch.arange(m, device=DEV)
    bits = (x["tree_mask"][:, j // 32] >> (j % 32).int()) & 1
    out = torch.zeros((b, m, m), dtype=torch.bool, device=DEV)
    out[x["row_seq"], x["row_node"]] = bits != 0
    return out


def _plain_tree(x):
    b, m, longest = x["kv_len"].numel(), x["max_q"], x["max_kv"]
    total, starts = x["kv_len"].long(), x["q_indptr"].long()
    cached = total - (starts[1:] - starts[:-1])
    t = torch.arange(longest, device=DEV)
    # every sequence's keys up to the longest's; what lies past its own is hidden
    first = x["page_indptr"].long()[:-1, None]
    index = torch.minimum(t[None, :], total[:, None] - 1) // PAGE
    k, v = _rows(x["cache"], x["page_indices"].long()[first + index], (t % PAGE).expand(b, -1))
    k = k.permute(0, 2, 3, 1).reshape(b * KVH, DIM, longest)
    v = v.masked_fill((t >= total[:, None])[..., None, None], 0.0)
    v = v.permute(0, 2, 1, 3).reshape(b * KVH, longest, DIM)
    q = torch.zeros((b, m, QH, DIM), device=DEV)
    at = torch.zeros((b, m), dtype=torch.long, device=DEV)
    q[x["row_seq"], x["row_node"]] = x["q"].float()
    at[x["row_seq"], x["row_node"]] = x["positions"].long()
    node = t[None, :] - cached[:, None]                           # the key's node, if it is one
    inside = node.clamp(0, m - 1)
    seen = _seen_nodes(x).gather(2, inside[:, None, :].expand(-1, m, -1))
    seen = torch.where(node[:, None, :] < 0, True, seen & (t < total[:, None])[:, None, :])
    if x["window"]:
        place = torch.where(node < 0, t[None, :], at.gather(1, inside))
        seen = seen & (place[:, None, :] > at[:, :, None] - x["window"])
    q = q.view(b, m, KVH, GROUP, DIM).permute(0, 2, 3, 1, 4).reshape(b * KVH, GROUP * m, DIM)
    s = (torch.matmul(q, k) * SCALE).view(b, KVH, GROUP, m, longest)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    sinks = x["sinks"].float().view(1, KVH, GROUP, 1, 1)
    top = torch.maximum(s.amax(-1, keepdim=True), sinks)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True) + torch.exp(sinks - top)
    o = torch.matmul(p.view(b * KVH, GROUP * m, longest), v).view(b, KVH, GROUP, m, DIM) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, m, QH, DIM)
    return o[x["row_seq"], x["row_node"]].to(BF)


def _plain_commit(x):
    cache, seq, node = x["cache"], x["row_seq"], x["row_node"]
    b, m = x["kv_len"].numel(), x["max_q"]
    starts = x["q_indptr"].long()
    cached = x["kv_len"].long() - (starts[1:] - starts[:-1])
    parent = starts[seq] + x["parents"].long().clamp(min=0)
    # a node is accepted where it and all its ancestors are what the model chose
    good = torch.zeros((b, m), dtype=torch.bool, device=DEV)
    good[seq, node] = (x["chosen"][parent] == x["tokens"]) | (node == 0)
    real = torch.zeros((b, m), dtype=torch.bool, device=DEV)
    real[seq, node] = True
    taken = real & (good[:, None, :] | ~_seen_nodes(x)).all(-1)
    count = taken.sum(1)
    j = torch.arange(m, device=DEV)
    path = torch.where(taken, j, m).sort(1)[0]
    path = torch.where(path < m, path, -1)
    last = path.gather(1, (count - 1)[:, None])[:, 0]
    chosen = x["chosen"][starts[:-1] + last]
    sb, si = torch.nonzero((path >= 0) & (path != j), as_tuple=True)
    first = x["page_indptr"].long()[sb]
    src, dst = cached[sb] + path[sb, si], cached[sb] + si
    pages = x["page_indices"].long()
    sp, dp, sa, da = pages[first + src // PAGE], pages[first + dst // PAGE], src % PAGE, dst % PAGE
    if cache.dtype == BF:
        cache[:, dp, :, :, da] = cache[:, sp, :, :, sa]
    else:
        kc, vc, sc = _parts(cache)
        kc[:, dp, :, da] = kc[:, sp, :, sa]
        vc[:, dp, :, da // 4, :, :, da % 4] = vc[:, sp, :, sa // 4, :, :, sa % 4]
        sc[:, dp, :, :, da] = sc[:, sp, :, :, sa]
    return path[seq, node].int(), count.int(), chosen, cache


def _plain_beams(x):
    # in 64 bits: which of two near candidates comes first hangs on their last bits
    n, b = x["scores"].shape
    v = x["logits"].double()
    top = v.amax(-1, keepdim=True)
    total = torch.log(torch.exp(v - top).sum(-1, keepdim=True))
    score = x["scores"].double().view(n * b, 1) + ((v - top) - total)
    score = torch.where(torch.isnan(score), -math.inf, score).view(n, -1)
    value, index = torch.sort(score, dim=1, descending=True, stable=True)
    value, index, w = value[:, :x["k"]], index[:, :x["k"]], v.shape[1]
    beam = torch.div(index, w, rounding_mode="floor")
    return value.float(), beam.int(), (index - beam * w).int()


def _plain_pages(x):
    x["cache"][:, x["dst"].long()] = x["cache"][:, x["src"].long()]
    return x["cache"]


_PLAIN = {"tree": _plain_tree, "commit": _plain_commit, "beams": _plain_beams,
          "pages": _plain_pages}


# -- what a pass cannot do without -------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "beams":
        rows = case["requests"] * case["beams"]
        n = rows * case["vocab"]
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + rows * 4
                + case["requests"] * case["k"] * 12, "flops": 3.0 * n}
    page = BF_PAGE_BYTES if case["cache"] == "bf16" else PAGE_BYTES
    if kind == "pages":
        return {"bytes": case["layers"] * (-(-case["pages"] // 2) + case["pages"]) * page
                + 8 * case["pages"], "flops": 0.0}
    lengths = _lengths(case)
    row = page // PAGE
    n = sum(m for _, m in lengths)
    if kind == "commit":
        # a tree's path has a fifth of its nodes on average, about half of which move
        return {"bytes": n * 16 + case["layers"] * max(1, n // 10) * 2 * row, "flops": float(n)}
    window = WINDOW if case["window"] else 0
    depth = 6                                 # nodes that a node of a tree sees, about
    pairs = sum(m * ((min(c, window) if window else c) + min(m, depth)) for c, m in lengths)
    keys = sum((min(c, window) if window else c) + m for c, m in lengths)
    return {"bytes": keys * row + n * (QH * DIM * 4 + 8), "flops": pairs * QH * 4.0 * DIM}


# -- the same in 64 bits, apart from the forms above ---------------------------------------------

def _values(cache, pages, kv):
    """Keys (kv 0) or values (1) of whole pages, [tokens, 8, 64] float64."""
    mine = cache[pages]
    p = mine.shape[0]
    if cache.dtype == BF:
        return mine[:, kv].double().permute(0, 2, 1, 3).reshape(p * PAGE, KVH, DIM)
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    value = np.where(e == 0, f / 8.0 * 2.0 ** -6, (1 + f / 8.0) * np.exp2(e - 7.0))
    value = np.where((c & 127) == 127, np.nan, np.where(c & 128, -value, value))
    table = torch.from_numpy(value).to(DEV)
    scale = torch.exp2(mine[:, 2 * CODES:].view(p, KVH, 2, PAGE)[:, :, kv].double() - 127.0)
    codes = mine[:, kv * CODES:(kv + 1) * CODES].int()
    if kv == 0:
        r = table[codes].view(p, KVH, PAGE, DIM)
    else:
        r = table[codes].view(p, KVH, 4, 16, 4, 4).permute(0, 1, 2, 5, 4, 3)
        r = r.reshape(p, KVH, PAGE, DIM)
    return (r * scale[..., None]).permute(0, 2, 1, 3).reshape(p * PAGE, KVH, DIM)


def exact(case, seed):
    kind = case["kind"]
    with torch.no_grad():
        x = _inputs(case, seed)
        if kind == "beams":
            n, b = x["scores"].shape
            best = []
            for r in range(n):
                rows = x["logits"][r * b:(r + 1) * b].double()
                lse = torch.logsumexp(rows, dim=1, keepdim=True)
                s = (rows - lse + x["scores"][r].double()[:, None]).flatten()
                best.append(torch.topk(s, x["k"]).values)
            return torch.stack(best), None, None
        if kind == "pages":
            if x["cache"].dtype != BF:
                return None
            want = x["cache"].double()
            for s, d in zip(x["src"].tolist(), x["dst"].tolist()):
                want[:, d] = want[:, s]
            return want
        starts, parents = x["q_indptr"].tolist(), x["parents"].tolist()
        pages, indptr = x["page_indices"].tolist(), x["page_indptr"].tolist()
        if kind == "commit":
            if x["cache"].dtype != BF:
                return None
            want, tokens, chosen = x["cache"].double(), x["tokens"].tolist(), x["chosen"].tolist()
            for i, (c, m) in enumerate(x["lengths"]):
                at, path = 0, [0]
                while True:
                    after = [j for j in range(m) if parents[starts[i] + j] == at
                             and tokens[starts[i] + j] == chosen[starts[i] + at]]
                    if not after:
                        break
                    at = after[0]
                    path.append(at)
                for to, node in enumerate(path):
                    s, d = c + node, c + to
                    sp, dp = pages[indptr[i] + s // PAGE], pages[indptr[i] + d // PAGE]
                    want[:, dp, :, :, d % PAGE] = want[:, sp, :, :, s % PAGE]
            return None, None, None, want
        window, out = WINDOW if case["window"] else 0, []
        positions = x["positions"].tolist()
        for i, (c, m) in enumerate(x["lengths"]):
            mine = x["page_indices"][indptr[i]:indptr[i + 1]].long()
            seen = torch.zeros((m, c + m), dtype=torch.bool)
            seen[:, :c] = True
            pos = positions[starts[i]:starts[i + 1]]
            for node in range(m):
                for up in _ancestors(parents[starts[i]:starts[i + 1]], node):
                    seen[node, c + up] = True
            where = torch.tensor(list(range(c)) + pos)
            if window:
                seen &= where[None, :] > torch.tensor(pos)[:, None] - window
            seen = seen.to(DEV)
            k = _values(x["cache"], mine, 0)[:c + m]
            v = _values(x["cache"], mine, 1)[:c + m]
            q = x["q"][starts[i]:starts[i + 1]].double()
            heads = []
            for h in range(QH):
                s = q[:, h] @ k[:, h // GROUP].t() / 8.0
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                lse = torch.logsumexp(s, dim=1, keepdim=True)
                o = torch.exp(s - lse) @ v[:, h // GROUP]
                heads.append(o * torch.sigmoid(lse - x["sinks"][h].double()))
            out.append(torch.stack(heads, dim=1))
        return torch.cat(out)
