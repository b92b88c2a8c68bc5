"""Paged KV cache for the attention block (host side).

Mirrors the part of mlc-llm's PagedKVCache the reference drives
(engine.py:41-53,97-131,133-174; model/transformer.py:153-175): sequences
are added, optionally given a sliding window, extended by ``begin_forward``
with the number of tokens each one appends, and shortened by ``popn``.  The
data live on the GPU in one bf16 tensor [layers, pages, 2 (k, v), kv_heads,
16, head_dim] (mlc's per-layer page layout, stacked), pages of 16 tokens
shared by all layers of a sequence, allocated from a free list.

``begin_forward`` builds the tables the kernels read -- each sequence's page
list, its length after the append, the positions and cache slots of the
appended tokens -- and copies them into device buffers allocated once at
construction, so the forward itself allocates nothing and can be captured in
a HIP graph (the tables are inputs of the graph: refresh them with
``begin_forward`` before each replay; ``static_span`` fixes the decode
attention's split count at the pool's capacity for a captured forward, whose
empty splits return at once and merge to the same result).

Sliding window: the reference's cache keeps only the window's pages for its
"mha_sliding" layers; this cache keeps every token and the kernels attend to
the last ``window`` positions in those layers, which gives the same result
with one page table for all layers.

With ``dtype=torch.float8_e4m3fn`` the cache holds 8-bit rows with a scale byte
each (the format of include/attn_gfx950.h): one uint8 tensor [layers, pages,
16640], half a bf16 cache's bytes, quantised as it is written and read by the
8-bit attention kernels.  The tables are the same.

Sequences may share pages: ``branch`` lets several go on from what one holds (beams), at
no cost but the page lists'.  A page that others hold too and that a forward would write to is
copied first, in all layers by one launch.  A forward lists a shared page once a sequence, so its
lists may be longer than the pool: the tables have room for ``max_listed`` entries (by default a
whole pool a sequence, up to 2^22 more than the pool has), and a forward that lists more is refused.

``begin_tree`` appends a tree of drafted tokens to each sequence in place of a chunk: the tables
then also have each node's mask over its tree, and positions by depth.  Masks and parents are new
tensors, built on the host in each call: a forward of trees is not for capture in a graph.
"""
from __future__ import annotations

import dataclasses
from collections import Counter

import numpy as np
import torch

PAGE_SIZE = 16
FP8_PAGE_BYTES = 16640  # of a page of an 8-bit cache
SHARED_LISTED = 1 << 22  # entries of a forward's page lists beyond the pool's size
STAGED = 64             # tokens of the largest fused decode projection
TREE_MAX_NODES = 1024   # of a sequence's tree of drafted tokens


@dataclasses.dataclass
class _Seq:
    length: int = 0
    pages: list = dataclasses.field(default_factory=list)
    window: int = 0


@dataclasses.dataclass
class ForwardTables:
    """Device tables of one forward (views into the cache's buffers)."""
    batch: int
    num_tokens: int
    max_q_len: int
    max_kv_len: int
    q_indptr: torch.Tensor      # [batch + 1] int32
    positions: torch.Tensor     # [num_tokens] int32
    slots: torch.Tensor         # [num_tokens] int32 (page * 16 + offset)
    page_indptr: torch.Tensor   # [batch + 1] int32
    page_indices: torch.Tensor  # [pages] int32
    kv_len: torch.Tensor        # [batch] int32
    windows: tuple              # per sequence: sliding window (0 = none)
    # of a forward of trees: bit j % 32 of word j / 32, node i sees node j of its sequence;
    # each node's parent in its tree (-1: the root)
    tree_mask: torch.Tensor | None = None  # [num_tokens, words] int32
    parents: torch.Tensor | None = None    # [num_tokens] int32

    @property
    def is_decode(self) -> bool:
        return self.max_q_len == 1 and self.tree_mask is None


class PagedKVCache:
    def __init__(self, num_layers: int, num_pages: int, max_batch: int, max_tokens: int,
                 kv_heads: int = 8, head_dim: int = 64, device="cuda",
                 dtype=torch.bfloat16, max_listed: int | None = None):
        self.num_layers = num_layers
        self.num_pages = num_pages
        self.max_batch = max_batch
        self.max_tokens = max_tokens
        if max_listed is None:
            max_listed = min(max_batch * num_pages, num_pages + SHARED_LISTED)
        self.max_listed = max(max_listed, num_pages)  # (without sharing it is never more)
        self.fp8 = dtype == torch.float8_e4m3fn
        if self.fp8:
            if (kv_heads, head_dim) != (8, 64):
                raise ValueError("the 8-bit cache is built for 8 key/value heads of 64")
            self.data = torch.zeros((num_layers, num_pages, FP8_PAGE_BYTES), dtype=torch.uint8,
                                    device=device)
            # where the fused decode projections append a step's bf16 rows, to be quantised
            # from there (every layer in turn, on one stream)
            self.staging = torch.zeros((STAGED // PAGE_SIZE, 2, kv_heads, PAGE_SIZE, head_dim),
                                       dtype=torch.bfloat16, device=device)
            self.staging_slots = torch.arange(STAGED, dtype=torch.int32, device=device)
        elif dtype.is_floating_point and dtype.itemsize == 1:
            raise ValueError(f"a cache holds bf16 or float8_e4m3fn rows, not {dtype}")
        else:
            self.data = torch.zeros((num_layers, num_pages, 2, kv_heads, PAGE_SIZE, head_dim),
                                    dtype=dtype, device=device)
        self.free = list(range(num_pages - 1, -1, -1))  # pop() hands out page 0 first
        self._refs = [0] * num_pages                     # sequences that hold a page
        self.seqs: dict[int, _Seq] = {}
        # The forward tables live in one device buffer at fixed offsets (kernels
        # captured in a graph keep their addresses), uploaded from a pinned
        # staging buffer of the same layout.  A forward of at most max_batch
        # tokens (every decode step) keeps its positions and slots in short
        # arrays ahead of the page indices, so its tables are one contiguous
        # range and one copy; a longer forward uses the long arrays at the end
        # (three copies, each spanning only what the forward uses).  Last the pages that a
        # forward copies before it writes to them, sources and then destinations.
        sizes = (max_batch + 1, max_batch + 1, max_batch, max_batch, max_batch, self.max_listed,
                 max_tokens, max_tokens, 2 * max_batch)
        self._tables_dev = torch.zeros(sum(sizes), dtype=torch.int32, device=device)
        # two staging buffers used in turn: a forward waits only for the copy
        # made from its buffer two forwards ago (an event), not for the stream
        self._pinned = [torch.zeros(sum(sizes), dtype=torch.int32,
                                    pin_memory=torch.cuda.is_available()) for _ in range(2)]
        self._stage_events: list = [None, None]
        self._stage = 0
        self._table_offsets, views, off = [], [], 0
        for k in sizes:
            self._table_offsets.append(off)
            views.append(self._tables_dev[off:off + k])
            off += k
        (self._q_indptr, self._page_indptr, self._kv_len, self._positions_short,
         self._slots_short, self._page_indices, self._positions, self._slots,
         self._copies) = views
        self.tables: ForwardTables | None = None
        self._decode_ws: torch.Tensor | None = None
        self._decode_ws_held: list = []
        # decode attention's key bound for a captured forward (0: per forward)
        self.static_span = 0

    def decode_workspace(self, batch: int, span: int) -> torch.Tensor:
        """The decode attention's split buffers for `batch` sequences attending
        to at most `span` keys; grown here only (``reserve_decode`` sizes it
        up front for callers that capture the forward in a graph)."""
        import attn_native
        size, make = ((attn_native.decode_fp8_workspace_bytes, attn_native.decode_fp8_workspace)
                      if self.fp8 else
                      (attn_native.decode_workspace_bytes, attn_native.decode_workspace))
        if self._decode_ws is None or self._decode_ws.numel() < size(batch, span):
            # a buffer a captured graph holds stays alive in _decode_ws_held
            self._decode_ws = make(batch, span, self.data.device)
        return self._decode_ws

    def reserve_decode(self, batch: int, span: int, for_graph: bool = False) -> None:
        """Size the decode workspace now.  With ``for_graph`` the buffer is
        kept alive as long as the cache: a graph captured after this call
        holds its address, and a later, larger call gets a new buffer rather
        than freeing the captured one."""
        ws = self.decode_workspace(batch, span)
        if for_graph and all(h is not ws for h in self._decode_ws_held):
            self._decode_ws_held.append(ws)

    # -- sequences (vm.builtin.kv_state_* of engine.py:41-53) -------------------
    def layer(self, i: int) -> torch.Tensor:
        return self.data[i]

    def add_sequence(self, seq_id: int) -> None:
        if seq_id in self.seqs:
            raise ValueError(f"sequence {seq_id} exists")
        self.seqs[seq_id] = _Seq()

    def enable_sliding_window(self, seq_id: int, window: int, sink_size: int = 0) -> None:
        if sink_size:
            raise ValueError("attention sinks in the cache (sink_size > 0) are not supported; "
                             "the reference runs with 0 (engine.py:62, 120)")
        self.seqs[seq_id].window = int(window)

    def _take(self) -> int:
        page = self.free.pop()
        self._refs[page] = 1
        return page

    def _drop(self, pages) -> None:
        for page in reversed(pages):
            self._refs[page] -= 1
            if self._refs[page] == 0:
                self.free.append(page)

    def remove_sequence(self, seq_id: int) -> None:
        self._drop(self.seqs.pop(seq_id).pages)

    def branch(self, seq_ids, parents, new_ids=None) -> None:
        """Sequence ``new_ids[i]`` goes on from what ``seq_ids[parents[i]]`` holds, sharing its
        pages; the sequences ``seq_ids`` end (``new_ids``, by default the first of them, may
        name them again)."""
        seq_ids, parents = list(seq_ids), [int(p) for p in parents]
        new_ids = seq_ids[:len(parents)] if new_ids is None else list(new_ids)
        if len(new_ids) != len(parents) or len(set(new_ids)) != len(new_ids):
            raise ValueError(f"{len(parents)} branches need as many different sequences, "
                             f"not {new_ids}")
        if len(set(seq_ids)) != len(seq_ids) or any(s not in self.seqs for s in seq_ids):
            raise ValueError(f"sequences {seq_ids} are not all there, or not different")
        if any(not 0 <= p < len(seq_ids) for p in parents):
            raise ValueError(f"parents {parents} of {len(seq_ids)} sequences")
        taken = [s for s in new_ids if s in self.seqs and s not in seq_ids]
        if taken:
            raise ValueError(f"sequence {taken[0]} exists")
        old = [self.seqs.pop(s) for s in seq_ids]
        for sid, p in zip(new_ids, parents):
            self.seqs[sid] = _Seq(old[p].length, list(old[p].pages), old[p].window)
            for page in old[p].pages:
                self._refs[page] += 1
        for s in old:
            self._drop(s.pages)

    def clear(self) -> None:
        for sid in list(self.seqs):
            self.remove_sequence(sid)

    def popn(self, seq_id: int, n: int) -> None:
        s = self.seqs[seq_id]
        if not 0 <= n <= s.length:
            raise ValueError(f"popn({n}) on a sequence of {s.length} tokens")
        s.length -= n
        keep = -(-s.length // PAGE_SIZE)
        self._drop(s.pages[keep:])
        del s.pages[keep:]

    def total_sequence_length(self) -> int:
        return sum(s.length for s in self.seqs.values())

    def seq_len(self, seq_id: int) -> int:
        return self.seqs[seq_id].length

    # -- a sequence's rows -----------------------------------------------------------
    def slots_of(self, seq_id: int, start: int = 0, stop: int | None = None) -> torch.Tensor:
        """The cache slots (page * 16 + offset) of a sequence's tokens start .. stop - 1."""
        s = self.seqs[seq_id]
        stop = s.length if stop is None else stop
        if not 0 <= start <= stop <= s.length:
            raise ValueError(f"tokens {start}..{stop} of a sequence of {s.length}")
        return torch.tensor([s.pages[p // PAGE_SIZE] * PAGE_SIZE + p % PAGE_SIZE
                             for p in range(start, stop)], dtype=torch.int32,
                            device=self.data.device)

    def read(self, seq_id: int, layer: int, start: int = 0,
             stop: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """k and v [n, kv_heads, head_dim] of a sequence's tokens start .. stop - 1 in one layer
        (an 8-bit cache's as the bf16 values that its rows stand for)."""
        slots = self.slots_of(seq_id, start, stop)
        if self.fp8:
            import attn_native
            return attn_native.kv_read_fp8(self.layer(layer), slots)
        page, at = slots.long() // PAGE_SIZE, slots.long() % PAGE_SIZE
        data = self.layer(layer)
        return data[page, 0, :, at], data[page, 1, :, at]

    def quantize_from(self, seq_id: int, source: "PagedKVCache", source_id: int) -> None:
        """A new sequence ``seq_id`` of this 8-bit cache with the tokens and the window of
        ``source_id`` of a bf16 cache of as many layers: its rows quantised, in every layer."""
        import attn_native
        if (not self.fp8 or source.data.dtype != torch.bfloat16
                or source.data.shape[2:] != self.staging.shape[1:]
                or source.num_layers != self.num_layers
                or source.data.device != self.data.device):
            raise ValueError("quantize_from takes a sequence of a bf16 cache into an 8-bit cache "
                             "of as many layers and the same heads on the same device")
        old = source.seqs[source_id]
        need = -(-old.length // PAGE_SIZE)
        if need > len(self.free):
            raise MemoryError(f"KV cache full: {need} pages needed, {len(self.free)} free")
        self.add_sequence(seq_id)
        s = self.seqs[seq_id]
        s.pages = [self._take() for _ in range(need)]
        s.length, s.window = old.length, old.window
        try:
            if s.length:
                mine, theirs = self.slots_of(seq_id), source.slots_of(source_id)
                for i in range(self.num_layers):
                    attn_native.kv_quantize_fp8(source.layer(i), theirs, self.layer(i), mine)
        except Exception:  # its rows are not there: no sequence
            self.remove_sequence(seq_id)
            raise

    def _copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        if self.data.is_cuda and (self.fp8 or self.data.dtype == torch.bfloat16):
            import attn_native
            attn_native.kv_copy_pages(self.data, src, dst)
        else:
            self.data[:, dst.long()] = self.data[:, src.long()]

    # -- one forward ---------------------------------------------------------------
    def _shares_last(self, s: _Seq) -> bool:
        """Whether a sequence's next token goes to a page that others hold too."""
        return s.length % PAGE_SIZE != 0 and self._refs[s.pages[-1]] > 1

    def begin_tree(self, seq_ids, parents) -> ForwardTables:
        """``begin_forward`` for a tree of drafted tokens each: ``parents[i]`` lists its nodes'
        parents within the tree, -1 first (the last sampled token) and every other one
        before its node.  Nodes lie one after the other behind the cached tokens; a node's
        position is the number of those plus its depth.  ``popn`` takes back what is not
        accepted, after ``attn_native.tree_commit`` has moved what is."""
        parents = [[int(p) for p in tree] for tree in parents]
        seq_ids = list(seq_ids)
        if len(seq_ids) != len(parents) or len(set(seq_ids)) != len(seq_ids):
            raise ValueError(f"{len(parents)} trees need as many different sequences, not {seq_ids}")
        longest = max((len(tree) for tree in parents), default=0)
        words = max(1, -(-longest // 32))
        if longest > TREE_MAX_NODES:
            raise ValueError(f"a tree of {longest} nodes, at most {TREE_MAX_NODES}")
        depths, masks = [], []
        for sid, tree in zip(seq_ids, parents):
            if tree[:1] != [-1] or any(not 0 <= p < i for i, p in enumerate(tree) if i):
                raise ValueError("a tree's nodes come after their parents, the root (-1) first")
            depth, sees = [0] * len(tree), [1] * len(tree)
            for i, p in enumerate(tree):
                if i:
                    depth[i], sees[i] = depth[p] + 1, sees[p] | 1 << i
            depths.append(depth)
            masks += [[(x >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for x in sees]
        flat = np.array([p for tree in parents for p in tree], dtype=np.int32)
        mask = np.array(masks, dtype=np.uint32).view(np.int32).reshape(-1, words)
        flat, mask = (torch.from_numpy(x).to(self.data.device) for x in (flat, mask))
        tables = self.begin_forward(seq_ids, [len(tree) for tree in parents], depths)
        tables.parents, tables.tree_mask = flat, mask
        return tables

    def begin_forward(self, seq_ids, append_lengths, depths=None) -> ForwardTables:
        """Append ``append_lengths[i]`` tokens to sequence ``seq_ids[i]``
        (pages allocated as needed) and upload the tables of this forward.  ``depths[i]``: the
        tokens' positions behind the sequence's end, where they do not follow one another."""
        seq_ids, append_lengths = list(seq_ids), [int(a) for a in append_lengths]
        batch, n = len(seq_ids), sum(append_lengths)
        if batch > self.max_batch or n > self.max_tokens:
            raise ValueError(f"forward of {batch} sequences / {n} tokens exceeds the cache's "
                             f"{self.max_batch} / {self.max_tokens}")
        if min(append_lengths, default=1) < 1:
            raise ValueError("every sequence of a forward appends at least one token")
        grown, listed = {}, 0  # the sequences' lengths, and the page lists' entries
        for s, a in zip(seq_ids, append_lengths):
            grown[s] = grown.get(s, self.seqs[s].length) + a
            listed += -(-grown[s] // PAGE_SIZE)
        if listed > self.max_listed:
            raise MemoryError(f"the forward's sequences list {listed} pages, the cache's tables "
                              f"have room for {self.max_listed} (max_listed)")
        need = sum(max(0, -(-n // PAGE_SIZE) - len(self.seqs[s].pages)) for s, n in grown.items())
        # a copy for each that writes to a shared page; the last of its holders keeps it
        writers = [self.seqs[s].pages[-1] for s in grown if self._shares_last(self.seqs[s])]
        if writers:
            need += sum(w - (w == self._refs[page]) for page, w in Counter(writers).items())
        if need > len(self.free):
            raise MemoryError(f"KV cache full: {need} pages needed, {len(self.free)} free")
        q_indptr, positions, slots, page_indptr, page_indices, kv_len = [0], [], [], [0], [], []
        copies = []
        for i, (sid, a) in enumerate(zip(seq_ids, append_lengths)):
            s = self.seqs[sid]
            if writers and self._shares_last(s):  # others keep that page
                shared = s.pages[-1]
                s.pages[-1] = self._take()
                self._drop([shared])
                copies.append((shared, s.pages[-1]))
            while len(s.pages) * PAGE_SIZE < s.length + a:
                s.pages.append(self._take())
            positions.extend(range(s.length, s.length + a) if depths is None
                             else (s.length + d for d in depths[i]))
            for p in range(s.length, s.length + a):
                slots.append(s.pages[p // PAGE_SIZE] * PAGE_SIZE + p % PAGE_SIZE)
            s.length += a
            q_indptr.append(q_indptr[-1] + a)
            page_indices.extend(s.pages)
            page_indptr.append(len(page_indices))
            kv_len.append(s.length)
        j = self._stage
        if self._stage_events[j] is not None:
            self._stage_events[j].synchronize()  # this buffer's previous copy is done
        host, offs = self._pinned[j], self._table_offsets
        short = n <= self.max_batch
        parts = [q_indptr, page_indptr, kv_len, page_indices]
        part_offs = [offs[0], offs[1], offs[2], offs[5]]
        pos_off, slot_off = (offs[3], offs[4]) if short else (offs[6], offs[7])
        for vals, off in zip(parts + [positions, slots], part_offs + [pos_off, slot_off]):
            host[off:off + len(vals)] = torch.tensor(vals, dtype=torch.int32)
        ranges = [(0, offs[5] + len(page_indices))]
        if not short:
            ranges += [(pos_off, pos_off + n), (slot_off, slot_off + n)]
        if copies:
            ranges.append((offs[8], offs[8] + 2 * len(copies)))
            host[offs[8]:offs[8] + 2 * len(copies)] = torch.tensor(copies, dtype=torch.int32).t().flatten()
        for a, b in ranges:
            self._tables_dev[a:b].copy_(host[a:b], non_blocking=True)
        if self.data.is_cuda:
            ev = torch.cuda.Event()
            ev.record()
            self._stage_events[j] = ev
            self._stage = j ^ 1
        if copies:
            self._copy_pages(*self._copies[:2 * len(copies)].split(len(copies)))
        self.tables = ForwardTables(
            batch=batch, num_tokens=n, max_q_len=max(append_lengths),
            max_kv_len=max(kv_len), q_indptr=self._q_indptr[:batch + 1],
            positions=(self._positions_short if short else self._positions)[:n],
            slots=(self._slots_short if short else self._slots)[:n],
            page_indptr=self._page_indptr[:batch + 1],
            page_indices=self._page_indices[:max(1, len(page_indices))],
            kv_len=self._kv_len[:batch],
            windows=tuple(self.seqs[s].window for s in seq_ids))
        return self.tables

    def end_forward(self) -> None:
        self.tables = None
