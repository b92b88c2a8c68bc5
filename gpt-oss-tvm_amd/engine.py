"""Decode-loop engine on MI355X: the reference's ``Engine`` (engine.py:14-183)
without the TVM compile step.

The model runs eagerly on torch's current stream through the HIP kernels of
libmoe_gfx950; the KV cache is ``model.kv_cache.PagedKVCache``; sampling is
the GPU top-p sampler (``attn_sample_top_p``) with the reference's fixed
parameters (temperature 0.7, top_p 0.9, uniform sample 0.5: engine.py:40).
A chat loop drives it exactly as the reference's chat.py does: ``prefill``
(or ``extend``) the prompt, ``sample``, then ``decode`` + ``sample`` per
generated token, ``popn`` to roll the cache back.  ``kv_dtype`` torch.float8_e4m3fn
keeps the cache in 8 bits: half its bytes in memory and in every decode step.

Beyond one continuation at a time: ``decode_tree`` verifies a tree of drafted tokens in one
forward and gives the tokens that ``decode`` and ``sample`` would have given one by one (but
where the kernels' rounding, another over a tree, decides between two), and ``beam_search``
follows the best continuations by their probability (``max_batch`` beams).
"""
from __future__ import annotations

from pathlib import Path

import numpy as np
import torch

import attn_native as A
from model.config import GPTOssConfig
from model.transformer import GPTOssForCausalLM


class Engine:
    next_seq_id = 0

    def __init__(self, model_path: str | Path | None = None, config: GPTOssConfig | None = None,
                 device: str = "cuda", max_total_seq_len: int | None = None,
                 kv_dtype: torch.dtype = torch.bfloat16, max_batch: int = 1):
        if model_path is not None:
            self.model_path = Path(model_path)
            self.config = config or GPTOssConfig.from_file(self.model_path / "config.json")
        elif config is not None:
            self.model_path, self.config = None, config
        else:
            raise ValueError("give a checkpoint directory or a config")
        self.device = torch.device(device)
        self.model = GPTOssForCausalLM(self.config, device=self.device)
        if self.model_path is not None:
            import weights
            weights.TorchCheckpoint(self.model_path, self.device).load_into(self.model)
        cw = self.config.context_window_size or 40960
        self.paged_kv_cache = self.model.create_paged_kv_cache(
            max_batch, max_total_seq_len or cw, self.config.prefill_chunk_size, 16, self.device,
            dtype=kv_dtype)
        self.sample_parameters = {"temperature": 0.7, "top_p": 0.9, "random_seed": 0.5}
        self._sample_ws = A.sample_workspace(1, self.device)
        self._token = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._tree_ws: torch.Tensor | None = None  # the sampler's, for a tree's nodes

    # -- sequences (engine.py:109-131) ---------------------------------------------
    def clear_kv_cache(self) -> None:
        self.paged_kv_cache.clear()

    def begin_sequence(self, sliding_window_size: int | None = None,
                       sink_size: int | None = None) -> int:
        seq_id = self.__class__.next_seq_id
        self.__class__.next_seq_id += 1
        self.paged_kv_cache.add_sequence(seq_id)
        sliding_window_size = sliding_window_size or self.config.sliding_window_size
        if sliding_window_size > 0:
            self.paged_kv_cache.enable_sliding_window(seq_id, sliding_window_size, sink_size or 0)
        return seq_id

    def popn(self, seq_id: int, n: int) -> None:
        self.paged_kv_cache.popn(seq_id, n)

    def get_kv_total_seq_len(self) -> int:
        return self.paged_kv_cache.total_sequence_length()

    # -- forward passes (engine.py:133-174) --------------------------------------------
    def _ids(self, input_tokens) -> torch.Tensor:
        if isinstance(input_tokens, torch.Tensor):
            return input_tokens.to(device=self.device, dtype=torch.int32).reshape(-1)
        return torch.from_numpy(np.ascontiguousarray(input_tokens, dtype=np.int32).reshape(-1)).to(
            self.device)

    def _run(self, fn, input_tokens, sequence_id: int) -> torch.Tensor:
        ids = self._ids(input_tokens)
        embed = self.model.embed(ids)
        self.paged_kv_cache.begin_forward([sequence_id], [ids.numel()])
        try:
            return fn(embed, self.paged_kv_cache)
        finally:
            self.paged_kv_cache.end_forward()

    @torch.no_grad()
    def prefill(self, input_tokens, sequence_id: int = 0) -> torch.Tensor:
        return self._run(self.model.prefill, input_tokens, sequence_id)

    @torch.no_grad()
    def decode(self, input_tokens, sequence_id: int = 0) -> torch.Tensor:
        return self._run(self.model.decode, input_tokens, sequence_id)

    @torch.no_grad()
    def extend(self, input_tokens, sequence_id: int = 0) -> torch.Tensor:
        return self._run(self.model.extend, input_tokens, sequence_id)

    # -- several continuations at once ---------------------------------------------------
    @torch.no_grad()
    def decode_tree(self, input_tokens, parents, sequence_id: int = 0) -> list[int]:
        """One step over a tree of drafted tokens: ``input_tokens[0]`` is the last sampled token
        (as ``decode`` takes it), every other one a draft for the place after
        ``parents[i]`` < i (``parents[0]`` is -1).  Each node's next token is sampled as
        ``sample`` does; the nodes on the way from the root that were sampled stay in the
        cache.  Returns the new tokens, the accepted ones and the one sampled after the last
        of them: at least one, and the next call's root is the last."""
        ids, parents = self._ids(input_tokens), list(parents)
        n, cache, p = len(parents), self.paged_kv_cache, self.sample_parameters
        if ids.numel() != n:
            raise ValueError(f"{ids.numel()} tokens and {n} parents")
        if self._tree_ws is None or self._tree_ws.numel() < n * self._sample_ws.numel():
            self._tree_ws = A.sample_workspace(n, self.device)
        tables = cache.begin_tree([sequence_id], [parents])
        try:
            logits = self.model.decode_logits_bf16(self.model.embed(ids), cache)
            chosen = A.sample_top_p(logits, p["temperature"], p["top_p"], p["random_seed"],
                                    self._tree_ws)
            path, count, after = A.tree_commit(
                cache.data, tables.page_indptr, tables.page_indices, tables.kv_len,
                tables.q_indptr, n, ids, tables.parents, chosen)
            self._token.copy_(after)
            new = torch.cat([count, after, ids[path.clamp(min=0).long()]]).tolist()
        except Exception:
            cache.popn(sequence_id, n)
            raise
        finally:
            cache.end_forward()
        accepted = new[0]
        cache.popn(sequence_id, n - accepted)
        return new[3:2 + accepted] + [new[1]]

    @torch.no_grad()
    def beam_search(self, input_tokens, width: int, max_new_tokens: int, stop_tokens=(),
                    length_penalty: float = 0.0) -> list[tuple[list[int], float]]:
        """The ``width`` best continuations of a prompt found by beam search: at most
        ``max_new_tokens`` tokens each (a stop token ends one), with the sum of their log
        probabilities, best first by that sum over length ** ``length_penalty``.  It goes on
        until no beam can come to more than the ``width`` best that have ended; beams that
        have not are results only with all ``max_new_tokens`` tokens.  The beams share
        the prompt's pages and each other's; the engine's cache needs room for ``width``
        sequences (``max_batch``) and is left as it was."""
        cache, stops = self.paged_kv_cache, set(int(t) for t in stop_tokens)
        vocab = self.config.vocab_size
        # of the best width (1 + stops) continuations no more than width stops end
        k = min(width * (1 + len(stops)), width * vocab)
        if not 1 <= width <= cache.max_batch or k > A.MAX_BEAMS or max_new_tokens < 1:
            raise ValueError(f"beam search of width {width} with {len(stops)} stop tokens and "
                             f"{max_new_tokens} new tokens: the cache has room for "
                             f"{cache.max_batch} sequences, the selection for {A.MAX_BEAMS}")
        beams = [([], 0.0)]
        ended: list[tuple[list[int], float]] = []
        seqs = [self.begin_sequence()]

        def worth(beam):
            return beam[1] / max(1, len(beam[0])) ** length_penalty

        def settled():  # sums only fall, so a beam comes to no more than this one's at best
            longest = max_new_tokens if length_penalty > 0 else len(beams[0][0]) + 1
            best = beams[0][1] / longest ** length_penalty
            return len(ended) >= width and sorted(map(worth, ended))[-width] >= best

        try:
            logits = self.prefill(input_tokens, seqs[0]).view(1, vocab)
            for step in range(max_new_tokens):
                scores = torch.tensor([[s for _, s in beams]], dtype=torch.float32,
                                      device=self.device)
                best = A.beam_top_k(logits, scores, min(k, len(beams) * vocab))
                best = zip(*(t[0].tolist() for t in best))
                live, parents = [], []
                for score, parent, token in best:
                    if score == float("-inf") or len(live) == width:
                        break
                    if token in stops:
                        ended.append((beams[parent][0] + [token], score))
                    else:
                        live.append((beams[parent][0] + [token], score))
                        parents.append(parent)
                beams = live
                if not live or step == max_new_tokens - 1:
                    break
                if settled():
                    beams = []
                    break
                new = seqs[:len(live)]
                while len(new) < len(live):
                    new.append(self.__class__.next_seq_id)
                    self.__class__.next_seq_id += 1
                cache.branch(seqs, parents, new)
                seqs = new
                embed = self.model.embed(self._ids([tokens[-1] for tokens, _ in live]))
                cache.begin_forward(seqs, [1] * len(live))
                try:
                    logits = self.model.decode_logits_bf16(embed, cache)
                finally:
                    cache.end_forward()
        finally:
            for sid in seqs:
                if sid in cache.seqs:
                    cache.remove_sequence(sid)
        return sorted(ended + beams, key=worth, reverse=True)[:width]

    # -- the decode step in one HIP graph ---------------------------------------------
    def _step_body(self) -> None:
        embed = self.model.embed(self._token)
        lb = self.model.decode_logits_bf16(embed, self.paged_kv_cache)
        self._graph_logits_bf16 = lb
        p = self.sample_parameters
        A.sample_top_p(lb[-1:], p["temperature"], p["top_p"], p["random_seed"], self._sample_ws,
                       self._token)

    @property
    def graph_logits(self) -> torch.Tensor:
        """fp32 logits [1, 1, vocab] of the last captured decode step (its bf16
        logits, converted on request)."""
        return self._graph_logits_bf16.float().view(1, -1, self.config.vocab_size)

    @torch.no_grad()
    def capture_decode(self, sequence_id: int) -> None:
        """Capture one decode step of ``sequence_id`` -- embedding of the last
        sampled token, every layer, final norm, unembedding, sampling into the
        same token buffer -- in a HIP graph (``decode_sample`` replays it).

        Nothing is allocated inside the step: the KV cache's forward tables
        are fixed device buffers refreshed by ``begin_forward`` before each
        replay, every MoE block's workspace is reserved for one token, and the
        decode attention's split count is fixed at the pool's capacity
        (``static_span``).  The workspaces the graph captures are held for the
        life of the model, so a later, longer prefill or extend (which grows
        the eager workspaces) leaves them in place.  The warm-up and capture
        steps are rolled back."""
        c = self.paged_kv_cache
        c.static_span = c.num_pages * 16
        c.reserve_decode(1, c.static_span, for_graph=True)
        for blk in self.model.model.block:
            blk.mlp.reserve(1, for_graph=True)
        token = self._token.clone()  # the warm-up step samples over it
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.begin_forward([sequence_id], [1])
            self._step_body()
            c.end_forward()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        c.popn(sequence_id, 1)
        self._token.copy_(token)
        c.begin_forward([sequence_id], [1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step_body()
        c.end_forward()
        c.popn(sequence_id, 1)
        self._graph, self._graph_seq = graph, sequence_id

    def decode_sample(self, sequence_id: int) -> torch.Tensor:
        """One captured decode step fed with the last sampled token
        (``sample_device`` / ``sample`` wrote it): the next token, as the
        1-element device tensor the following step reads; its logits are in
        ``graph_logits``."""
        if getattr(self, "_graph", None) is None or self._graph_seq != sequence_id:
            raise RuntimeError(f"capture_decode({sequence_id}) first")
        self.paged_kv_cache.begin_forward([sequence_id], [1])
        self._graph.replay()
        self.paged_kv_cache.end_forward()
        return self._token

    def sample_device(self, logits: torch.Tensor) -> torch.Tensor:
        """The sampled token id as a 1-element int32 device tensor (no host sync).

        The logits are the unembedding's bf16 values in fp32; they go back to
        bf16 exactly for the sampler."""
        p = self.sample_parameters
        lb = logits.reshape(-1, logits.shape[-1])[-1:].to(torch.bfloat16)
        return A.sample_top_p(lb, p["temperature"], p["top_p"], p["random_seed"],
                              self._sample_ws, self._token)

    def sample(self, logits: torch.Tensor) -> int:
        """engine.py:165-167: one token id from the last row of ``logits``."""
        return int(self.sample_device(logits).item())
