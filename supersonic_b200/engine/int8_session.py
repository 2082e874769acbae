"""A model's sequences in 8 bits: its projections as int8 weights with a scale per output channel, its keys and values as int8 codes
with a scale per block of tokens and head, and, with a budget, sequences that are cut down to their first, latest and most attended
tokens whenever they outgrow it.

    session = Int8Session(engine.model, max_tokens=65536, budget=2048)
    tokens = session.generate([[128000, 9906, 1917]], max_new_tokens=32)

A step runs the model's own embedding, norms, rotation tables, feed-forward activation and head; the projections go through
``int8_ops.linear`` and the attention through ``int8_ops.append`` and ``int8_ops.attention``.  A sequence's *position* counts every
token it was given (keys stay rotated by the positions they had); its *place* is where the next token goes in the cache, which is the
smaller one once tokens were evicted.  Every kv head of every layer keeps tokens of its own.

For ``LlamaForCausalLM`` models (rotary attention and a gated feed-forward behind pre-norms), in bfloat16 and float32; the embedding
and the head stay in the model's type, as in the modelled project's 8-bit lane (crates/runner/src/llama31_engine.rs:289-430).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import numpy as np
import torch

from ..cache import PAGE_TOKENS, CacheFull, Int8Pages, pages_for
from ..csrc import int8_ops, ops
from ..csrc.kernel_sets import NormedInput
from ..parts.attention import Attention
from ..parts.block import PreNormBlock
from ..parts.feed_forward import SwiGLU
from .batch import StepEntry, batch_over, pack_entries, plan_chunks
from .model import Model, StepContext


@dataclass
class _Layer:
    block: PreNormBlock
    pages: Int8Pages
    weights: dict = field(default_factory=dict)      # name -> (codes, scale of every output channel)


class Int8Session:
    """``max_tokens``: tokens that the cache holds in all, in whole pages (a sequence that is cut takes its budget's pages beside its own
    for as long as that lasts); ``budget``: tokens a sequence may keep (None: all), of which the first ``first`` and the latest
    ``recent`` stay in any case; ``slack``: tokens it may grow beyond that before it is cut down to it again; ``observe``: how many of a
    step's last rows account for what they attend to.

    The 8-bit weights are made from the model's and lie beside them, as the cache lies beside the model's own (:meth:`bytes_held`)."""

    def __init__(self, model: Model, max_tokens: int, max_sequences: int = 64, budget: Optional[int] = None, first: int = 4,
                 recent: Optional[int] = None, slack: int = PAGE_TOKENS, block: int = 16, observe: int = 32):
        self.model, self.device, self.dtype = model, model.device, model.dtype
        self.budget, self.first = budget, first
        self.recent = (budget // 2 if budget else 0) if recent is None else recent
        self.slack, self.observe = slack, observe
        if budget is not None and (budget <= 0 or slack < 1 or first < 0 or self.recent < 0 or first + self.recent > budget):
            raise ValueError(f"a budget of {budget} tokens has no room for the first {first} and the latest {self.recent}")
        n_pages = pages_for(max_tokens)
        stops = model.spec.schedule
        if [s.layer for s in stops] != list(range(len(model.blocks))) or len({s.cache for s in stops}) != len(stops) \
                or any(s.before is not None or not s.writes_cache for s in stops) or hasattr(getattr(model, "embedding", None), "cache_need"):
            raise ValueError("an 8-bit session runs every layer once, in order, each with a cache of its own and nothing between them")
        self.layers: List[_Layer] = []
        for b in model.blocks:
            mixer, ff, rotary = b.mixer, getattr(b, "feed_forward", None), getattr(b, "position", None)
            if type(b) is not PreNormBlock or not isinstance(mixer, Attention) or not isinstance(ff, SwiGLU) or ff.act is not None \
                    or getattr(rotary, "rotary_tables", None) is None or rotary.interleaved or rotary.rotary_dim % 16:
                raise ValueError("an 8-bit session runs layers of rotary attention and a silu-gated feed-forward behind pre-norms")
            if mixer.window is not None and budget is not None:
                raise ValueError("a window counts positions, which a sequence's places are no longer once it was cut to a budget")
            layer = _Layer(b, Int8Pages.allocate(n_pages, mixer.n_kv, mixer.head_dim, block, weights=budget is not None, device=self.device))
            for name, w in (("qkv", mixer.w_qkv), ("o", mixer.w_o), ("gate_up", ff.w_gate_up), ("down", ff.w_down)):
                codes = torch.empty(w.shape, dtype=torch.int8, device=self.device)
                scale = torch.empty(w.shape[0], dtype=torch.float32, device=self.device)
                int8_ops.quantize_rows(w, codes, scale)
                layer.weights[name] = (codes, scale)
            self.layers.append(layer)
        self.n_pages = n_pages
        self.free = list(range(n_pages - 1, -1, -1))
        self.held: List[List[int]] = [[] for _ in range(max_sequences)]
        self.position = [0] * max_sequences          # tokens given
        self.length = [0] * max_sequences            # tokens held
        self.open_slots = set()
        per_seq = n_pages if budget is None else min(n_pages, pages_for(budget + slack + model.step_token_budget))
        self.table_host = torch.zeros((max_sequences, per_seq), dtype=torch.int32)
        self.table = self.table_host.to(self.device)          # changed in place: captured steps read it
        self.graphs = {}                                       # sequences -> a captured step of single tokens

    # ---- sequences -----------------------------------------------------------------------
    def open(self) -> int:
        for slot in range(len(self.held)):
            if slot not in self.open_slots:
                self.open_slots.add(slot)
                self.position[slot] = self.length[slot] = 0
                return slot
        raise CacheFull(f"all {len(self.held)} sequences are open")

    def close(self, slot: int) -> None:
        self.free += self.held[slot]
        self.held[slot] = []
        self.open_slots.discard(slot)

    def _take(self, n: int) -> List[int]:
        if n > len(self.free):
            raise CacheFull(f"{n} more pages of 64 tokens are needed, {len(self.free)} are free")
        return [self.free.pop() for _ in range(n)]

    def _write_table(self, slots) -> None:
        for slot in slots:
            pages = self.held[slot]
            self.table_host[slot, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self.table.copy_(self.table_host)

    def _plan(self, slots, counts) -> list:
        """A step of these new tokens as chunks, each a list of (entry, first, end) and the groups of sequences that are cut behind it
        (:meth:`_cuts`); CacheFull if there is no room for one of them.

        A chunk has the model's ``step_token_budget`` tokens at most.  A sequence that fits its row of the page table, and the cache
        beside the pages of its cut, is cut behind its last token.  One that does not is cut behind every chunk in which it outgrows its
        budget, and chunks are as small as leaves room for that."""
        width, per, limit = self.table_host.shape[1], pages_for(self.budget or 0), self.model.step_token_budget
        length, spans, free = {s: self.length[s] for s in slots}, {s: len(self.held[s]) for s in slots}, len(self.free)
        whole = [True] * len(slots)
        if self.budget is not None:
            cut_at = self.budget + self.slack
            for i, (slot, n) in enumerate(zip(slots, counts)):
                pages = pages_for(length[slot] + n)
                whole[i] = pages <= width and (length[slot] + n < cut_at or pages + per <= self.n_pages)
            if not all(whole):
                limit = max(1, min(limit, min(width, self.n_pages - per) * PAGE_TOKENS - cut_at + 1))
        chunks = []
        for pieces in [[(i, 0, n) for i, n in enumerate(counts)]] if sum(counts) <= limit else plan_chunks(counts, limit):
            cut = []
            for i, first, end in pieces:
                slot = slots[i]
                length[slot] += end - first
                pages = max(spans[slot], pages_for(length[slot]))
                if pages > width:
                    raise CacheFull(f"a sequence of {length[slot]} tokens spans {pages} pages, its table has {width}")
                free -= pages - spans[slot]
                spans[slot] = pages
                if self.budget is not None and length[slot] >= cut_at and (end == counts[i] or not whole[i]):
                    cut.append(slot)
            if free < 0:
                raise CacheFull(f"{-free} more pages of 64 tokens are needed than are free")
            groups = self._cuts(cut, free, spans)
            for slot in cut:
                free += spans[slot] - per
                spans[slot], length[slot] = per, self.budget
            chunks.append((pieces, groups))
        return chunks

    def _reserve(self, slots, counts) -> None:
        """Pages for these new tokens, and their rows of the page table."""
        grown = []
        for slot, n in zip(slots, counts):
            more = pages_for(self.length[slot] + n) - len(self.held[slot])
            if more > 0:
                self.held[slot] += self._take(more)
                grown.append(slot)
        if grown:
            self._write_table(grown)

    def _cuts(self, slots: List[int], free: int, spans) -> List[List[int]]:
        """Sequences of ``spans[slot]`` pages in the groups that they are cut in: a cut sequence moves to pages of its own beside its old
        ones, so as many go together as ``free`` pages hold, and a group's old pages make room for the next."""
        per, groups = pages_for(self.budget or 0), []
        while slots:
            n = min(len(slots), free // per)
            if n == 0:
                raise CacheFull(f"cutting a sequence takes {per} pages of 64 tokens beside its own, {free} are free")
            groups.append(slots[:n])
            free += sum(spans[s] for s in slots[:n]) - n * per
            slots = slots[n:]
        return groups

    # ---- the step ------------------------------------------------------------------------
    def step(self, entries: Sequence[StepEntry]) -> torch.Tensor:
        """Run the entries' tokens; float32 logits [wanted, vocab], as :meth:`Model.step` gives them.  More tokens than the model's
        ``step_token_budget`` run as several steps.  A step that is refused, for want of pages for its tokens or for the cuts behind it
        too, has changed nothing."""
        for e in entries:
            if e.slot not in self.open_slots:
                raise ValueError(f"slot {e.slot} is not open")
        packed = pack_entries(entries, [self.position[e.slot] for e in entries], self.model.vocab_size)
        self.model._check_positions(packed.max_total)
        chunks = self._plan(packed.slots, packed.counts)
        if len(chunks) == 1:
            return self._run(packed, chunks[0][1])
        rows, order = [], []
        for pieces, cuts in chunks:
            part = [StepEntry(entries[i].slot, entries[i].tokens[first:end], [w - first for w in entries[i].want if first <= w < end])
                    for i, first, end in pieces]
            rows.append(self._run(pack_entries(part, [self.position[e.slot] for e in part]), cuts))
            order += [(i, j) for i, first, end in pieces for j, w in enumerate(entries[i].want) if first <= w < end]
        back = sorted(range(len(order)), key=order.__getitem__)       # an entry's wanted rows come in the order it named them
        return torch.cat(rows)[torch.tensor(back, dtype=torch.int64, device=self.device)]

    def _run(self, packed, cuts) -> torch.Tensor:
        """One chunk, and the cuts behind it."""
        slots, counts = packed.slots, packed.counts
        self._reserve(slots, counts)
        starts = [self.length[s] for s in slots]
        places = [np.arange(a, a + n) for a, n in zip(starts, counts)]
        flat = np.concatenate([packed.flat] + places + [starts]).astype(np.int32)      # the step's integers, then the cache's
        if self.model.use_graphs and packed.n_want == packed.n_tokens == packed.n_seqs:
            logits = self._captured(packed, flat)
        else:
            logits = self._forward(packed, torch.from_numpy(flat).to(self.device))
        for slot, n in zip(slots, counts):
            self.position[slot] += n
            self.length[slot] += n
        for group in cuts:
            self._evict(group)
        return logits

    def _captured(self, packed, flat) -> torch.Tensor:
        """A step of one token a sequence: its launches are recorded the first time there are that many sequences, and replayed over
        the integers and the page table as they are then."""
        n = packed.n_seqs
        if n not in self.graphs:
            ints = torch.from_numpy(flat).to(self.device)
            side = torch.cuda.Stream(device=self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side):                     # once uncaptured: what is set up at first use; padding, so nothing is written
                idle = ints.clone()
                idle[2 * n:4 * n] = -1                        # the slots, by token and by sequence
                self._forward(packed, idle)
            torch.cuda.current_stream(self.device).wait_stream(side)
            torch.cuda.synchronize(self.device)
            graph, waits = torch.cuda.CUDAGraph(), ops.bounded_wait_launches()
            with torch.cuda.graph(graph):
                logits = self._forward(packed, ints)
            self.graphs[n] = (graph, ints, logits, ops.bounded_wait_launches() - waits)
        graph, ints, logits, waits = self.graphs[n]
        ints.copy_(torch.from_numpy(flat))
        graph.replay()
        ops.note_bounded_wait_launches(waits)
        return logits.clone()                                 # the graph's own buffer is written by its next replay

    def _forward(self, packed, ints) -> torch.Tensor:
        """``ints``: the packed step's integers, every token's place in its cache, every sequence's tokens held before the step."""
        model, T, n = self.model, packed.n_tokens, packed.flat.shape[0]
        batch, place, seq_start = batch_over(ints[:n], packed), ints[n:n + T], ints[n + T:]
        ctx = StepContext(batch, model.cache, model.kernels, self.dtype)
        residual = model.embedding(ctx, batch.token_ids)
        new = lambda width: torch.empty((T, width), dtype=self.dtype, device=self.device)       # noqa: E731
        for layer in self.layers:
            b, w = layer.block, layer.weights
            mixer, ff = b.mixer, b.feed_forward
            cos, sin, _ = b.position.rotary_tables()
            qkv, attn = new((mixer.n_q + 2 * mixer.n_kv) * mixer.head_dim), new(mixer.n_q * mixer.head_dim)
            int8_ops.linear(NormedInput(ctx, residual, b.mixer_norm).tensor(), *w["qkv"], qkv)
            int8_ops.append(qkv, cos, sin, batch.pos, place, batch.slot_of_token, self.table, layer.pages, qkv, mixer.n_q)
            int8_ops.attention(qkv, layer.pages, self.table, batch.cu_new, seq_start, batch.seq_slot, batch.max_new, attn, mixer.n_q,
                               mixer.scale, window=mixer.window, weigh_last=self.observe if self.budget is not None else 0)
            int8_ops.linear(attn, *w["o"], residual, accumulate=True)
            gate_up, inner = new(w["gate_up"][0].shape[0]), new(ff.inter)
            int8_ops.linear(NormedInput(ctx, residual, b.feed_forward_norm).tensor(), *w["gate_up"], gate_up)
            ops.swiglu(gate_up, inner, interleaved=ff.layout == "interleaved")
            int8_ops.linear(inner, *w["down"], residual, accumulate=True)
        if batch.n_want == 0:
            return torch.empty((0, model.vocab_size), dtype=torch.float32, device=self.device)
        return model.head(ctx, model.final_norm(ctx, residual, rows=batch.want_rows))

    def _evict(self, slots: List[int]) -> None:
        """Cut these sequences down to the budget: every layer moves what it keeps to the same new pages, the old ones are free again."""
        budget, per = self.budget, pages_for(self.budget)
        B = len(slots)
        new = [self._take(per) for _ in slots]
        as_ints = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)               # noqa: E731
        new_table, seq_slot, lengths = as_ints(new), as_ints(slots), as_ints([self.length[s] for s in slots])
        for layer in self.layers:
            kept = torch.empty((B, layer.pages.k.shape[1], budget), dtype=torch.int32, device=self.device)
            int8_ops.evict(layer.pages, self.table, seq_slot, lengths, new_table, budget, self.first, self.recent, kept)
        for slot, pages in zip(slots, new):
            self.free += self.held[slot]
            self.held[slot] = pages
            self.length[slot] = min(self.length[slot], budget)
        self._write_table(slots)

    # ---- greedy generation ---------------------------------------------------------------
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 8, stop_token_ids: Sequence[int] = ()) -> List[List[int]]:
        """Greedy tokens for each prompt, all prompts in one batch; a sequence ends at one of ``stop_token_ids`` (the model's own are in
        its ``spec.stop_token_ids``)."""
        slots: List[int] = []
        out: List[List[int]] = [[] for _ in prompts]
        try:
            for _ in prompts:
                slots.append(self.open())
            live = list(range(len(prompts)))
            entries = [StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]
            while live and max_new_tokens > 0:
                picks = self.step(entries).argmax(-1).tolist()
                ops.check_device_errors(self.device)
                for i, t in zip(live, picks):
                    out[i].append(int(t))
                live = [i for i in live if out[i][-1] not in stop_token_ids and len(out[i]) < max_new_tokens]
                entries = [StepEntry(slots[i], [out[i][-1]], [0]) for i in live]
        finally:
            for s in slots:
                self.close(s)
        return out

    def bytes_held(self) -> int:
        """Device bytes of the 8-bit weights and cache."""
        return sum(layer.pages.bytes_held() + sum(c.numel() + 4 * s.numel() for c, s in layer.weights.values()) for layer in self.layers)
