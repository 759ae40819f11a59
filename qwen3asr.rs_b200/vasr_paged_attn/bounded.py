"""Speculative decoding over a cache that stays within a budget.

One step per call, for a batch of sequences: the last emitted token and K drafted ones go through
the decoder as a window of K + 1 rows (``fused.qk_norm_mrope_append`` appends them and clears their
scores, ``eviction.paged_attention_scored`` attends and scores the cache with the window's first
row, the only one known to stay), ``speculative.verify_draft_tokens`` keeps a prefix of the drafts
and draws the next token, and once a sequence's pages run full every sequence longer than the budget
is shrunk to it by ``eviction.evict_kv``, layer by layer and kv head by kv head. Positions run on
while the cache shrinks, so a token's position is no longer its place in the cache.

The reference decodes one greedy token a step over a cache that only grows
(vasr-models/src/model/paged_batch_engine.rs:609-730); with temperature 0 and a budget that is
never reached the tokens here are the same.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
import torch.nn.functional as F

from . import _lib, eviction, fused, speculative
from . import mistralrs_paged_attn as pa
from .engine import RandomQwen3Decoder, allocate_paged_cache

MAX_WINDOW = 64  # rows a sequence that paged_attention_scored takes


def lookup_drafts(tokens: Sequence[int], count: int) -> list[int]:
    """Drafts read off the sequence itself: what followed the last earlier occurrence of its last
    two tokens (of its last token; else that token again)."""
    n = len(tokens)
    if count == 0:
        return []
    for width in (2, 1):
        tail = list(tokens[n - width:])
        for at in range(n - width - 1, -1, -1):
            if list(tokens[at:at + width]) == tail:
                found = list(tokens[at + width:at + width + count])
                return found + [found[-1]] * (count - len(found))
    return [tokens[-1]] * count


class BoundedSpeculativeDecoder:
    """A batch of sequences decoded K drafts at a time in pages for ``capacity`` tokens each.

    ``budget`` tokens (``num_sink`` first, ``num_recent`` last, the rest by score) stay when a
    sequence's next window would not fit. ``temperature`` 0 is greedy.
    """

    def __init__(self, model: RandomQwen3Decoder, num_seqs: int, num_drafts: int, capacity: int, budget: int,
                 num_sink: int = 4, num_recent: int = 32, block_size: int = 16, temperature: float = 0.0,
                 sections: Sequence[int] = (24, 20, 20), seed: int = 0):
        window = num_drafts + 1
        if budget + window > capacity or num_sink + num_recent > budget:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "budget must leave room for a window, and hold sinks and recent tokens")
        cfg = model.cfg
        self.model, self.num_seqs, self.num_drafts = model, num_seqs, num_drafts
        self.budget, self.num_sink, self.num_recent = budget, num_sink, num_recent
        self.block_size, self.temperature, self.sections = block_size, float(temperature), tuple(sections)
        dev = self.device = model.device
        cols = -(-capacity // block_size)
        self.capacity = cols * block_size
        blocks = num_seqs * cols + 1  # block 0 is the null block
        self.caches = allocate_paged_cache(cfg, blocks, block_size, dev, dtype=model.dtype)
        self.scores = [eviction.allocate_score_cache(kc) for kc, _ in self.caches]
        self.block_tables = (1 + torch.arange(num_seqs * cols, dtype=torch.int32, device=dev)).view(num_seqs, cols)
        self.context_lens = torch.zeros(num_seqs, dtype=torch.int32, device=dev)  # tokens in the cache
        self.next_positions = torch.zeros(num_seqs, dtype=torch.int64, device=dev)
        self.tokens: list[list[int]] = [[] for _ in range(num_seqs)]
        self.evictions = 0
        self.max_positions = model.rope_cos.shape[0]
        self._gen = torch.Generator(device=dev).manual_seed(seed)

    def _layers(self, ids: torch.Tensor, rows: int, score_rows: Optional[int]) -> torch.Tensor:
        """ids [B, rows], appended behind the cached tokens; logits [B, rows, vocab]."""
        cfg = self.model.cfg
        b, dev, bs = self.num_seqs, self.device, self.block_size
        step = torch.arange(rows, device=dev)
        places = self.context_lens.long()[:, None] + step
        slots = (self.block_tables.long().gather(1, places // bs) * bs + places % bs).flatten()
        # text: the time, height and width streams are one (a broadcast over the axes)
        positions = (self.next_positions[:, None] + step).flatten().expand(len(self.sections), b * rows)
        lens = self.context_lens + rows
        x = F.embedding(ids.flatten(), self.model.embed)
        for l, (kc, vc), scores in zip(self.model.layers, self.caches, self.scores):
            h = F.rms_norm(x, (cfg.hidden_size,), l["in_norm"], cfg.rms_norm_eps)
            q = fused.qk_norm_mrope_append(h @ l["w_qkv"].t(), l["q_norm"], l["k_norm"], cfg.rms_norm_eps,
                                           self.model.rope_cos, self.model.rope_sin, positions, self.sections,
                                           kc, vc, slots, cfg.num_heads, score_cache=scores)
            attn = eviction.paged_attention_scored(
                q.view(b, rows, cfg.num_heads, cfg.head_dim), None, None, kc, vc, scores, self.block_tables,
                lens, self.capacity, cfg.head_dim ** -0.5, score_rows=score_rows)
            x.addmm_(attn.view(b * rows, -1), l["w_o"].t())
            h = F.rms_norm(x, (cfg.hidden_size,), l["post_norm"], cfg.rms_norm_eps)
            gate, up = (h @ l["w_gate_up"].t()).split(cfg.intermediate_size, dim=1)
            x.addmm_(F.silu(gate) * up, l["w_down"].t())
        x = F.rms_norm(x, (cfg.hidden_size,), self.model.final_norm, cfg.rms_norm_eps)
        return (x @ self.model.embed.t()).view(b, rows, -1)

    def _make_room(self, rows: int, longest: int) -> None:
        """Shrinks every sequence to the budget once one of them has no place for ``rows`` more."""
        if longest + rows <= self.capacity:
            return
        if min(longest, self.budget) + rows > self.capacity:  # the slots would lie past the block table
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, f"no room for {rows} tokens beside a budget of {self.budget}")
        lens = self.context_lens
        for (kc, vc), scores in zip(self.caches, self.scores):
            _, lens = eviction.evict_kv(kc, vc, scores, self.block_tables, self.context_lens, self.capacity,
                                        self.budget, self.num_sink, self.num_recent)
        self.context_lens = lens
        self.evictions += 1

    def prefill(self, prompts: Sequence[Sequence[int]], window: int = 16) -> None:
        """Prompts of one length, ``window`` tokens at a time (fewer where an eviction leaves room for
        fewer, and at most the attention's 64); all but the last token, which the first step's window
        begins with. Every row of a prompt's windows scores the cache."""
        length = len(prompts[0])
        if length < 1 or any(len(p) != length for p in prompts) or len(prompts) != self.num_seqs:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "prompts must be num_seqs sequences of one length")
        if window < 1:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "window must be at least one token")
        if length - 1 > self.max_positions:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, f"a prompt of {length} tokens leaves the rotary tables")
        # a decoder that has decoded before starts afresh: the appends clear the slots' old scores
        self.context_lens = torch.zeros_like(self.context_lens)
        self.next_positions = torch.zeros_like(self.next_positions)
        self.evictions = 0
        self.tokens = [list(p) for p in prompts]
        ids = torch.tensor(self.tokens, device=self.device)
        at = 0
        while at < length - 1:
            longest = int(self.context_lens.max())
            rows = min(window, MAX_WINDOW, length - 1 - at)
            if longest + rows > self.capacity:
                rows = min(rows, self.capacity - min(longest, self.budget))
            self._make_room(rows, longest)
            self._layers(ids[:, at:at + rows], rows, None)
            self.context_lens = self.context_lens + rows
            self.next_positions += rows
            at += rows

    def step(self) -> list[list[int]]:
        """The tokens that this step adds to each sequence: the accepted drafts and one more.

        Positions run on while the cache is shrunk: near the end of the rotary tables a step drafts
        less, and one past it is refused."""
        b, dev = self.num_seqs, self.device
        at = max(len(t) for t in self.tokens) - 1  # the window's first position
        if at >= self.max_positions:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, f"position {at} leaves the rotary tables")
        k = min(self.num_drafts, self.max_positions - 1 - at)
        drafts = torch.tensor([lookup_drafts(t, k) for t in self.tokens], dtype=torch.int32, device=dev).view(b, k)
        last = torch.tensor([t[-1] for t in self.tokens], device=dev)
        self._make_room(k + 1, int(self.context_lens.max()))
        logits = self._layers(torch.cat([last[:, None], drafts.long()], 1), k + 1, 1)
        uniform = race = None
        if self.temperature > 0:
            uniform = torch.rand((b, k), device=dev, generator=self._gen)
            race = torch.empty((b, logits.shape[2]), device=dev).exponential_(generator=self._gen)
        out, accepted = speculative.verify_draft_tokens(logits, drafts, None, uniform, race,
                                                        temperature=self.temperature)
        # the window's first row and the accepted drafts stay; what follows is written over
        self.context_lens = self.context_lens + 1 + accepted
        self.next_positions += 1 + accepted
        added = [row[:n + 1] for row, n in zip(out.tolist(), accepted.tolist())]
        for t, new in zip(self.tokens, added):
            t.extend(new)
        return added

    def device_error(self) -> int:
        return pa.device_error(device=self.device)
