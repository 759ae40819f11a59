"""A cache that stays within a budget: scored decode attention and eviction.

Beside the pages of a layer the caller keeps ``score_cache`` [num_blocks, Hkv, block_size] (f32):
the attention weight that every cached token has gathered so far. ``paged_attention_scored`` adds
to it while it attends, ``fused.qk_norm_mrope_append`` clears it for the tokens that it appends,
and ``evict_kv`` keeps, per kv head, the tokens of the largest scores. The reference has no
counterpart; the calls go next to ``paged_attention`` at
vasr-models/src/model/thinker_text.rs:1126-1139.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _calls, _lib
from ._calls import calls


def allocate_score_cache(key_cache: torch.Tensor) -> torch.Tensor:
    """Zeroed scores for the pages of ``key_cache``."""
    nb, hkv, _, bs, _ = key_cache.shape
    return torch.zeros((nb, hkv, bs), dtype=torch.float32, device=key_cache.device)


def paged_attention_scored_workspace_bytes(num_seqs: int, query_len: int, score_rows: int, num_heads: int,
                                           num_kv_heads: int, head_dim: int, block_size: int,
                                           max_context_len: int) -> int:
    return int(_lib.lib().vasr_pa_paged_attention_scored_workspace_size(
        num_seqs, query_len, score_rows, num_heads, num_kv_heads, head_dim, block_size, max_context_len))


def reserve_paged_attention_scored_workspace(device: torch.device, nbytes: int,
                                             stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Make sure the stream's scratch holds ``nbytes``, so that calls on it do not have to grow it.

    Calls that a CUDA graph captures take theirs from the graph's own memory."""
    return _calls.reserve(_calls.SCORED, device, nbytes, stream)


def paged_attention_scored(q: torch.Tensor, k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                           key_cache: torch.Tensor, value_cache: torch.Tensor, score_cache: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor, max_context_len: int,
                           softmax_scale: float, softcapping: float = 1.0, decay: float = 1.0,
                           score_rows: Optional[int] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's newest token(s) over its pages; adds their weights to the scores.

    ``q`` is [B, Hq, D], or [B, W, Hq, D] for a window of the last W tokens (already appended and
    counted in ``context_lens``); row i sees the tokens up to its own position. Returns q's shape.
    Every token j below the context length gets
    ``score = decay * score + sum of the weights`` that the first ``score_rows`` rows (default:
    all) and the query heads of its kv head give it. A window with drafted tokens passes
    ``score_rows=1``: only the first row is known to stay."""
    return calls().scored(q, k_scale, v_scale, key_cache, value_cache, score_cache, block_tables, context_lens,
                          max_context_len, softmax_scale, softcapping, decay, score_rows, out)


def evict_kv(key_cache: torch.Tensor, value_cache: torch.Tensor, score_cache: torch.Tensor,
             block_tables: torch.Tensor, context_lens: torch.Tensor, max_context_len: int, budget: int,
             num_sink: int, num_recent: int, budgets: Optional[torch.Tensor] = None,
             out_block_tables: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keep at most ``budget`` tokens of every sequence, per kv head; (kept indices, new lengths).

    Kept are the first ``num_sink`` tokens, the last ``num_recent`` and those of the largest scores
    (lower index on equal ones). Their K, V and scores move, in their old order, to the first
    places of the sequence's pages, or to the pages of ``out_block_tables`` (disjoint from the old
    ones). ``budgets`` (u32/i32 [B]) lowers the budget per sequence. kept is int32
    [B, Hkv, budget] (ascending old indices, then -1), the lengths int32 [B]: min(context, budget).
    Pages past ceil(length / block_size) are free for reuse; the caller goes on with the new
    lengths, and with positions that no longer equal the token's place in the cache."""
    return calls().evict(key_cache, value_cache, score_cache, block_tables, context_lens, max_context_len, budget,
                         num_sink, num_recent, budgets, out_block_tables)
