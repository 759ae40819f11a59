"""A cache that stays within a budget: scored decode attention and eviction.

Beside the pages of a layer the caller keeps ``score_cache`` [num_blocks, Hkv, block_size] (f32):
the attention weight that every cached token has gathered so far. ``paged_attention_scored`` adds
to it while it attends, ``fused.qk_norm_mrope_append`` clears it for the tokens that it appends,
and ``evict_kv`` keeps, per kv head, the tokens of the largest scores. The reference has no
counterpart; the calls go next to ``paged_attention`` at
vasr-models/src/model/thinker_text.rs:1126-1139.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from .fused import _check_score_cache
from .mistralrs_paged_attn import (_DTYPE_CODE, _INDEX32, FP8_CACHE, StreamWorkspaces, _check_scales,
                                   _cuda_index, _raw_stream, cache_geometry, dtype_code)

_SCRATCH = StreamWorkspaces("paged_attention_scored")


def allocate_score_cache(key_cache: torch.Tensor) -> torch.Tensor:
    """Zeroed scores for the pages of ``key_cache``."""
    nb, hkv, _, bs, _ = key_cache.shape
    return torch.zeros((nb, hkv, bs), dtype=torch.float32, device=key_cache.device)


@functools.lru_cache(maxsize=256)
def paged_attention_scored_workspace_bytes(num_seqs: int, query_len: int, score_rows: int, num_heads: int,
                                           num_kv_heads: int, head_dim: int, block_size: int,
                                           max_context_len: int) -> int:
    return int(_lib.lib().vasr_pa_paged_attention_scored_workspace_size(
        num_seqs, query_len, score_rows, num_heads, num_kv_heads, head_dim, block_size, max_context_len))


def reserve_paged_attention_scored_workspace(device: torch.device, nbytes: int,
                                             stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Make sure the stream's scratch holds ``nbytes``; call before a CUDA-graph capture."""
    return _SCRATCH.reserve_for(device, nbytes, stream)


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
    dev = _cuda_index(q, key_cache, value_cache, score_cache, block_tables, context_lens)
    nb, hkv, d, bs = cache_geometry(key_cache, value_cache)
    shape, strides = q.shape, q.stride()
    if len(shape) == 3:
        (b, hq, dq), window, q_stride = shape, 1, strides[0]
    elif len(shape) == 4:
        (b, window, hq, dq), q_stride = shape, strides[1] if shape[1] > 1 else strides[0]
        if b > 1 and window > 1 and strides[0] != window * q_stride:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "q's rows must follow one another at one token stride")
    else:
        dq = -1
    if dq != d or strides[-1] != 1 or (strides[-2] != d and hq > 1):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, f"q must be [B, Hq, {d}] or [B, W, Hq, {d}] with packed heads, got {tuple(shape)}")
    if b * window == 1:
        q_stride = hq * d
    dtype = q.dtype
    code = cache_code = dtype_code(dtype)
    if key_cache.dtype == FP8_CACHE:
        _check_scales(k_scale, v_scale, q.device)
        cache_code = _lib.FP8_E4M3
    elif dtype != key_cache.dtype:
        raise _lib.VasrPaError(_lib.EINVAL_DTYPE, "q dtype must equal the cache dtype")
    _check_score_cache(score_cache, nb, hkv, bs, dev)
    if block_tables.dtype not in _INDEX32 or block_tables.dim() != 2 or block_tables.shape[0] != b:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "block_tables must be u32/i32 [B, cols]")
    if context_lens.dtype not in _INDEX32 or context_lens.shape != (b,):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "context_lens must be u32/i32 [B]")
    block_tables = block_tables.contiguous()
    context_lens = context_lens.contiguous()
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != dev or not out.is_contiguous():
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "out must be contiguous with q's shape and dtype")
    rows = window if score_rows is None else score_rows
    stream = _raw_stream(dev)
    ws = _SCRATCH.reserve(dev, stream, paged_attention_scored_workspace_bytes(b, window, rows, hq, hkv, d, bs,
                                                                              max_context_len))
    st = _lib.lib().vasr_pa_paged_attention_scored(
        out.data_ptr(), q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), score_cache.data_ptr(),
        block_tables.data_ptr(), context_lens.data_ptr(), b, window, rows, hq, hkv, d, bs, nb,
        block_tables.shape[1], max_context_len, softmax_scale, softcapping, decay, q_stride, code, cache_code,
        None if code == cache_code else k_scale.data_ptr(), None if code == cache_code else v_scale.data_ptr(),
        ws.data_ptr(), ws.numel(), stream)
    _lib.check(st, "paged_attention_scored")
    return out


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
    dev = _cuda_index(key_cache, value_cache, score_cache, block_tables, context_lens)
    nb, hkv, d, bs = cache_geometry(key_cache, value_cache)
    _check_score_cache(score_cache, nb, hkv, bs, dev)
    if block_tables.dtype not in _INDEX32 or block_tables.dim() != 2:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "block_tables must be u32/i32 [B, cols]")
    b, cols = block_tables.shape
    if context_lens.dtype not in _INDEX32 or context_lens.shape != (b,):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "context_lens must be u32/i32 [B]")
    block_tables = block_tables.contiguous()
    context_lens = context_lens.contiguous()
    out_ptr, out_cols = None, 0
    if out_block_tables is not None:
        if (out_block_tables.dtype not in _INDEX32 or out_block_tables.dim() != 2
                or out_block_tables.shape[0] != b or out_block_tables.get_device() != dev):
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "out_block_tables must be u32/i32 [B, cols] on the cache device")
        out_block_tables = out_block_tables.contiguous()
        out_ptr, out_cols = out_block_tables.data_ptr(), out_block_tables.shape[1]
    if budgets is not None:
        if budgets.dtype not in _INDEX32 or budgets.shape != (b,) or budgets.get_device() != dev:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "budgets must be u32/i32 [B] on the cache device")
        budgets = budgets.contiguous()
    code = _lib.FP8_E4M3 if key_cache.dtype == FP8_CACHE else _DTYPE_CODE.get(key_cache.dtype, -1)
    kept = block_tables.new_empty((b, hkv, max(budget, 0)), dtype=torch.int32)
    lens = block_tables.new_empty((b,), dtype=torch.int32)
    st = _lib.lib().vasr_pa_evict_kv(
        key_cache.data_ptr(), value_cache.data_ptr(), score_cache.data_ptr(), block_tables.data_ptr(), cols,
        out_ptr, out_cols, context_lens.data_ptr(), max_context_len,
        None if budgets is None else budgets.data_ptr(), budget, num_sink, num_recent, kept.data_ptr(),
        lens.data_ptr(), b, hkv, d, bs, nb, code, _raw_stream(dev))
    _lib.check(st, "evict_kv")
    return kept, lens
