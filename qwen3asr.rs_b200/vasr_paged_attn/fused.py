"""Fused pre-attention step: q/k RMSNorm + rotary embedding + KV append (one launch).

Replaces the per-layer chain of vasr-models/src/model/thinker_text.rs:1041-1109
(q_norm, k_norm, mRoPE — 1-D RoPE for equal position streams — and
reshape_and_cache) with ``vasr_pa_fused_qk_norm_rope_append``; the ``mrope``
forms take one position per axis (time, height, width) and token.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence

import torch

from . import _lib
from .mistralrs_paged_attn import (FP8_CACHE, _check_scales, _cuda_index, _raw_stream, _require_cuda,
                                   _stream, cache_geometry, dtype_code)


def qk_norm_rope_append(qkv: torch.Tensor, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor,
                        eps: float, cos_table: torch.Tensor, sin_table: torch.Tensor,
                        positions: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                        slot_mapping: torch.Tensor, num_heads: int,
                        q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv [T, (Hq + 2 Hkv) * D] -> q [T, Hq, D]; k and v are appended to the pages."""
    dev = _require_cuda(qkv, key_cache, value_cache, positions, slot_mapping, cos_table, sin_table)
    nb, hkv, d, bs = cache_geometry(key_cache, value_cache)
    t = int(qkv.shape[0])
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (num_heads + 2 * hkv) * d:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "qkv must be [T, (Hq + 2 Hkv) * D] with unit column stride")
    if cos_table.dtype != torch.float32 or sin_table.shape != cos_table.shape or cos_table.shape[1] != d // 2:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "cos/sin tables must be f32 [max_position, D / 2]")
    if positions.dtype != torch.int64 or slot_mapping.dtype != torch.int64:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "positions / slot_mapping must be int64")
    if q_out is None:
        q_out = torch.empty((t, num_heads, d), dtype=qkv.dtype, device=dev)
    st = _lib.lib().vasr_pa_fused_qk_norm_rope_append(
        q_out.data_ptr(), qkv.data_ptr(), qkv.stride(0), q_norm_weight.data_ptr(),
        k_norm_weight.data_ptr(), float(eps), cos_table.contiguous().data_ptr(),
        sin_table.contiguous().data_ptr(), int(cos_table.shape[0]), positions.contiguous().data_ptr(),
        key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.contiguous().data_ptr(), t,
        num_heads, hkv, d, bs, nb, dtype_code(qkv.dtype), _stream(dev))
    _lib.check(st, "fused_qk_norm_rope_append")
    return q_out


@functools.lru_cache(maxsize=64)
def _sections(sections: tuple) -> tuple:
    """(C array, its address, axes, rotated pairs) of the axis sections."""
    held = (ctypes.c_int32 * len(sections))(*sections)
    return held, ctypes.addressof(held), len(sections), sum(sections)


def _mrope_tables(cos_table, sin_table, positions, sections, tokens: int):
    """Checks shared by the multi-axis forms; (positions with unit token stride, axis stride)."""
    _, _, axes, half = sections
    shape = cos_table.shape
    if (cos_table.dtype != torch.float32 or sin_table.dtype != torch.float32 or len(shape) != 2
            or shape[1] != half or sin_table.shape != shape):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "cos/sin tables must be f32 [max_position, sum(sections)]")
    if not (cos_table.is_contiguous() and sin_table.is_contiguous()):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "cos/sin tables must be contiguous")
    if positions.dtype != torch.int64 or positions.shape != (axes, tokens):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "positions must be int64 [axes, T]")
    axis_stride, token_stride = positions.stride()
    if token_stride != 1 and tokens > 1:
        return positions.contiguous(), tokens
    return positions, axis_stride


def qk_norm_mrope_append(qkv: torch.Tensor, q_norm_weight: Optional[torch.Tensor],
                         k_norm_weight: Optional[torch.Tensor], eps: float, cos_table: torch.Tensor,
                         sin_table: torch.Tensor, positions: torch.Tensor, sections: Sequence[int],
                         key_cache: torch.Tensor, value_cache: torch.Tensor,
                         slot_mapping: torch.Tensor, num_heads: int, interleaved: bool = True,
                         k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                         score_cache: Optional[torch.Tensor] = None,
                         q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv [T, (Hq + 2 Hkv) * D] -> q [T, Hq, D]; k and v are appended to the pages.

    q and k get a per-head RMSNorm (no norm when both weights are None) and the rotation by
    ``positions`` [axes, T] (int64): frequency i of the sum(sections) rotated pairs takes the axis
    that ``sections`` gives it, laid out one section after another or interleaved (frequencies a,
    a + n, ... belong to axis a of n, what is left over to axis 0). One rounding, at the end.
    Negative slots are not appended. fp8 pages need k_scale / v_scale. ``score_cache``
    [num_blocks, Hkv, block_size] (f32) is set to 0 at every appended slot, as
    ``eviction.paged_attention_scored`` expects of new tokens."""
    dev = _cuda_index(qkv, key_cache, value_cache, positions, slot_mapping, cos_table, sin_table)
    nb, hkv, d, bs = cache_geometry(key_cache, value_cache)
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (num_heads + 2 * hkv) * d:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "qkv must be [T, (Hq + 2 Hkv) * D] with unit column stride")
    t, width = qkv.shape
    sections = _sections(tuple(sections))
    positions, axis_stride = _mrope_tables(cos_table, sin_table, positions, sections, t)
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (t,):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "slot_mapping must be int64 [T]")
    slot_mapping = slot_mapping.contiguous()
    dtype = qkv.dtype
    code = cache_code = dtype_code(dtype)
    if key_cache.dtype == FP8_CACHE:
        _check_scales(k_scale, v_scale, qkv.device)
        cache_code = _lib.FP8_E4M3
    elif key_cache.dtype != dtype:
        raise _lib.VasrPaError(_lib.EINVAL_DTYPE, "qkv dtype must equal the cache dtype")
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise _lib.VasrPaError(_lib.EINVAL_POINTER, "q and k norm weights go together")
    if q_norm_weight is not None:
        for w in (q_norm_weight, k_norm_weight):
            if w.dtype != dtype or w.shape != (d,) or w.get_device() != dev or not w.is_contiguous():
                raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "norm weights must be [D] of qkv's dtype on its device")
    if score_cache is not None:
        _check_score_cache(score_cache, nb, hkv, bs, dev)
    if q_out is None:
        q_out = qkv.new_empty((t, num_heads, d))
    elif (q_out.shape != (t, num_heads, d) or q_out.dtype != dtype or q_out.get_device() != dev
          or not q_out.is_contiguous()):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "q_out must be a contiguous [T, Hq, D] of qkv's dtype")
    st = _lib.lib().vasr_pa_fused_qk_norm_mrope_append(
        q_out.data_ptr(), qkv.data_ptr(), qkv.stride(0) if t > 1 else width,
        None if q_norm_weight is None else q_norm_weight.data_ptr(),
        None if k_norm_weight is None else k_norm_weight.data_ptr(), eps, cos_table.data_ptr(),
        sin_table.data_ptr(), cos_table.shape[0], positions.data_ptr(), axis_stride, sections[1], sections[2],
        interleaved, key_cache.data_ptr(), value_cache.data_ptr(),
        None if score_cache is None else score_cache.data_ptr(), slot_mapping.data_ptr(), t, num_heads, hkv, d,
        bs, nb, code, cache_code, None if code == cache_code else k_scale.data_ptr(),
        None if code == cache_code else v_scale.data_ptr(), _raw_stream(dev))
    _lib.check(st, "fused_qk_norm_mrope_append")
    return q_out


def _check_score_cache(score_cache: torch.Tensor, nb: int, hkv: int, bs: int, dev: int) -> None:
    if (score_cache.dtype != torch.float32 or score_cache.shape != (nb, hkv, bs) or score_cache.get_device() != dev
            or not score_cache.is_contiguous()):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE,
                               f"score_cache must be a contiguous f32 [{nb}, {hkv}, {bs}] on the cache device")


def mrope(x: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
          sections: Sequence[int], interleaved: bool = True, inverse: bool = False,
          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate x [T, H, D] by ``positions`` [axes, T] (see ``qk_norm_mrope_append``).

    ``inverse`` turns back; as the rotation is orthogonal that is also the gradient: with
    y = mrope(x), dL/dx = mrope(dL/dy, inverse=True). ``out`` may be x; dims past 2 * sum(sections)
    pass unchanged."""
    dev = _cuda_index(x, cos_table, sin_table, positions)
    if x.dim() != 3 or x.stride(2) != 1:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "x must be [T, H, D] with unit dim stride")
    t, h, d = x.shape
    sections = _sections(tuple(sections))
    positions, axis_stride = _mrope_tables(cos_table, sin_table, positions, sections, t)
    if out is None:
        out = x.new_empty((t, h, d))
    elif out.shape != x.shape or out.dtype != x.dtype or out.get_device() != dev or out.stride(2) != 1:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "out must have x's shape and dtype, with unit dim stride")
    out_token, out_head, _ = out.stride()
    x_token, x_head, _ = x.stride()
    st = _lib.lib().vasr_pa_mrope(
        out.data_ptr(), out_token, out_head, x.data_ptr(), x_token, x_head, cos_table.data_ptr(),
        sin_table.data_ptr(), cos_table.shape[0], positions.data_ptr(), axis_stride, sections[1], sections[2],
        interleaved, inverse, t, h, d, dtype_code(x.dtype), _raw_stream(dev))
    _lib.check(st, "mrope")
    return out
