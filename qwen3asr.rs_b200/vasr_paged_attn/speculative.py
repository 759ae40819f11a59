"""Verification of drafted tokens on the device.

A drafter proposes K tokens a sequence, the target runs them in one window, and
``verify_draft_tokens`` keeps the prefix that leaves the target's distribution unchanged and draws
the token that follows. The reference decodes one greedy token a step
(vasr-models/src/model/generation.rs:443-460); ``temperature=0`` gives its tokens.
"""
from __future__ import annotations

import functools
from typing import Optional, Union

import torch

from . import _lib
from .mistralrs_paged_attn import StreamWorkspaces, _cuda_index, _raw_stream, dtype_code

_WORKSPACES = StreamWorkspaces("verify_draft_tokens")


@functools.lru_cache(maxsize=256)
def verify_draft_tokens_workspace_bytes(num_seqs: int, num_drafts: int, vocab: int) -> int:
    return int(_lib.lib().vasr_pa_verify_draft_tokens_workspace_size(num_seqs, num_drafts, vocab))


def reserve_verify_draft_tokens_workspace(device: torch.device, nbytes: int,
                                          stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Make sure the stream's workspace holds ``nbytes``; call before a CUDA-graph capture."""
    return _WORKSPACES.reserve_for(device, nbytes, stream)


def verify_draft_tokens(target_logits: torch.Tensor, draft_tokens: torch.Tensor,
                        draft_probs: Optional[torch.Tensor], uniform: Optional[torch.Tensor],
                        race: Optional[torch.Tensor], temperature: Union[float, torch.Tensor] = 1.0,
                        draft_lens: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens int32 [B, K + 1], accepted int32 [B]) of K drafted tokens a sequence.

    ``target_logits`` [B, K + 1, V] are the target's rows after 0, 1, ..., K drafts;
    ``draft_probs`` [B, K, V] what the drafter sampled from (None: it was certain of its tokens);
    ``uniform`` [B, K] in [0, 1) and ``race`` [B, V] ~ Exp(1) the random numbers (f32), which only
    a host-given temperature of 0 can leave out. Row b of tokens holds the accepted drafts, the
    next token, then -1. ``temperature`` is a number or f32 [B]; where it is 0 the row is greedy.
    ``draft_lens`` (int32 [B]) shortens drafts; K = 0 samples one token."""
    dev = _cuda_index(target_logits, draft_tokens)
    if target_logits.dim() != 3 or target_logits.stride(2) != 1:
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "target_logits must be [B, K + 1, V] with unit column stride")
    b, k1, vocab = target_logits.shape
    k = k1 - 1
    if draft_tokens.dtype != torch.int32 or draft_tokens.shape != (b, k):
        raise _lib.VasrPaError(_lib.EINVAL_SHAPE, f"draft_tokens must be int32 [{b}, {k}]")
    draft_tokens = draft_tokens.contiguous()
    probs_ptr, probs_seq, probs_row, probs_code = None, 0, 0, 0
    if draft_probs is not None:
        if draft_probs.shape != (b, k, vocab) or draft_probs.stride(2) != 1 or draft_probs.get_device() != dev:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "draft_probs must be [B, K, V] with unit column stride")
        probs_ptr, probs_code = draft_probs.data_ptr(), dtype_code(draft_probs.dtype)
        probs_seq, probs_row, _ = draft_probs.stride()
    uniform_ptr = None
    if uniform is not None:
        if uniform.dtype != torch.float32 or uniform.shape != (b, k) or uniform.get_device() != dev:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "uniform must be f32 [B, K]")
        uniform = uniform.contiguous()
        uniform_ptr = uniform.data_ptr()
    race_ptr, race_seq = None, 0
    if race is not None:
        if (race.dtype != torch.float32 or race.shape != (b, vocab) or race.get_device() != dev
                or race.stride(1) != 1):
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "race must be f32 [B, V] with unit column stride")
        race_ptr, race_seq = race.data_ptr(), race.stride(0)
    temps = temps_ptr = None
    if isinstance(temperature, torch.Tensor):
        if temperature.dtype != torch.float32 or temperature.shape != (b,) or temperature.get_device() != dev:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "temperature must be a number or f32 [B]")
        temps, temperature = temperature.contiguous(), 1.0
        temps_ptr = temps.data_ptr()
    lens_ptr = None
    if draft_lens is not None:
        if draft_lens.dtype != torch.int32 or draft_lens.shape != (b,) or draft_lens.get_device() != dev:
            raise _lib.VasrPaError(_lib.EINVAL_SHAPE, "draft_lens must be int32 [B]")
        draft_lens = draft_lens.contiguous()
        lens_ptr = draft_lens.data_ptr()
    tokens = draft_tokens.new_empty((b, k1))
    accepted = draft_tokens.new_empty((b,))
    stream = _raw_stream(dev)
    ws = _WORKSPACES.reserve(dev, stream, verify_draft_tokens_workspace_bytes(b, k, vocab))
    logits_seq, logits_row, _ = target_logits.stride()
    st = _lib.lib().vasr_pa_verify_draft_tokens(
        tokens.data_ptr(), accepted.data_ptr(), target_logits.data_ptr(), logits_seq, logits_row,
        dtype_code(target_logits.dtype), draft_tokens.data_ptr(), lens_ptr, probs_ptr, probs_seq, probs_row,
        probs_code, uniform_ptr, race_ptr, race_seq, temps_ptr, temperature, b, k, vocab, ws.data_ptr(),
        ws.numel(), stream)
    _lib.check(st, "verify_draft_tokens")
    return tokens, accepted
