"""Verification of drafted tokens on the device.

A drafter proposes K tokens a sequence, the target runs them in one window, and
``verify_draft_tokens`` keeps the prefix that leaves the target's distribution unchanged and draws
the token that follows. The reference decodes one greedy token a step
(vasr-models/src/model/generation.rs:443-460); ``temperature=0`` gives its tokens.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _calls, _lib
from ._calls import calls


def verify_draft_tokens_workspace_bytes(num_seqs: int, num_drafts: int, vocab: int) -> int:
    return int(_lib.lib().vasr_pa_verify_draft_tokens_workspace_size(num_seqs, num_drafts, vocab))


def reserve_verify_draft_tokens_workspace(device: torch.device, nbytes: int,
                                          stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Make sure the stream's workspace holds ``nbytes``, so that calls on it do not have to grow it.

    Calls that a CUDA graph captures take theirs from the graph's own memory."""
    return _calls.reserve(_calls.VERIFY, device, nbytes, stream)


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
    return calls().verify(target_logits, draft_tokens, draft_probs, uniform, race, temperature, draft_lens)
