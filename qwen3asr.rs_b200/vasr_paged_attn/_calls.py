"""The module ``_vasr_calls``: tensor checks, result allocation and the C-ABI call in one crossing.

Operators that are called once a layer and decode step go through it; a ctypes call of 20 to 30
arguments behind the same checks in Python cost more host time than their kernels take. Loading
fails loudly if the module has not been built.
"""
from __future__ import annotations

import ctypes
import importlib
import sys

import torch  # noqa: F401  (the module links against it)

from . import _lib

_NAMES = ("vasr_pa_mrope", "vasr_pa_fused_qk_norm_mrope_append", "vasr_pa_paged_attention_scored",
          "vasr_pa_paged_attention_scored_workspace_size", "vasr_pa_evict_kv", "vasr_pa_verify_draft_tokens",
          "vasr_pa_verify_draft_tokens_workspace_size")
_MODULE = None

# kinds of workspaces (reserve)
SCORED, VERIFY = 0, 1


def calls():
    """The module, bound to the kernel library that the ctypes binding has loaded."""
    global _MODULE
    if _MODULE is None:
        where = str(_lib._PKG_ROOT / "lib")
        if where not in sys.path:
            sys.path.insert(0, where)
        module = importlib.import_module("_vasr_calls")
        dll = _lib.lib()
        module.bind(_lib.VasrPaError, *(ctypes.cast(getattr(dll, n), ctypes.c_void_p).value for n in _NAMES))
        _MODULE = module
    return _MODULE


def reserve(kind: int, device, nbytes: int, stream) -> torch.Tensor:
    """The (device, stream) workspace of one kind of call, at least ``nbytes`` long."""
    s = stream if stream is not None else torch.cuda.current_stream(torch.device(device))
    return calls().reserve(kind, s.device.index, s.cuda_stream, nbytes)
