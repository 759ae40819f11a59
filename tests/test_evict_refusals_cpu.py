"""Refusals of the eviction's entry point, one fault at a time: each case's base call has nothing
else to refuse (with no sequences it is accepted)."""
import ctypes

import pytest

from test_operators_capi_cpu import ODD, P, refuse
from vasr_paged_attn import _lib

LENS = ctypes.c_void_p(512)  # of its own: the old lengths are no place for the new ones
BASE = dict(kc=P, vc=P, scores=P, bt=P, cols=4, obt=None, ocols=0, ctx=P, bound=64, budgets=None, budget=32, sink=4,
            recent=8, kept=P, lens=LENS, b=4, hkv=8, d=128, bs=16, nb=10, dtype=_lib.BF16, stream=None)


def call(**change):
    refuse(_lib.lib().vasr_pa_evict_kv, BASE, [(change, change.pop("status"))])


@pytest.mark.parametrize("name", ["kc", "vc", "scores", "bt", "ctx", "kept", "lens"])
def test_null_pointers(name):
    call(**{name: None}, status=_lib.EINVAL_POINTER)


@pytest.mark.parametrize("name", ["kc", "vc", "scores", "bt", "ctx", "kept", "lens", "budgets"])
def test_misaligned_pointers(name):
    call(**{name: ODD}, status=_lib.EINVAL_ALIGN)


def test_the_lengths_as_their_own_output():
    call(lens=P, status=_lib.EINVAL_POINTER)


def test_misaligned_output_tables():
    call(obt=ODD, ocols=2, status=_lib.EINVAL_ALIGN)


def test_no_sequences():
    call(b=0, status=_lib.OK)
    call(b=0, kept=None, lens=None, status=_lib.OK)
