"""Refusals of the rotary, scored-attention, eviction and verification entry points: every one is
answered on the host, before any CUDA call, by the status that its fault has."""
import ctypes

import pytest

from vasr_paged_attn import _lib

P = ctypes.c_void_p(256)      # never read: validation comes first
ODD = ctypes.c_void_p(257)
BIG = 1 << 40


def refuse(fn, base, cases):
    names = list(base)
    for change, status in cases:
        a = dict(base, **change)
        assert set(a) == set(names), change
        assert fn(*[a[n] for n in names]) == status, change


def sections(*s):
    return (ctypes.c_int32 * len(s))(*s)


ROPE = dict(cos=P, sin=P, max_position=1024, positions=P, axis_stride=64, sections=sections(24, 20, 20), axes=3,
            interleaved=1)


def test_mrope_refusals():
    base = dict(out=P, ots=1024, ohs=128, x=P, xts=1024, xhs=128, **ROPE, inverse=0, t=4, h=8, d=128, dtype=_lib.BF16,
                stream=None)
    refuse(_lib.lib().vasr_pa_mrope, base, [
        (dict(dtype=_lib.FP8_E4M3), _lib.EINVAL_DTYPE), (dict(t=-1), _lib.EINVAL_SHAPE),
        (dict(h=0), _lib.EINVAL_SHAPE), (dict(d=126), _lib.EINVAL_SHAPE), (dict(axes=0), _lib.EINVAL_SHAPE),
        (dict(axes=5), _lib.EINVAL_SHAPE), (dict(sections=None), _lib.EINVAL_SHAPE),
        (dict(sections=sections(70, -6, 0)), _lib.EINVAL_SHAPE), (dict(sections=sections(0, 0, 0)), _lib.EINVAL_SHAPE),
        (dict(sections=sections(10, 44, 10)), _lib.EINVAL_SHAPE),      # axis 1 would need 130 frequencies
        (dict(max_position=0), _lib.EINVAL_SHAPE), (dict(axis_stride=-1), _lib.EINVAL_SHAPE),
        (dict(ots=900), _lib.EINVAL_SHAPE), (dict(ohs=127), _lib.EINVAL_SHAPE),    # rows of out overlap
        (dict(cos=None), _lib.EINVAL_POINTER), (dict(x=None), _lib.EINVAL_POINTER), (dict(out=None), _lib.EINVAL_POINTER),
        (dict(x=ODD), _lib.EINVAL_ALIGN), (dict(sin=ODD), _lib.EINVAL_ALIGN), (dict(positions=ODD), _lib.EINVAL_ALIGN),
        (dict(t=0), _lib.OK)])


def test_mrope_append_refusals():
    base = dict(q_out=P, qkv=P, stride=4096, qw=P, kw=P, eps=1e-6, **ROPE, kc=P, vc=P, scores=P, slots=P, t=4, hq=16,
                hkv=8, d=128, bs=16, nb=10, dtype=_lib.BF16, cache=_lib.BF16, ks=None, vs=None, stream=None)
    refuse(_lib.lib().vasr_pa_fused_qk_norm_mrope_append, base, [
        (dict(dtype=9), _lib.EINVAL_DTYPE), (dict(cache=_lib.F16), _lib.EINVAL_DTYPE),
        (dict(bs=24), _lib.EINVAL_BLOCKSIZE), (dict(nb=0), _lib.EINVAL_SHAPE), (dict(hq=0), _lib.EINVAL_SHAPE),
        (dict(d=100), _lib.EINVAL_SHAPE), (dict(d=640, stride=20480), _lib.ENOT_SUPPORTED),
        (dict(stride=4095), _lib.EINVAL_SHAPE), (dict(t=-1), _lib.EINVAL_SHAPE),
        (dict(d=120, stride=3840, sections=sections(20, 20, 20), cache=_lib.FP8_E4M3, ks=P, vs=P), _lib.EINVAL_SHAPE),
        (dict(cache=_lib.FP8_E4M3), _lib.EINVAL_POINTER), (dict(qw=None), _lib.EINVAL_POINTER),
        (dict(kc=None), _lib.EINVAL_POINTER), (dict(slots=None), _lib.EINVAL_POINTER),
        (dict(kc=ctypes.c_void_p(264)), _lib.EINVAL_ALIGN), (dict(qkv=ODD), _lib.EINVAL_ALIGN),
        (dict(scores=ODD), _lib.EINVAL_ALIGN), (dict(sections=sections(30, 30, 30)), _lib.EINVAL_SHAPE),
        (dict(t=0), _lib.OK)])


def test_scored_refusals():
    lib = _lib.lib()
    size = lib.vasr_pa_paged_attention_scored_workspace_size
    need = size(4, 2, 1, 16, 8, 128, 16, 64)
    assert need > 0 and size(4, 2, 3, 16, 8, 128, 16, 64) == 0 and size(4, 2, 1, 16, 6, 128, 16, 64) == 0
    assert size(4, 2, 1, 16, 8, 128, 12, 64) == 0 and size(0, 2, 1, 16, 8, 128, 16, 64) == 0
    base = dict(out=P, q=P, kc=P, vc=P, scores=P, bt=P, ctx=P, b=4, w=2, rows=1, hq=16, hkv=8, d=128, bs=16, nb=10,
                cols=4, bound=64, scale=0.1, cap=1.0, decay=1.0, stride=2048, dtype=_lib.BF16, cache=_lib.BF16, ks=None,
                vs=None, ws=P, wsb=need, stream=None)
    refuse(lib.vasr_pa_paged_attention_scored, base, [
        (dict(dtype=7), _lib.EINVAL_DTYPE), (dict(cache=_lib.F32), _lib.EINVAL_DTYPE),
        (dict(bs=64), _lib.EINVAL_BLOCKSIZE), (dict(hq=12), _lib.EINVAL_SHAPE), (dict(w=0), _lib.EINVAL_SHAPE),
        (dict(rows=3), _lib.EINVAL_SHAPE), (dict(rows=0), _lib.EINVAL_SHAPE), (dict(cols=0), _lib.EINVAL_SHAPE),
        (dict(cap=0.0), _lib.EINVAL_SHAPE), (dict(decay=-0.5), _lib.EINVAL_SHAPE), (dict(decay=1.5), _lib.EINVAL_SHAPE),
        (dict(decay=float("nan")), _lib.EINVAL_SHAPE), (dict(stride=2047), _lib.EINVAL_SHAPE),
        (dict(b=70000), _lib.EINVAL_SHAPE), (dict(w=65), _lib.ENOT_SUPPORTED),
        (dict(scores=None), _lib.EINVAL_POINTER), (dict(cache=_lib.FP8_E4M3), _lib.EINVAL_POINTER),
        (dict(q=ctypes.c_void_p(264)), _lib.EINVAL_ALIGN), (dict(stride=2049), _lib.EINVAL_ALIGN),
        (dict(ws=None), _lib.EINVAL_WORKSPACE), (dict(wsb=need - 1), _lib.EINVAL_WORKSPACE),
        (dict(ws=ctypes.c_void_p(272)), _lib.EINVAL_ALIGN), (dict(b=0), _lib.OK)])


def test_evict_refusals():
    base = dict(kc=P, vc=P, scores=P, bt=P, cols=4, obt=None, ocols=0, ctx=P, bound=64, budgets=None, budget=32, sink=4,
                recent=8, kept=P, lens=P, b=4, hkv=8, d=128, bs=16, nb=10, dtype=_lib.BF16, stream=None)
    refuse(_lib.lib().vasr_pa_evict_kv, base, [
        (dict(dtype=5), _lib.EINVAL_DTYPE), (dict(bs=4), _lib.EINVAL_BLOCKSIZE), (dict(budget=0), _lib.EINVAL_SHAPE),
        (dict(sink=25), _lib.EINVAL_SHAPE), (dict(sink=-1), _lib.EINVAL_SHAPE), (dict(recent=-1), _lib.EINVAL_SHAPE),
        (dict(sink=0x7fffffff, recent=0x7fffffff), _lib.EINVAL_SHAPE), (dict(bound=0), _lib.EINVAL_SHAPE),
        (dict(obt=P, ocols=0), _lib.EINVAL_SHAPE), (dict(obt=P, ocols=1), _lib.EINVAL_SHAPE),  # 32 tokens need 2 blocks
        (dict(d=120, dtype=_lib.FP8_E4M3), _lib.EINVAL_SHAPE), (dict(kept=None), _lib.EINVAL_POINTER),
        (dict(lens=None), _lib.EINVAL_POINTER), (dict(vc=ctypes.c_void_p(264)), _lib.EINVAL_ALIGN),
        (dict(kept=ODD), _lib.EINVAL_ALIGN), (dict(b=0), _lib.OK)])


def test_evict_refuses_the_lengths_as_their_own_output():
    base = dict(kc=P, vc=P, scores=P, bt=P, cols=4, obt=None, ocols=0, ctx=P, bound=64, budgets=None, budget=32, sink=4,
                recent=8, kept=P, lens=P, b=4, hkv=8, d=128, bs=16, nb=10, dtype=_lib.BF16, stream=None)
    refuse(_lib.lib().vasr_pa_evict_kv, base, [(dict(), _lib.EINVAL_POINTER), (dict(b=0), _lib.OK)])


def test_verify_refusals():
    lib = _lib.lib()
    need = lib.vasr_pa_verify_draft_tokens_workspace_size(4, 3, 1000)
    assert need > 0 and lib.vasr_pa_verify_draft_tokens_workspace_size(0, 3, 1000) == 0
    base = dict(tokens=P, accepted=P, logits=P, lss=4000, lrs=1000, dtype=_lib.BF16, drafts=P, lens=None, probs=P,
                pss=3000, prs=1000, pdtype=_lib.F32, uniform=P, race=P, rss=1000, temps=None, temp=1.0, b=4, k=3, v=1000,
                ws=P, wsb=need, stream=None)
    refuse(lib.vasr_pa_verify_draft_tokens, base, [
        (dict(dtype=3), _lib.EINVAL_DTYPE), (dict(pdtype=3), _lib.EINVAL_DTYPE), (dict(v=0), _lib.EINVAL_SHAPE),
        (dict(v=BIG, lrs=BIG, prs=BIG), _lib.EINVAL_SHAPE), (dict(k=-1), _lib.EINVAL_SHAPE),
        (dict(lrs=999), _lib.EINVAL_SHAPE), (dict(prs=999), _lib.EINVAL_SHAPE), (dict(b=70000), _lib.EINVAL_SHAPE),
        (dict(race=None), _lib.EINVAL_POINTER), (dict(uniform=None), _lib.EINVAL_POINTER),
        (dict(drafts=None), _lib.EINVAL_POINTER), (dict(tokens=None), _lib.EINVAL_POINTER),
        (dict(logits=ODD), _lib.EINVAL_ALIGN), (dict(probs=ctypes.c_void_p(258)), _lib.EINVAL_ALIGN),
        (dict(ws=None), _lib.EINVAL_WORKSPACE), (dict(wsb=need - 1), _lib.EINVAL_WORKSPACE), (dict(b=0), _lib.OK)])


def test_python_entry_points_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from vasr_paged_attn import eviction, fused, speculative

    x = torch.zeros(2, 2, 128)
    pos = torch.zeros(3, 2, dtype=torch.int64)
    table = torch.zeros(8, 64)
    with pytest.raises(_lib.VasrPaError) as e:
        fused.mrope(x, table, table, pos, (24, 20, 20))
    assert e.value.status == _lib.EINVAL_POINTER
    kc, vc = torch.zeros(2, 1, 16, 16, 8, dtype=torch.bfloat16), torch.zeros(2, 1, 128, 16, dtype=torch.bfloat16)
    s, bt, n = torch.zeros(2, 1, 16), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(_lib.VasrPaError):
        eviction.evict_kv(kc, vc, s, bt, n, 16, 8, 0, 0)
    with pytest.raises(_lib.VasrPaError):
        eviction.paged_attention_scored(torch.zeros(1, 2, 128, dtype=torch.bfloat16), None, None, kc, vc, s, bt, n, 16, 0.1)
    with pytest.raises(_lib.VasrPaError):
        speculative.verify_draft_tokens(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), None, None, None)
