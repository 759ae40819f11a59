"""Rotary embedding with several position axes against its formula in 64 bits.

Tolerance: the f32 arithmetic of a norm and a rotation is off by at most about (2 + log2 D) f32
roundoffs of the row's largest rotated value, taken as 2^-20 of it; the store then rounds once.
"""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import _lib, fused, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu
MAXPOS = 512


def tables(half, dev):
    inv = 1e4 ** (-np.arange(half) / half)
    ang = np.arange(MAXPOS)[:, None] * inv
    cos, sin = torch.from_numpy(np.cos(ang)).float(), torch.from_numpy(np.sin(ang)).float()
    return cos.to(dev), sin.to(dev)


def close(got, want, dtype, slack=0.0):
    got = ref.f64(got)
    tol = ref.ROUND[dtype] * np.abs(want) + ref.TINY[dtype] + 2.0 ** -20 * (np.abs(want).max(-1, keepdims=True) + 1) + slack
    return bool((np.abs(got - want) <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,h,d,sections,interleaved", [
    (1, 1, 128, (24, 20, 20), True), (37, 5, 128, (24, 20, 20), False), (300, 3, 64, (12, 10, 10), True),
    (9, 2, 256, (48, 40, 40), False), (65, 4, 96, (11, 11, 10), True), (17, 2, 128, (16, 0, 8), False),
    (33, 3, 80, (5, 7), False), (5, 2, 128, (64,), True), (40, 2, 128, (16, 16, 16, 16), True),
    (21, 3, 128, (11, 10, 10), True)])
def test_rotation_and_its_inverse(cuda_device, dtype, t, h, d, sections, interleaved):
    rng = np.random.default_rng(t * 131 + d)
    cos, sin = tables(sum(sections), cuda_device)
    pos = rng.integers(0, MAXPOS, (len(sections), t))
    x = torch.from_numpy(rng.standard_normal((t, h, d), np.float32) * 3).to(dtype).to(cuda_device)
    p = torch.from_numpy(pos).to(cuda_device)
    for inverse in (False, True):
        y = fused.mrope(x, cos, sin, p, sections, interleaved=interleaved, inverse=inverse)
        want = ref.rotate(ref.f64(x), ref.f64(cos), ref.f64(sin), pos, sections, interleaved, inverse)
        assert close(y, want, dtype)
        tail = 2 * sum(sections)
        assert torch.equal(y[..., tail:], x[..., tail:])
    assert pa.device_error() == 0


def test_strided_rows_in_place_and_head_major(cuda_device):
    rng = np.random.default_rng(3)
    t, h, d, sections = 19, 4, 128, (24, 20, 20)
    cos, sin = tables(64, cuda_device)
    pos = rng.integers(0, MAXPOS, (3, 2 * t))
    p = torch.from_numpy(pos).to(cuda_device)[:, ::2]           # strided in tokens: copied
    pos = pos[:, ::2]
    wide = torch.from_numpy(rng.standard_normal((t, h * d + 24), np.float32)).to(cuda_device)
    x = wide[:, 8:8 + h * d].view(t, h, d)                       # 32-byte offset, padded rows
    want = ref.rotate(ref.f64(x), ref.f64(cos), ref.f64(sin), pos, sections, True)
    assert close(fused.mrope(x, cos, sin, p, sections), want, torch.float32)
    odd = torch.from_numpy(rng.standard_normal((t * h * d + 1,), np.float32)).to(torch.bfloat16).to(cuda_device)
    y = odd[1:].view(t, h, d)                                    # 2-byte aligned
    want16 = ref.rotate(ref.f64(y), ref.f64(cos), ref.f64(sin), pos, sections, True)
    assert close(fused.mrope(y, cos, sin, p, sections), want16, torch.bfloat16)
    major = x.transpose(0, 1).contiguous().transpose(0, 1)       # [H, T, D] in memory
    out = torch.empty_like(major)
    assert out.stride() == major.stride()
    assert close(fused.mrope(major, cos, sin, p, sections, out=out), want, torch.float32)
    kept = wide.clone()
    fused.mrope(x, cos, sin, p, sections, out=x)                 # in place
    assert close(x, want, torch.float32)
    assert torch.equal(wide[:, :8], kept[:, :8]) and torch.equal(wide[:, 8 + h * d:], kept[:, 8 + h * d:])


def test_equal_axes_by_a_broadcast_and_gradient(cuda_device):
    """One position stream expanded over the axes equals a single axis; the gradient of
    sum(y g) is the inverse rotation of g, by the formula and by differences."""
    rng = np.random.default_rng(4)
    t, h, d, sections = 7, 2, 64, (12, 10, 10)
    cos, sin = tables(32, cuda_device)
    one = torch.from_numpy(rng.integers(0, MAXPOS, (1, t))).to(cuda_device)
    x = torch.from_numpy(rng.standard_normal((t, h, d), np.float32)).to(cuda_device)
    y = fused.mrope(x, cos, sin, one.expand(3, t), sections)
    assert torch.equal(y, fused.mrope(x, cos, sin, one, (32,)))
    pos = torch.from_numpy(rng.integers(0, MAXPOS, (3, t))).to(cuda_device)
    g = torch.from_numpy(rng.standard_normal((t, h, d), np.float32)).to(cuda_device)
    grad = fused.mrope(g, cos, sin, pos, sections, inverse=True)
    a = (ref.f64(cos), ref.f64(sin), pos.cpu().numpy(), sections, True)
    for _ in range(8):  # the map is linear: a difference is exact up to rounding
        e = np.zeros((t, h, d))
        at = tuple(rng.integers(0, s) for s in (t, h, d))
        e[at] = 0.5
        diff = ((ref.rotate(ref.f64(x) + e, *a) - ref.rotate(ref.f64(x) - e, *a)) * ref.f64(g)).sum()
        assert abs(diff - ref.f64(grad)[at]) <= 2.0 ** -19 * 4


def append_case(rng, t, hq, hkv, d, bs, dtype, dev, run):
    nb = -(-t // run) * (-(-run // bs) + 1) + 2
    qkv = torch.from_numpy(rng.standard_normal((t, (hq + 2 * hkv) * d), np.float32) * 2).to(dtype).to(dev)
    # runs of consecutive tokens that start anywhere in a page, blocks in seeded order
    ids = rng.permutation(np.arange(1, nb))
    slots, used = [], 0
    while len(slots) < t:
        n = min(run, t - len(slots))
        off = int(rng.integers(0, bs)) if run > 1 else int(rng.integers(0, bs))
        need = -(-(off + n) // bs)
        blk = ids[used:used + need]
        used += need
        j = off + np.arange(n)
        slots += (blk[j // bs] * bs + j % bs).tolist()
    return qkv, np.array(slots), nb


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None),
                                         (torch.bfloat16, torch.float8_e4m3fn), (torch.float32, torch.float8_e4m3fn)])
@pytest.mark.parametrize("t,run,hq,hkv,d,bs,sections,norm", [
    (1, 1, 16, 8, 128, 16, (24, 20, 20), True), (64, 1, 16, 8, 128, 16, (24, 20, 20), True),
    (131, 57, 4, 1, 128, 8, (24, 20, 20), True), (100, 33, 6, 2, 64, 32, (12, 10, 10), False),
    (70, 70, 3, 3, 256, 16, (30, 20, 20), True), (45, 7, 5, 5, 96, 16, (11, 11, 10), True),
    (600, 200, 16, 8, 128, 16, (24, 20, 20), True), (515, 130, 2, 1, 128, 32, (16, 8, 8), True)])
def test_fused_append(cuda_device, dtype, cache, t, run, hq, hkv, d, bs, sections, norm):
    dev = cuda_device
    cdt = cache or dtype
    if cache is not None and d % 16:
        pytest.skip("fp8 pages hold 16 dims a chunk")
    rng = np.random.default_rng(t * 7 + d)
    cos, sin = tables(sum(sections), dev)
    qkv, slots, nb = append_case(rng, t, hq, hkv, d, bs, dtype, dev, run)
    slots[::9] = -1                                              # padded rows
    pos = rng.integers(0, MAXPOS, (len(sections), t))
    x = 16 // torch.empty((), dtype=cdt).element_size()
    kc = torch.full((nb, hkv, d // x, bs, x), float("nan")).to(cdt).to(dev)
    vc = torch.full((nb, hkv, d, bs), float("nan")).to(cdt).to(dev)
    before = ref.raw(kc), ref.raw(vc)
    scores = torch.full((nb, hkv, bs), 7.0, device=dev)
    qw = torch.from_numpy(1 + 0.1 * rng.standard_normal(d)).to(dtype).to(dev) if norm else None
    kw = torch.from_numpy(1 + 0.1 * rng.standard_normal(d)).to(dtype).to(dev) if norm else None
    ks = torch.tensor([0.03], device=dev) if cache else None
    vs = torch.tensor([0.05], device=dev) if cache else None
    q = fused.qk_norm_mrope_append(qkv, qw, kw, 1e-6, cos, sin, torch.from_numpy(pos).to(dev), sections, kc, vc,
                                   torch.from_numpy(slots).to(dev), hq, k_scale=ks, v_scale=vs, score_cache=scores)
    r = ref.f64(qkv).reshape(t, hq + 2 * hkv, d)
    qn, kn, vn = r[:, :hq], r[:, hq:hq + hkv], r[:, hq + hkv:]
    if norm:
        qn, kn = ref.rms_norm(qn, ref.f64(qw), 1e-6), ref.rms_norm(kn, ref.f64(kw), 1e-6)
    a = (ref.f64(cos), ref.f64(sin), pos, sections, True)
    assert close(q, ref.rotate(qn, *a), dtype)
    kt, vt = ref.token_major(kc, vc)
    live = slots >= 0
    want_k, want_v = ref.rotate(kn, *a)[live], vn[live]
    if cache is not None:
        want_k, want_v = (np.clip(w / s, -448, 448) for w, s in ((want_k, float(ks)), (want_v, float(vs))))
    assert close(torch.from_numpy(kt[slots[live]]), want_k, cdt)
    assert close(torch.from_numpy(vt[slots[live]]), want_v, cdt)
    if cache is None:
        assert np.array_equal(vt[slots[live]], vn[live])
    # nothing else was touched, and the scores of the appended slots are cleared
    touched = np.zeros(nb * bs, bool)
    touched[slots[live]] = True
    for got, old, spread in ((ref.raw(kc), before[0], (0, 3, 1, 2, 4)), (ref.raw(vc), before[1], (0, 3, 1, 2))):
        g, o = (z.transpose(spread).reshape(nb * bs, -1) for z in (got, old))
        assert np.array_equal(g[~touched], o[~touched])
    s = scores.cpu().numpy().transpose(0, 2, 1).reshape(nb * bs, hkv)
    assert (s[touched] == 0).all() and (s[~touched] == 7).all()
    assert pa.device_error() == 0


def test_large_append_matches_small_ones(cuda_device):
    """A prompt-sized call gives the bits of the same tokens appended a few at a time."""
    dev, t, hq, hkv, d, bs, sections = cuda_device, 4500, 4, 2, 128, 16, (24, 20, 20)
    rng = np.random.default_rng(8)
    cos, sin = tables(64, dev)
    qkv, slots, nb = append_case(rng, t, hq, hkv, d, bs, torch.bfloat16, dev, 700)
    slots[100:110] = -1
    slots = torch.from_numpy(slots).to(dev)
    pos = torch.from_numpy(rng.integers(0, MAXPOS, (3, t))).to(dev)
    w = torch.ones(d, dtype=torch.bfloat16, device=dev)
    got = []
    for step in (t, 50):
        kc = torch.zeros(nb, hkv, d // 8, bs, 8, dtype=torch.bfloat16, device=dev)
        vc = torch.zeros(nb, hkv, d, bs, dtype=torch.bfloat16, device=dev)
        q = [fused.qk_norm_mrope_append(qkv[i:i + step], w, w, 1e-6, cos, sin, pos[:, i:i + step], sections, kc, vc,
                                        slots[i:i + step], hq) for i in range(0, t, step)]
        got.append((torch.cat(q), kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_ids_out_of_range_are_flagged_and_skipped(cuda_device):
    dev, t, hq, hkv, d, bs, nb = cuda_device, 6, 2, 1, 128, 16, 4
    cos, sin = tables(64, dev)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, device=dev).to(torch.bfloat16)
    kc = torch.zeros(nb, hkv, 16, bs, 8, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros(nb, hkv, d, bs, dtype=torch.bfloat16, device=dev)
    slots = torch.tensor([3, nb * bs, 1 << 40, 5, -1, -(1 << 40)], device=dev)
    pos = torch.zeros(3, t, dtype=torch.int64, device=dev)
    args = (1e-6, cos, sin, pos, (24, 20, 20), kc, vc, slots, hq)
    pa.device_error()
    fused.qk_norm_mrope_append(qkv, None, None, *args)
    assert pa.device_error() == _lib.DERR_SLOT_RANGE
    used = (vc != 0).any(2)[:, 0].flatten().nonzero().flatten().tolist()
    assert used == [3, 5]
    pos[1, 2], pos[2, 3] = MAXPOS, -1                            # clamped to the table's ends
    q = fused.mrope(qkv.view(t, -1, d), cos, sin, pos, (24, 20, 20))
    assert pa.device_error() == _lib.DERR_POSITION_RANGE
    want = ref.rotate(ref.f64(qkv).reshape(t, -1, d), ref.f64(cos), ref.f64(sin),
                      pos.clamp(0, MAXPOS - 1).cpu().numpy(), (24, 20, 20), True)
    assert close(q, want, torch.bfloat16)


def test_other_stream_and_empty_call(cuda_device):
    dev = cuda_device
    cos, sin = tables(64, dev)
    x = torch.randn(50, 3, 128, device=dev)
    pos = torch.randint(0, MAXPOS, (3, 50), device=dev)
    want = fused.mrope(x, cos, sin, pos, (24, 20, 20))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fused.mrope(x, cos, sin, pos, (24, 20, 20))
    s.synchronize()
    assert torch.equal(got, want)
    assert fused.mrope(x[:0], cos, sin, pos[:, :0], (24, 20, 20)).shape == (0, 3, 128)
