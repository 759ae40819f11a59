"""Scored decode attention against its formula in 64 bits.

Tolerances. A raw score is an f32 sum of D products: off by at most D 2^-23 of sum |q k| scale
(tensor cores may truncate, hence 2^-23), about 2^-16 `reach` for D = 128, and a weight by that
fraction of itself, plus a few roundoffs of exp2 and of the sums: 2^-18. The weights that multiply
V may be rounded to the query's type (f16 over fp8 pages), the output is rounded once:
|out error| <= u (max |v| + |out|) + weight error max |v|.
"""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import _lib, eviction, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def check(dev, dtype, cache, lens, hq, hkv, d, bs, window=1, rows=None, softcap=1.0, decay=1.0, seed=0,
          bound=None, extra_cols=0):
    rng = np.random.default_rng(seed)
    kc, vc, tables = ref.make_pool(rng, lens, hkv, d, bs, cache, dev, extra_cols=extra_cols)
    q = torch.from_numpy(rng.standard_normal((len(lens), window, hq, d), np.float32)).to(dtype).to(dev)
    scores = torch.from_numpy(rng.random((kc.shape[0], hkv, bs), np.float32) * 0.1).to(dev)
    old = scores.clone()
    fp8 = cache == FP8
    ks = torch.tensor([0.7], device=dev) if fp8 else None
    vs = torch.tensor([1.6], device=dev) if fp8 else None
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor(list(lens), dtype=torch.int32, device=dev)
    bound = max(max(lens), 1) if bound is None else bound
    args = (bt, ctx, bound, d ** -0.5, softcap)
    out = eviction.paged_attention_scored(q, ks, vs, kc, vc, scores, *args, decay=decay, score_rows=rows)
    want, want_s, added, reach = ref.scored(q, kc, vc, old, tables, lens, d ** -0.5, softcap, decay, rows,
                                            ref.f64(ks)[0] if fp8 else 1.0, ref.f64(vs)[0] if fp8 else 1.0)
    rel = d * 2.0 ** -23 * reach + 2.0 ** -18
    vmax = np.nanmax(np.abs(ref.f64(vc))) * (1.6 if fp8 else 1.0)
    got = ref.f64(out)
    up = 2.0 ** -11 if fp8 and dtype != torch.float32 else ref.ROUND[dtype]
    tol = up * vmax + ref.ROUND[dtype] * np.abs(want) + rel * vmax
    assert (np.abs(got - want) <= tol).all(), float(np.nanmax(np.abs(got - want) / tol))
    tol = rel * added + 2.0 ** -22 * np.abs(want_s)
    assert (np.abs(ref.f64(scores) - want_s) <= tol).all()
    # untouched scores keep their bits
    idle = np.ones(scores.shape, bool).transpose(0, 2, 1).reshape(-1, hkv).copy()
    for i, n in enumerate(lens):
        idle[ref.slots_of(tables[i], int(n), bs)] = False
    same = (ref.raw(scores) == ref.raw(old)).transpose(0, 2, 1).reshape(-1, hkv)
    assert same[idle].all()
    assert pa.device_error() == 0
    # the same call on the same inputs gives the same bits
    again = old.clone()
    out2 = eviction.paged_attention_scored(q, ks, vs, kc, vc, again, *args, decay=decay, score_rows=rows)
    assert torch.equal(out, out2) and torch.equal(scores, again)
    return q, kc, vc, old, bt, ctx


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
         (torch.bfloat16, FP8), (torch.float16, FP8)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (4, 4), (8, 2), (8, 1)])
def test_single_token(cuda_device, dtype, cache, bs, hq, hkv):
    check(cuda_device, dtype, cache, (1, bs, bs + 1, 257, 15, 700, 0), hq, hkv, 128, bs, seed=bs + hq)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("window,rows,hq,hkv", [(2, 1, 4, 2), (5, 1, 16, 8), (5, 5, 16, 8), (8, 3, 4, 2), (3, 2, 6, 1),
                                                (16, 16, 2, 2), (4, 4, 16, 2)])
def test_window(cuda_device, dtype, cache, window, rows, hq, hkv):
    check(cuda_device, dtype, cache, (1, 3, 16, 17, window, 301, 64, 0), hq, hkv, 128, 16, window=window, rows=rows,
          seed=window)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_long_context_and_loose_bound(cuda_device, dtype, cache):
    check(cuda_device, dtype, cache, (9001, 2, 1025), 4, 2, 128, 16, bound=20000, extra_cols=700, seed=5)
    check(cuda_device, dtype, cache, (3000, 1024, 2049), 2, 1, 128, 32, window=3, seed=6)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_other_head_dims(cuda_device, dtype, cache):
    check(cuda_device, dtype, cache, (130, 16, 3), 4, 2, 64, 16, seed=7)
    check(cuda_device, dtype, cache, (130, 16, 3), 4, 2, 256, 16, window=2, seed=8)
    check(cuda_device, dtype, cache, (40, 5), 3, 1, 48 if cache != FP8 else 80, 8, seed=9)


@pytest.mark.parametrize("dtype,cache", TYPES[:4])
def test_softcap_and_decay(cuda_device, dtype, cache):
    check(cuda_device, dtype, cache, (33, 600), 4, 2, 128, 16, softcap=5.0, decay=0.75, seed=10)
    check(cuda_device, dtype, cache, (33, 600), 4, 2, 128, 16, window=4, decay=0.0, seed=11)


def test_large_and_tiny_queries_over_fp8_pages(cuda_device):
    """bf16 queries beyond f16's range, rows of one call many orders apart."""
    rng = np.random.default_rng(1)
    dev = cuda_device
    kc, vc, tables = ref.make_pool(rng, (40, 40), 2, 128, 16, FP8, dev)
    kc = (kc.float() * 2.0 ** -6).to(FP8)
    q = torch.from_numpy(rng.standard_normal((2, 1, 4, 128), np.float32))
    q[0] *= 3e5
    q[1] *= 1e-12
    q = q.to(torch.bfloat16).to(dev)
    ks, vs = torch.tensor([2.0 ** -10], device=dev), torch.tensor([1.0], device=dev)
    scores = torch.zeros(kc.shape[0], 2, 16, device=dev)
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor([40, 40], dtype=torch.int32, device=dev)
    out = eviction.paged_attention_scored(q, ks, vs, kc, vc, scores, bt, ctx, 40, 128 ** -0.5)
    want, want_s, added, reach = ref.scored(q, kc, vc, torch.zeros_like(scores), tables, (40, 40), 128 ** -0.5,
                                            k_scale=2.0 ** -10)
    rel = 128 * 2.0 ** -23 * reach + 2.0 ** -18 + 2.0 ** -11 * reach * 2.0 ** -10
    assert (np.abs(ref.f64(scores) - want_s) <= rel * added + 1e-7).all()
    assert (np.abs(ref.f64(out) - want) <= (2.0 ** -8 + 2.0 ** -11 + rel) * 5).all()


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_values_not_finite_in_masked_places(cuda_device, dtype, cache):
    """K and V of the window's last token are NaN / inf: the rows before it do not see them."""
    dev = cuda_device
    lens, w, bs = (50, 33, 16), 3, 16
    rng = np.random.default_rng(2)
    kc, vc, tables = ref.make_pool(rng, lens, 2, 128, bs, cache, dev)
    q = torch.from_numpy(rng.standard_normal((3, w, 4, 128), np.float32)).to(dtype).to(dev)
    bt, fp8 = torch.from_numpy(tables).to(dev), cache == FP8
    sc = [torch.ones(1, device=dev)] * 2 if fp8 else [None, None]
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    def run():
        s = torch.zeros(kc.shape[0], 2, bs, device=dev)
        return eviction.paged_attention_scored(q, *sc, kc, vc, s, bt, ctx, 50, 128 ** -0.5, score_rows=2), s
    clean, clean_s = run()
    for i, n in enumerate(lens):
        blk, off = int(tables[i, (n - 1) // bs]), (n - 1) % bs
        nan = float("nan")
        kf, vf = kc[blk].float(), vc[blk].float()
        kf[:, :, off] = nan if i < 2 else (448.0 if fp8 else float("inf"))
        vf[:, :, off] = nan if i else (nan if fp8 else float("inf"))
        kc[blk], vc[blk] = kf.to(cache), vf.to(cache)
    dirty, dirty_s = run()
    assert torch.equal(dirty[:, :w - 1], clean[:, :w - 1])
    assert torch.equal(dirty_s, clean_s)
    assert bool(dirty[:2, w - 1].float().isnan().all())           # what is seen is not hidden
    assert pa.device_error() == 0


def test_strided_queries_streams_and_graph(cuda_device):
    dev = cuda_device
    q, kc, vc, old, bt, ctx = check(dev, torch.bfloat16, torch.bfloat16, (100, 513, 64), 4, 2, 128, 16, seed=12)
    want_s = old.clone()
    want = eviction.paged_attention_scored(q[:, 0], None, None, kc, vc, want_s, bt, ctx, 600, 0.1)
    wide = torch.zeros(3, 4 * 128 + 2 * 2 * 128, dtype=torch.bfloat16, device=dev)
    wide[:, :512] = q.view(3, 512)
    s = old.clone()
    got = eviction.paged_attention_scored(wide[:, :512].view(3, 4, 128), None, None, kc, vc, s, bt, ctx, 600, 0.1)
    assert torch.equal(got, want) and torch.equal(s, want_s)
    stream = torch.cuda.Stream()
    need = eviction.paged_attention_scored_workspace_bytes(3, 1, 1, 4, 2, 128, 16, 600)
    eviction.reserve_paged_attention_scored_workspace(dev, need, stream)
    s = old.clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = eviction.paged_attention_scored(q[:, 0], None, None, kc, vc, s, bt, ctx, 600, 0.1)
    torch.cuda.current_stream().wait_stream(stream)
    s.copy_(old)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(s, want_s)
    del g


def test_agrees_with_paged_attention(cuda_device):
    """The outputs of the call without scores, within the same rounding of the weights."""
    dev = cuda_device
    q, kc, vc, old, bt, ctx = check(dev, torch.bfloat16, torch.bfloat16, (1500, 200, 831), 16, 8, 128, 16, seed=13)
    plain = pa.paged_attention(q[:, 0], None, None, kc, vc, bt, ctx, None, 1500, 128 ** -0.5)
    out = eviction.paged_attention_scored(q[:, 0], None, None, kc, vc, old, bt, ctx, 1500, 128 ** -0.5)
    assert float((plain.float() - out.float()).abs().max()) <= 2.0 ** -7 * 5


def test_ids_and_lengths_out_of_range(cuda_device):
    dev = cuda_device
    rng = np.random.default_rng(3)
    kc, vc, tables = ref.make_pool(rng, (64, 40), 2, 128, 16, torch.bfloat16, dev)
    kc[0], vc[0] = 0, 0
    q = torch.randn(2, 4, 128, device=dev).to(torch.bfloat16)
    scores = torch.zeros(kc.shape[0], 2, 16, device=dev)
    bt = torch.from_numpy(tables).to(dev)
    bt[0, 1] = kc.shape[0]
    ctx = torch.tensor([64, 40], dtype=torch.int32, device=dev)
    pa.device_error()
    out = eviction.paged_attention_scored(q, None, None, kc, vc, scores, bt, ctx, 64, 0.1)
    assert pa.device_error() == _lib.DERR_BLOCK_RANGE
    assert bool(out.float().isfinite().all())
    bt[0, 1] = int(tables[0, 1])
    ctx[1] = 1000                                                # past the table and the bound
    eviction.paged_attention_scored(q, None, None, kc, vc, scores, bt, ctx, 64, 0.1)
    assert pa.device_error() & _lib.DERR_CTX_RANGE


@pytest.mark.parametrize("dtype,cache", [(torch.float16, torch.float16), (torch.bfloat16, FP8), (torch.float16, FP8)])
def test_many_small_weights_beside_a_large_one(cuda_device, dtype, cache):
    """One token 2^20 times as heavy as each of 6000 others, whose values all point one way: weights
    far below f16's smallest value next to the largest still reach the output."""
    dev, n, d, bs = cuda_device, 6001, 128, 16
    rng = np.random.default_rng(20)
    kc, vc, tables = ref.make_pool(rng, (n,), 1, d, bs, cache, dev, fill=False)
    k = torch.zeros(kc.shape[0] * bs, 1, d)
    v = torch.full((kc.shape[0] * bs, 1, d), 400.0)
    sl = ref.slots_of(tables[0], n, bs)
    k[sl[0], 0, 0] = 1.0
    v[sl[0]] = 0.0
    x = kc.shape[-1]
    kc = k.view(-1, bs, 1, d // x, x).permute(0, 2, 3, 1, 4).contiguous().to(cache).to(dev)
    vc = v.view(-1, bs, 1, d).permute(0, 2, 3, 1).contiguous().to(cache).to(dev)
    q = torch.zeros(1, 1, 2, d, dtype=dtype, device=dev)
    q[..., 0] = 20 * float(np.log(2.0))
    scores = torch.zeros(kc.shape[0], 1, bs, device=dev)
    one = torch.ones(1, device=dev) if cache == FP8 else None
    out = eviction.paged_attention_scored(q, one, one, kc, vc, scores, torch.from_numpy(tables).to(dev),
                                          torch.tensor([n], dtype=torch.int32, device=dev), n, 1.0)
    want, _, _, reach = ref.scored(q, kc, vc, torch.zeros_like(scores), tables, (n,), 1.0)
    # P to 11 bits, or to f16's spacing of 2^-31 of the largest weight; V 400, the sum of weights near 1
    rel = 128 * 2.0 ** -23 * reach + 2.0 ** -18
    tol = (ref.ROUND[dtype] + 2.0 ** -11 + rel) * want + 6000 * 2.0 ** -32 * 400
    assert (want > 1).all() and (np.abs(ref.f64(out) - want) <= tol).all()


def test_loose_bound_leaves_the_order_of_the_stream(cuda_device):
    """Contexts of one split under a bound of many: the join has nothing to do, and what follows on
    the stream still sees the finished output and scores."""
    dev = cuda_device
    rng = np.random.default_rng(21)
    lens = [900] * 64
    kc, vc, tables = ref.make_pool(rng, lens, 8, 128, 16, torch.bfloat16, dev, extra_cols=200)
    q = torch.from_numpy(rng.standard_normal((64, 16, 128), np.float32)).to(torch.bfloat16).to(dev)
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = []
    for _ in range(20):
        s = torch.zeros(kc.shape[0], 8, 16, device=dev)
        out = eviction.paged_attention_scored(q, None, None, kc, vc, s, bt, ctx, 4000, 128 ** -0.5)
        got.append((out.clone(), s.clone()))  # ordered behind the call by the stream alone
    torch.cuda.synchronize()
    for out, s in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(s, got[0][1])
    # the 16 query heads' weights of every sequence sum to 16
    assert abs(float(got[-1][1].double().sum()) - 64 * 16) < 64 * 16 * 1e-4


def test_a_captured_graph_outlives_a_larger_call(cuda_device):
    """The workspace grows for the larger call; the graph still works in the one it was captured with."""
    dev = cuda_device
    q, kc, vc, old, bt, ctx = check(dev, torch.bfloat16, torch.bfloat16, (900, 513, 64), 4, 2, 128, 16, seed=31)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        need = eviction.paged_attention_scored_workspace_bytes(3, 1, 1, 4, 2, 128, 16, 900)
        small = eviction.reserve_paged_attention_scored_workspace(dev, need)
        s = old.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = eviction.paged_attention_scored(q[:, 0], None, None, kc, vc, s, bt, ctx, 900, 0.1)
        s.copy_(old)
        g.replay()
        want, want_s = out.clone(), s.clone()
        large = eviction.reserve_paged_attention_scored_workspace(dev, 2 * small.numel())
        assert large.data_ptr() != small.data_ptr() and large.numel() >= 2 * small.numel()
        at, size = small.data_ptr(), small.numel()
        del small
        taken = [torch.full((size,), 255, dtype=torch.uint8, device=dev) for _ in range(4)]
        assert all(t.data_ptr() + size <= at or at + size <= t.data_ptr() for t in taken)  # still held
        s.copy_(old)
        g.replay()
        assert torch.equal(out, want) and torch.equal(s, want_s)
        assert all(bool((t == 255).all()) for t in taken)
    torch.cuda.synchronize()
