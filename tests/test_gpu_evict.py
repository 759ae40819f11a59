"""Eviction: the selection against a sort on the host, the move against a permutation of bits."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import _lib, eviction, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def scores_for(rng, nb, hkv, bs, kind):
    s = np.exp(rng.standard_normal((nb, hkv, bs)) * 2).astype(np.float32)
    if kind == "ties":
        s = np.round(s).astype(np.float32)          # many equal values, zeros among them
    elif kind == "equal":
        s[:] = 0.25
    elif kind == "odd":                             # every special value
        pick = rng.integers(0, 8, s.shape)
        for i, v in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45]):
            s[pick == i] = v
        s[pick == 6] *= -1
    return s


def check(dev, dtype, lens, hkv, d, bs, budget, sink, recent, kind="plain", in_place=True, budgets=None, seed=0,
          bound=None):
    rng = np.random.default_rng(seed)
    kc, vc, tables = ref.make_pool(rng, lens, hkv, d, bs, dtype, dev, spare=0)
    out_tables = None
    if not in_place:
        n_old = kc.shape[0]
        # fresh pages behind the old ones
        cols = -(-min(budget, max(lens)) // bs) + 1
        out_tables = (n_old + rng.permutation(len(lens) * cols)).astype(np.int32).reshape(len(lens), cols)
        grow = len(lens) * cols
        kc = torch.cat([kc.float(), torch.full((grow, *kc.shape[1:]), float("nan"), device=dev)]).to(dtype)
        vc = torch.cat([vc.float(), torch.full((grow, *vc.shape[1:]), float("nan"), device=dev)]).to(dtype)
    nb = kc.shape[0]
    s = scores_for(rng, nb, hkv, bs, kind)
    scores = torch.from_numpy(s).to(dev)
    lim = [budget] * len(lens) if budgets is None else [min(budget, x) for x in budgets]
    want = ref.evict_indices(s, tables, lens, lim, sink, recent)
    spread = {5: (0, 3, 1, 2, 4), 4: (0, 3, 1, 2), 3: (0, 2, 1)}
    old = [ref.raw(x).transpose(spread[x.dim()]).reshape(nb * bs, hkv, -1) for x in (kc, vc, scores)]
    kept, new_lens = eviction.evict_kv(
        kc, vc, scores, torch.from_numpy(tables).to(dev), torch.tensor(list(lens), dtype=torch.int32, device=dev),
        max(max(lens), 1) if bound is None else bound, budget, sink, recent,
        budgets=None if budgets is None else torch.tensor(budgets, dtype=torch.int32, device=dev),
        out_block_tables=None if out_tables is None else torch.from_numpy(out_tables).to(dev))
    kept = kept.cpu().numpy()
    assert new_lens.tolist() == [min(n, b) for n, b in zip(lens, lim)]
    exp = [o.copy() for o in old]
    moved = np.zeros(nb * bs, bool)
    for i in range(len(lens)):
        to_table = tables[i] if out_tables is None else out_tables[i]
        for h in range(hkv):
            ids = np.array(want[i][h], np.int64)
            assert kept[i, h].tolist() == ids.tolist() + [-1] * (budget - len(ids)), (i, h)
            src = tables[i][ids // bs].astype(np.int64) * bs + ids % bs
            dst = ref.slots_of(to_table, len(ids), bs)
            for e, o in zip(exp, old):
                e[dst, h] = o[src, h]
    for x, e in zip((kc, vc, scores), exp):
        got = ref.raw(x).transpose(spread[x.dim()]).reshape(nb * bs, hkv, -1)
        assert np.array_equal(got, e)                # nothing else changed either
    assert pa.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, FP8])
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("in_place", [True, False])
def test_types_and_pages(cuda_device, dtype, bs, in_place):
    check(cuda_device, dtype, (200, 1, 75, 0, 64, 300), 2, 64, bs, 64, 3, 17, in_place=in_place, seed=bs)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
def test_equal_and_special_scores(cuda_device, kind, in_place):
    check(cuda_device, torch.bfloat16, (500, 129, 90), 3, 64, 16, 100, 4, 20, kind, in_place, seed=1)
    check(cuda_device, torch.bfloat16, (260,), 1, 128, 16, 7, 0, 0, kind, in_place, seed=2)


@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (50, 50, 0), (50, 0, 50), (50, 20, 30),
                                                (257, 4, 100), (399, 0, 1), (400, 4, 4), (1000, 4, 4)])
def test_budgets(cuda_device, budget, sink, recent):
    check(cuda_device, torch.bfloat16, (400, 33), 2, 128, 16, budget, sink, recent, seed=budget)


@pytest.mark.parametrize("in_place", [True, False])
def test_budget_per_sequence(cuda_device, in_place):
    check(cuda_device, torch.float16, (100, 100, 100, 20), 2, 64, 8, 60, 10, 20, budgets=[0, 25, 90, 15],
          in_place=in_place, seed=4)


@pytest.mark.parametrize("in_place", [True, False])
def test_long_sequences(cuda_device, in_place):
    check(cuda_device, torch.bfloat16, (9001, 4096), 2, 128, 16, 2500, 4, 512, in_place=in_place, seed=5, bound=9001)
    check(cuda_device, torch.bfloat16, (70001,), 1, 64, 32, 3001, 1, 64, "ties", in_place, seed=6)


@pytest.mark.parametrize("kind", ["plain", "ties", "equal"])
@pytest.mark.parametrize("seqs,hkv", [(4, 1), (4, 8), (4, 15), (4, 25), (5, 40)])
def test_long_and_short_together(cuda_device, seqs, hkv, kind):
    """Few and many (sequence, head)s share one long context's selection differently; the call's
    bound, not a sequence's own length, decides."""
    lens = (9001, 5, 0, 8193, 17)[:seqs]
    check(cuda_device, FP8, lens, hkv, 16, 16, 600, 3, 100, kind, True, seed=20, bound=9001)


def test_longer_than_the_keys_kept_at_hand(cuda_device):
    check(cuda_device, FP8, (50001,), 80, 16, 32, 900, 2, 64, "ties", True, seed=21)
    check(cuda_device, FP8, (400001,), 1, 16, 32, 900, 2, 64, "ties", False, seed=22)


def test_twice_in_place(cuda_device):
    """A second eviction works on what the first one left (the other sequences' pages untouched)."""
    dev, bs, hkv, d = cuda_device, 16, 2, 64
    rng = np.random.default_rng(7)
    kc, vc, tables = ref.make_pool(rng, (300,), hkv, d, bs, torch.float32, dev)
    scores = torch.from_numpy(scores_for(rng, kc.shape[0], hkv, bs, "plain")).to(dev)
    s0, k0 = scores.cpu().numpy().copy(), ref.token_major(kc, vc)[0]
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor([300], dtype=torch.int32, device=dev)
    first, ctx = eviction.evict_kv(kc, vc, scores, bt, ctx, 300, 128, 2, 30)
    second, ctx = eviction.evict_kv(kc, vc, scores, bt, ctx, 128, 40, 2, 10)
    assert ctx.tolist() == [40]
    ids = torch.gather(first, 2, second.long())
    sl = ref.slots_of(tables[0], 300, bs)
    for h in range(hkv):
        j = ids[0, h].cpu().numpy()
        want = ref.evict_indices(s0, tables, [300], [128], 2, 30)[0][h]
        assert set(j) <= set(want)
        got = ref.token_major(kc, vc)[0][sl[:40], h]
        assert np.array_equal(got, k0[sl[j], h])
    assert pa.device_error() == 0


def test_ids_out_of_range_are_flagged(cuda_device):
    dev = cuda_device
    rng = np.random.default_rng(8)
    kc, vc, tables = ref.make_pool(rng, (64,), 1, 64, 16, torch.bfloat16, dev)
    scores = torch.zeros(kc.shape[0], 1, 16, device=dev)
    bt = torch.from_numpy(tables).to(dev)
    bt[0, 2] = kc.shape[0] + 5
    ctx = torch.tensor([64], dtype=torch.int32, device=dev)
    pa.device_error()
    eviction.evict_kv(kc, vc, scores, bt, ctx, 64, 40, 0, 16)
    assert pa.device_error() == _lib.DERR_BLOCK_RANGE
    ctx[0] = 500
    bt[0, 2] = int(tables[0, 2])
    _, n = eviction.evict_kv(kc, vc, scores, bt, ctx, 64, 40, 0, 16)
    assert n.tolist() == [40] and pa.device_error() == _lib.DERR_CTX_RANGE


def test_stream_and_graph(cuda_device):
    dev, bs = cuda_device, 16
    rng = np.random.default_rng(9)
    kc, vc, tables = ref.make_pool(rng, (200, 90), 2, 64, bs, torch.bfloat16, dev)
    s = torch.from_numpy(scores_for(rng, kc.shape[0], 2, bs, "plain")).to(dev)
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor([200, 90], dtype=torch.int32, device=dev)
    sets = [[x.clone() for x in (kc, vc, s)] for _ in range(2)]
    kept, lens = eviction.evict_kv(*sets[0], bt, ctx, 200, 64, 2, 16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            kept2, lens2 = eviction.evict_kv(*sets[1], bt, ctx, 200, 64, 2, 16)
    torch.cuda.current_stream().wait_stream(stream)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, kept2) and torch.equal(lens, lens2)
    for a, b in zip(*sets):
        assert np.array_equal(ref.raw(a), ref.raw(b))
    del g
