"""The weights' precision in scored attention: rows of every tile shape keep more of a weight than
the query's type holds.

Keys are unit vectors and queries short fractions, so that every raw score is exact. A weight is
then off by a few roundoffs of f32 (the product with log2 e, one exponential, the sum: under 2^-18),
and reaches the output as two parts of at least 8 bits each, within 2^-16. The store rounds once:
|out error| <= u |out| + (2^-16 + 2^-18) sum p |v|.
"""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import eviction, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, FP8), (torch.float16, FP8)])
@pytest.mark.parametrize("window,hq", [(1, 2), (1, 4), (3, 2), (4, 2), (5, 2), (8, 2), (1, 16), (16, 2), (5, 8)])
@pytest.mark.parametrize("bs", [16, 32])
def test_weights_are_not_rounded_to_the_querys_type(cuda_device, dtype, cache, window, hq, bs):
    dev, d, lens = cuda_device, 128, (100, 41, 77)
    rng = np.random.default_rng(window * 100 + hq)
    kc, vc, tables = ref.make_pool(rng, lens, 1, d, bs, cache, dev)
    k = torch.zeros(kc.shape[0] * bs, 1, d)
    for i, n in enumerate(lens):
        k[ref.slots_of(tables[i], n, bs), 0, np.arange(n)] = 1.0
    x = kc.shape[-1]
    kc = k.view(-1, bs, 1, d // x, x).permute(0, 2, 3, 1, 4).contiguous().to(cache).to(dev)
    q = torch.from_numpy(rng.integers(-16, 17, (3, window, hq, d)) / 8.0).to(dtype).to(dev)
    one = torch.ones(1, device=dev) if cache == FP8 else None
    scores = torch.zeros(kc.shape[0], 1, bs, device=dev)
    out = eviction.paged_attention_scored(q, one, one, kc, vc, scores, torch.from_numpy(tables).to(dev),
                                          torch.tensor(lens, dtype=torch.int32, device=dev), 100, 1.0)
    want, _, _, _ = ref.scored(q, kc, vc, torch.zeros_like(scores), tables, lens, 1.0)
    # sum p |v|: the same attention over the values' magnitudes
    mass, _, _, _ = ref.scored(q, kc, vc.float().abs(), torch.zeros_like(scores), tables, lens, 1.0)
    tol = ref.ROUND[dtype] * np.abs(want) + ref.TINY[dtype] + (2.0 ** -16 + 2.0 ** -18) * mass
    off = np.abs(ref.f64(out) - want) / tol
    assert (off <= 1).all(), float(off.max())
    assert pa.device_error() == 0
