"""Scored attention with block ids outside the pool: recorded, and no page's scores are touched for them."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import _lib, eviction, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 3])
def test_ids_outside_the_pool_score_nothing(cuda_device, d, window):
    dev = cuda_device
    rng = np.random.default_rng(d + window)
    lens = (64, 40, 33)
    kc, vc, tables = ref.make_pool(rng, lens, 2, d, 16, torch.bfloat16, dev)
    kc[0], vc[0] = 0, 0
    q = torch.from_numpy(rng.standard_normal((3, window, 4, d), np.float32)).to(torch.bfloat16).to(dev)
    scores = torch.from_numpy(rng.random((kc.shape[0], 2, 16), np.float32)).to(dev)
    old = scores.clone()
    bt = torch.from_numpy(tables).to(dev)
    bt[0, 1], bt[0, 2], bt[2, 2] = kc.shape[0], 0x7FFFFFFF, -1
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    pa.device_error()
    out = eviction.paged_attention_scored(q, None, None, kc, vc, scores, bt, ctx, 64, d ** -0.5, decay=0.5)
    assert pa.device_error() == _lib.DERR_BLOCK_RANGE
    assert bool(out.float().isfinite().all())
    assert torch.equal(scores[0], old[0])  # the block whose pages are read in their place
    # the pages that the table does name are scored once, the others keep their bits
    live = np.zeros(kc.shape[0], bool)
    for i, n in enumerate(lens):
        live[[int(x) for x in bt[i, :-(-n // 16)].tolist() if 0 <= x < kc.shape[0]]] = True
    assert np.array_equal(ref.raw(scores)[~live], ref.raw(old)[~live])
    # sequence 1 is untouched by the others' ids
    sound = old.clone()
    want = eviction.paged_attention_scored(q[1:2], None, None, kc, vc, sound, bt[1:2], ctx[1:2], 64, d ** -0.5, decay=0.5)
    assert float((want.float() - out[1:2].float()).abs().max()) <= 2.0 ** -7 * 4
    ids = bt[1, :3].long()
    assert torch.allclose(scores[ids], sound[ids], rtol=1e-5, atol=1e-6)
    assert pa.device_error() == 0
