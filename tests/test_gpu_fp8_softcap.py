"""Softcapped decode over fp8 pages: the cap applies to scores that k_scale is part of.

Tolerance: the bf16 decode tolerance (2e-2) against the f64 oracle on the dequantised pages. With
the scale left out, scores of about one become scores of tens and run into the cap.
"""
import numpy as np
import pytest
import torch

import paged_ref as ref
from test_gpu_fp8 import D, HKV, HQ, _fp8_decode_case, _scales
from vasr_paged_attn import mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("bound", [0, 4096])  # a wide bound takes the wide instantiation
def test_the_cap_sees_the_scaled_scores(cuda_device, bs, bound):
    rng = np.random.default_rng(300 + bs)
    ctx = rng.integers(20, 400, size=64 if bound else 5).astype(np.int64)
    ctx[:3] = [1, 16, 399]
    ks, vs = 0.02, 0.015
    tables, kc, vc = _fp8_decode_case(rng, ctx, bs, ks, vs)
    q = torch.from_numpy(rng.standard_normal((len(ctx), HQ, D)).astype(np.float32)).to(torch.bfloat16)
    sk, sv = _scales(cuda_device, ks, vs)
    pa.device_error()
    out = pa.paged_attention(q.to(cuda_device), sk, sv,
                             torch.from_numpy(kc).to(cuda_device).view(torch.float8_e4m3fn),
                             torch.from_numpy(vc).to(cuda_device).view(torch.float8_e4m3fn),
                             torch.from_numpy(tables.astype(np.int32)).to(cuda_device),
                             torch.from_numpy(ctx.astype(np.int32)).to(cuda_device), None,
                             bound or int(ctx.max()), D ** -0.5, 2.0, None).float().cpu().numpy()
    kf = np.ascontiguousarray(ref.fp8_e4m3_decode(kc) * np.float32(ks))
    vf = np.ascontiguousarray(ref.fp8_e4m3_decode(vc) * np.float32(vs))
    exp = ref.paged_attention(np.ascontiguousarray(q.float().numpy()), kf, vf,
                              np.ascontiguousarray(tables.astype(np.uint32)), ctx.astype(np.uint32),
                              D ** -0.5, 2.0)
    assert np.abs(out - exp).max() <= 2e-2
    assert pa.device_error() == 0
