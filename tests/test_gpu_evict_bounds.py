"""Eviction under bounds on the context length that are far above the contexts."""
import pytest
import torch

from test_gpu_evict import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hkv,seqs", [(1, 1), (4, 3), (40, 4)])
@pytest.mark.parametrize("bound", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 10 ** 6])
def test_a_bound_far_above_the_contexts(cuda_device, hkv, seqs, bound):
    check(cuda_device, torch.bfloat16, (700, 33, 0, 190)[:seqs], hkv, 16, 16, 100, 4, 20, seed=hkv, bound=bound)
