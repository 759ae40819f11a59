"""The device error word: the bits of all units in one read, kept or cleared by it."""
import threading

import pytest
import torch

import operators_ref as ref
import numpy as np
from vasr_paged_attn import _lib, eviction, fused, mistralrs_paged_attn as pa

pytestmark = pytest.mark.gpu


def make_errors(dev):
    """A rotary position, a context length and a slot out of range: three units."""
    table = torch.zeros(4, 64, device=dev)
    pos = torch.full((3, 2), 9, dtype=torch.int64, device=dev)
    fused.mrope(torch.zeros(2, 2, 128, device=dev), table, table, pos, (24, 20, 20))
    kc, vc, tables = ref.make_pool(np.random.default_rng(1), (16,), 1, 128, 16, torch.bfloat16, dev)
    scores = torch.zeros(kc.shape[0], 1, 16, device=dev)
    eviction.evict_kv(kc, vc, scores, torch.from_numpy(tables).to(dev),
                      torch.tensor([99], dtype=torch.int32, device=dev), 16, 8, 0, 0)
    row = torch.zeros(1, 1, 128, dtype=torch.bfloat16, device=dev)
    pa.reshape_and_cache(row, row, None, None, kc, vc, torch.tensor([10 ** 6], device=dev))


ALL = _lib.DERR_POSITION_RANGE | _lib.DERR_CTX_RANGE | _lib.DERR_SLOT_RANGE


def test_units_are_read_together(cuda_device):
    pa.device_error()
    make_errors(cuda_device)
    assert pa.device_error(clear=False) == ALL
    assert pa.device_error(clear=False) == ALL
    assert pa.device_error() == ALL
    assert pa.device_error() == 0


def test_every_error_is_read_once(cuda_device):
    """Readers on streams of their own share what is reported; nothing is lost or seen twice."""
    pa.device_error()
    seen = []

    def read():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                seen.append(pa.device_error())

    make_errors(cuda_device)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=read) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(seen) == [0] * 199 + [ALL]
    assert pa.device_error() == 0
