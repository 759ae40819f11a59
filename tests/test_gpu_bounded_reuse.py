"""A bounded decoder used for one prompt after another."""
import pytest
import torch

from test_gpu_bounded import PROMPTS, small
from vasr_paged_attn.bounded import BoundedSpeculativeDecoder

pytestmark = pytest.mark.gpu


def run(dec, prompts, steps):
    dec.prefill(prompts)
    return [dec.step() for _ in range(steps)]


def test_a_second_prompt_is_decoded_as_by_a_fresh_decoder(cuda_device):
    model = small(torch.float32, cuda_device)
    make = lambda: BoundedSpeculativeDecoder(model, 3, 4, 64, 40, num_sink=2, num_recent=10)  # noqa: E731
    other = [[5, 80, 2, 2] * 12 + [i, 7] for i in (4, 9, 6)]
    fresh = make()
    want = run(fresh, PROMPTS, 30)
    used = make()
    run(used, other, 20)
    assert run(used, PROMPTS, 30) == want
    assert used.evictions == fresh.evictions and used.context_lens.tolist() == fresh.context_lens.tolist()
    # the scores of the tokens in the cache too: the appends clear what the first prompt left
    for a, b in zip(used.scores, fresh.scores):
        for i, n in enumerate(fresh.context_lens.tolist()):
            j = torch.arange(n, device=cuda_device)
            blk = fresh.block_tables[i].long()[j // 16]
            assert torch.equal(a[blk, :, j % 16], b[blk, :, j % 16])
    assert used.device_error() == 0


def test_a_prompt_wider_than_the_room_beside_the_budget(cuda_device):
    model = small(torch.bfloat16, cuda_device)
    dec = BoundedSpeculativeDecoder(model, 3, 3, 64, 60, num_sink=2, num_recent=10)
    run(dec, [p * 5 for p in PROMPTS], 30)
    assert dec.evictions >= 20 and int(dec.context_lens.max()) <= dec.capacity
    assert dec.device_error() == 0
