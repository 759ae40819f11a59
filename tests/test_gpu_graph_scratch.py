"""Scratch of the scored-attention and verification calls: graphs captured on one stream and
replayed on several at once do not share it, and none of it has to be cleared."""
import ctypes

import numpy as np
import pytest
import torch

import operators_ref as ref
from test_gpu_verify import inputs
from vasr_paged_attn import _lib, eviction, mistralrs_paged_attn as pa, speculative

pytestmark = pytest.mark.gpu


def scored_call(dev, seed):
    """A call of several splits, whose raw scores and partial results go through the scratch."""
    rng = np.random.default_rng(seed)
    lens = (3000, 2500, 1100, 64)
    kc, vc, tables = ref.make_pool(rng, lens, 4, 128, 16, torch.bfloat16, dev)
    q = torch.from_numpy(rng.standard_normal((4, 8, 128), np.float32)).to(torch.bfloat16).to(dev)
    bt = torch.from_numpy(tables).to(dev)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    scores = torch.zeros(kc.shape[0], 4, 16, device=dev)

    def call():
        return [eviction.paged_attention_scored(q, None, None, kc, vc, scores, bt, ctx, 3000, 128 ** -0.5, decay=0.0),
                scores]
    return call


def verify_call(dev, seed):
    rng = np.random.default_rng(seed)
    args = [x.to(dev) for x in inputs(rng, 6, 3, 40001, torch.bfloat16, torch.float32)]
    return lambda: list(speculative.verify_draft_tokens(*args, 0.9))


@pytest.mark.parametrize("make", [scored_call, verify_call])
def test_graphs_of_one_stream_replayed_on_two(cuda_device, make):
    dev = cuda_device
    calls = [make(dev, s) for s in (1, 2)]
    want = [[x.clone() for x in c()] for c in calls]
    stream = torch.cuda.Stream()  # nothing is reserved for it
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(c())
        graphs.append(g)
    bad = [torch.zeros((), dtype=torch.int64, device=dev) for _ in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(100):
        for g, s, out, w, b in zip(graphs, streams, outs, want, bad):
            with torch.cuda.stream(s):
                g.replay()
                for x, y in zip(out, w):
                    b += (x != y).sum()
    torch.cuda.synchronize()
    assert [int(b) for b in bad] == [0, 0]
    assert pa.device_error() == 0
    # and the calls outside the graphs go on
    assert all(torch.equal(x, y) for c, w in zip(calls, want) for x, y in zip(c(), w))


def test_the_verification_workspace_needs_no_clearing(cuda_device):
    dev = cuda_device
    rng = np.random.default_rng(3)
    b, k, v = 5, 3, 20001
    logits, drafts, probs, uniform, race = (x.to(dev) for x in inputs(rng, b, k, v, torch.float32, torch.float32))
    want = speculative.verify_draft_tokens(logits, drafts, probs, uniform, race, 0.9)
    need = speculative.verify_draft_tokens_workspace_bytes(b, k, v)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for fill in (255, 1, 0, 127):
        ws.fill_(fill)
        tokens = torch.full((b, k + 1), -7, dtype=torch.int32, device=dev)
        accepted = torch.full((b,), -7, dtype=torch.int32, device=dev)
        _lib.check(_lib.lib().vasr_pa_verify_draft_tokens(
            p(tokens), p(accepted), p(logits), (k + 1) * v, v, _lib.F32, p(drafts), None, p(probs), k * v, v, _lib.F32,
            p(uniform), p(race), v, None, 0.9, b, k, v, p(ws), need,
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "verify_draft_tokens")
        assert torch.equal(tokens, want[0]) and torch.equal(accepted, want[1])
