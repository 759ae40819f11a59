"""Draft verification against its definition in 64 bits.

Tokens and counts have to be equal. A decision closer than 2^-18 of its two sides (the f32 sum
over the vocabulary and one exponential are off by less) could fall either way; the seeds below
have none, which each test asserts by deciding again with the numbers moved by that much.
"""
import numpy as np
import pytest
import torch

import operators_ref as ref
from vasr_paged_attn import speculative

pytestmark = pytest.mark.gpu
NUDGE = 2.0 ** -18


def inputs(rng, b, k, v, dtype, probs, scale=3.0):
    logits = torch.from_numpy(rng.standard_normal((b, k + 1, v)) * scale).to(dtype)
    soft = torch.softmax(logits[:, :k].double() + torch.from_numpy(rng.standard_normal((b, k, v)) * 0.7), -1)
    drafts = (soft / torch.from_numpy(rng.exponential(size=(b, k, v)))).argmax(-1).int()
    uniform = torch.from_numpy(rng.random((b, k))).float().clamp(max=1 - 2.0 ** -24)
    race = torch.from_numpy(rng.exponential(size=(b, v))).float()
    return logits, drafts, (soft.to(probs) if probs else None), uniform, race


def check(dev, logits, drafts, probs, uniform, race, temperature, lens=None, sure=True):
    b = logits.shape[0]
    temps = np.full(b, temperature) if not isinstance(temperature, torch.Tensor) else ref.f64(temperature)
    def want(u, p):
        return ref.verify(ref.f64(logits), drafts.cpu().numpy(), p, u, ref.f64(race), temps,
                          None if lens is None else lens.cpu().numpy())
    u, p = ref.f64(uniform), None if probs is None else ref.f64(probs)
    tokens, accepted = want(u, p)
    if sure:
        for f in (1 - NUDGE, 1 + NUDGE):
            assert np.array_equal(want(u * f, p)[1], accepted)
    up = lambda x: x.to(dev) if isinstance(x, torch.Tensor) else x  # noqa: E731
    for _ in range(2):  # the workspace is left as it has to be
        got, n = speculative.verify_draft_tokens(up(logits), up(drafts), up(probs), up(uniform), up(race),
                                                 temperature=up(temperature), draft_lens=up(lens))
        assert n.cpu().numpy().tolist() == accepted.tolist()
        assert got.cpu().numpy().tolist() == tokens.tolist()
    return tokens, accepted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,k,v", [(1, 4, 1000), (7, 3, 32003), (3, 1, 8), (2, 8, 151), (4, 0, 5001), (1, 2, 1),
                                   (5, 5, 16385)])
def test_tokens_are_the_definitions(cuda_device, dtype, probs, b, k, v):
    rng = np.random.default_rng(b * 100 + k * 7 + v)
    check(cuda_device, *inputs(rng, b, k, v, dtype, probs), 1.0)
    temps = torch.from_numpy(rng.uniform(0.3, 2.0, b)).float()
    temps[0] = 0.0
    check(cuda_device, *inputs(rng, b, k, v, dtype, probs), temps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ragged_drafts(cuda_device, dtype):
    rng = np.random.default_rng(1)
    lens = torch.tensor([0, 1, 2, 3, 4, 2], dtype=torch.int32)
    logits, drafts, probs, uniform, race = inputs(rng, 6, 4, 999, dtype, torch.float32)
    for i, n in enumerate(lens.tolist()):           # rows past a sequence's drafts are not read
        logits[i, n + 1:] = float("nan")
        probs[i, n:] = float("nan")
        drafts[i, n:] = -5
    uniform *= 0.01                                  # most drafts pass
    check(cuda_device, logits, drafts, probs, uniform, race, 0.8, lens)


@pytest.mark.parametrize("probs", [None, torch.float32])
def test_greedy(cuda_device, probs):
    rng = np.random.default_rng(2)
    logits, drafts, q, uniform, race = inputs(rng, 6, 3, 700, torch.bfloat16, probs)
    best = logits[:, :3].float().argmax(-1).int()
    drafts[0], drafts[1, :2], drafts[2, 1:] = best[0], best[1, :2], best[2, 1:]
    tokens, accepted = check(cuda_device, logits, drafts, q, uniform, race, 0.0)
    assert accepted[0] == 3 and accepted[1] >= 2
    dev = cuda_device
    got, n = speculative.verify_draft_tokens(logits.to(dev), drafts.to(dev), None, None, None, temperature=0.0)
    assert got.cpu().numpy().tolist() == tokens.tolist() and n.cpu().tolist() == accepted.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_masked_and_special_logits(cuda_device, dtype, temperature):
    """-inf masks (a whole row too), the type's lowest value, +inf, NaN, equal maxima."""
    rng = np.random.default_rng(3)
    v = 600
    logits, drafts, probs, uniform, race = inputs(rng, 8, 2, v, dtype, torch.float32)
    drafts[:] = 5
    uniform[:] = 0.0
    logits[0, 0] = float("-inf")                     # nothing left
    logits[1, 0] = torch.finfo(dtype).min            # everything masked by the lowest value
    logits[2, 0, ::2] = float("-inf")
    logits[2, 0, 1::2] = torch.finfo(dtype).min
    logits[3, 0, 77] = float("inf")
    logits[3, 1, 100:103] = float("inf")
    logits[4, 0, 9:400] = float("nan")
    logits[5] = 0.0                                  # equal everywhere
    logits[6, 0, 5] = float("-inf")                  # the draft itself is masked
    logits[7] = float("nan")
    check(cuda_device, logits, drafts, probs, uniform, race, temperature, sure=False)
    check(cuda_device, logits, drafts, None, uniform, race, temperature, sure=False)


def test_no_rest_falls_back_to_the_target(cuda_device):
    """The drafter's row covers the target's everywhere, and the draft fails all the same."""
    rng = np.random.default_rng(4)
    logits, drafts, probs, uniform, race = inputs(rng, 3, 1, 300, torch.float32, torch.float32)
    probs[:] = 1.0
    uniform[:] = 0.999
    _, accepted = check(cuda_device, logits, drafts, probs, uniform, race, 1.0)
    assert (accepted == 0).all()


def test_drafts_outside_the_vocabulary_and_odd_noise(cuda_device):
    rng = np.random.default_rng(5)
    logits, drafts, probs, uniform, race = inputs(rng, 4, 2, 300, torch.float32, torch.float32)
    drafts[0, 0], drafts[1, 0] = -1, 300
    uniform[:] = 0.0
    race[2, 17] = 0.0                                # wins wherever its probability is positive
    probs[2] = 0.0
    for p in (probs, None):
        tokens, accepted = check(cuda_device, logits, drafts, p, uniform, race, 1.0, sure=False)
        assert accepted[0] == 0 and accepted[1] == 0
        assert tokens[2, accepted[2]] == 17


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(cuda_device, dtype):
    rng = np.random.default_rng(6)
    b, k, v = 3, 3, 1237
    logits, drafts, probs, uniform, race = inputs(rng, b, k, v, dtype, torch.float32)
    tokens, accepted = check(cuda_device, logits, drafts, probs, uniform, race, 1.0)
    dev = cuda_device
    wide = torch.zeros(b, k + 1, v + 11, dtype=dtype, device=dev)[..., 3:3 + v]
    wide.copy_(logits)
    qwide = torch.zeros(b, k, v + 5, device=dev)[..., 1:1 + v]
    qwide.copy_(probs)
    rwide = torch.zeros(b, v + 3, device=dev)[:, 2:2 + v]
    rwide.copy_(race)
    got, n = speculative.verify_draft_tokens(wide, drafts.to(dev), qwide, uniform.to(dev), rwide)
    assert got.cpu().numpy().tolist() == tokens.tolist() and n.cpu().tolist() == accepted.tolist()


def test_distribution(cuda_device):
    """Accepted or replaced, the first token is distributed as the target alone says: chi-square
    over 7 outcomes of 40000 tries, 6 degrees of freedom, under 40 (p < 1e-6 otherwise)."""
    dev, b, v = cuda_device, 40000, 7
    g = torch.Generator(device=dev).manual_seed(11)
    logits = torch.tensor([0.5, -1.0, 2.0, 0.0, 1.0, -2.0, 0.3], device=dev)
    q = torch.softmax(torch.tensor([1.0, 1.0, 0.0, 0.5, -1.0, 0.0, 0.0], device=dev), -1)
    drafts = torch.multinomial(q, b, replacement=True, generator=g).int().view(b, 1)
    uniform = torch.rand(b, 1, device=dev, generator=g)
    race = torch.empty(b, v, device=dev).exponential_(generator=g)
    tokens, _ = speculative.verify_draft_tokens(logits.expand(b, 2, v).contiguous(), drafts,
                                                q.expand(b, 1, v).contiguous(), uniform, race)
    seen = torch.bincount(tokens[:, 0].long(), minlength=v).double().cpu()
    want = torch.softmax(logits.double(), -1).cpu() * b
    assert float(((seen - want) ** 2 / want).sum()) < 40


def test_stream_and_graph(cuda_device):
    rng = np.random.default_rng(7)
    dev = cuda_device
    args = [x.to(dev) for x in inputs(rng, 4, 3, 30001, torch.bfloat16, torch.float32)]
    want = speculative.verify_draft_tokens(*args)
    stream = torch.cuda.Stream()
    speculative.reserve_verify_draft_tokens_workspace(
        dev, speculative.verify_draft_tokens_workspace_bytes(4, 3, 30001), stream)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            got = speculative.verify_draft_tokens(*args)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del g


def test_workspace_of_another_stream_is_filled_on_it(cuda_device):
    """Reserving for a stream that is not current zeroes the workspace in that stream's order."""
    dev = cuda_device
    rng = np.random.default_rng(41)
    logits, drafts, _, uniform, race = inputs(rng, 3, 2, 50000, torch.float32, None)
    ins = [torch.as_tensor(x).to(dev) for x in (logits, drafts, uniform, race)]
    want = speculative.verify_draft_tokens(ins[0], ins[1], None, ins[2], ins[3], 1.0)
    stream = torch.cuda.Stream()
    need = speculative.verify_draft_tokens_workspace_bytes(3, 2, 50000)
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # the current stream is busy: a fill on it would come after the call
    speculative.reserve_verify_draft_tokens_workspace(dev, need, stream)
    with torch.cuda.stream(stream):
        got = speculative.verify_draft_tokens(ins[0], ins[1], None, ins[2], ins[3], 1.0)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        again = speculative.verify_draft_tokens(ins[0], ins[1], None, ins[2], ins[3], 1.0)
    stream.synchronize()
    assert torch.equal(again[0], want[0])
