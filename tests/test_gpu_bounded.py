"""The speculative decoder over a bounded cache: the four operators in one step.

In f32 (no rounding of the weights, 24-bit sums) two forwards of one token differ by about 1e-5 of
a logit, so greedy tokens of a random decoder can be asked to be equal.
"""
import pytest
import torch

from vasr_paged_attn.bounded import BoundedSpeculativeDecoder, lookup_drafts
from vasr_paged_attn.engine import DecoderConfig, RandomQwen3Decoder


def test_lookup_drafts():
    assert lookup_drafts([1, 2, 3, 1, 2], 3) == [3, 1, 2]
    assert lookup_drafts([5, 1, 9, 2, 1], 2) == [9, 2]
    assert lookup_drafts([7], 3) == [7, 7, 7]
    assert lookup_drafts([4, 4], 2) == [4, 4]
    assert lookup_drafts([1, 2, 3], 0) == []


def small(dtype, dev):
    cfg = DecoderConfig(hidden_size=256, num_layers=3, num_heads=4, num_kv_heads=2, intermediate_size=320,
                        vocab_size=500, max_positions=4096)
    return RandomQwen3Decoder(cfg, dev, dtype=dtype, seed=5)


def decode(model, k, capacity, budget, steps_for, prompts, **kw):
    dec = BoundedSpeculativeDecoder(model, len(prompts), k, capacity, budget, **kw)
    dec.prefill(prompts)
    while min(len(t) for t in dec.tokens) < steps_for:
        for new in dec.step():
            assert 1 <= len(new) <= k + 1
    assert dec.device_error() == 0
    assert int(dec.context_lens.max()) <= dec.capacity
    # the last token is not in the cache yet
    assert dec.next_positions.tolist() == [len(t) - 1 for t in dec.tokens]
    return dec


PROMPTS = [[3, 17, 250, 9, 9, 11, 42] * 5 + [i] for i in (1, 2, 3)]


@pytest.mark.gpu
def test_drafts_do_not_change_greedy_tokens(cuda_device):
    model = small(torch.float32, cuda_device)
    plain = decode(model, 0, 512, 400, 120, PROMPTS)
    fast = decode(model, 4, 512, 400, 120, PROMPTS)
    for a, b in zip(plain.tokens, fast.tokens):
        assert a[:120] == b[:120]
    assert plain.evictions == fast.evictions == 0


@pytest.mark.gpu
def test_matches_a_forward_over_the_whole_sequence(cuda_device):
    """The tokens against dense attention in 64 bits over the same weights."""
    model = small(torch.float32, cuda_device)
    dec = decode(model, 3, 256, 200, 60, PROMPTS)
    cfg = model.cfg
    hq, hk, d = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
    ids = torch.tensor(dec.tokens[0][:60], device=cuda_device)
    n = len(ids)
    w = lambda t: t.double()  # noqa: E731
    norm = lambda x, g: x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * w(g)  # noqa: E731
    cos, sin = w(model.rope_cos[:n])[:, None], w(model.rope_sin[:n])[:, None]
    x = w(model.embed)[ids]
    mask = torch.full((n, n), float("-inf"), device=cuda_device, dtype=torch.float64).triu(1)
    for l in model.layers:
        qkv = (norm(x, l["in_norm"]) @ w(l["w_qkv"]).t()).view(n, hq + 2 * hk, d)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        turn = lambda y: torch.cat([y[..., :64] * cos - y[..., 64:] * sin, y[..., 64:] * cos + y[..., :64] * sin], -1)  # noqa: E731
        q, k = turn(norm(q, l["q_norm"])), turn(norm(k, l["k_norm"]))
        k, v = (y.repeat_interleave(hq // hk, 1) for y in (k, v))
        p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5 + mask, -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ w(l["w_o"]).t()
        g, u = (norm(x, l["post_norm"]) @ w(l["w_gate_up"]).t()).split(cfg.intermediate_size, 1)
        x = x + (torch.nn.functional.silu(g) * u) @ w(l["w_down"]).t()
    best = (norm(x, model.final_norm) @ w(model.embed).t()).argmax(-1).tolist()
    at = len(PROMPTS[0]) - 1
    assert best[at:n - 1] == dec.tokens[0][at + 1:n]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,temperature", [(torch.bfloat16, 0.0), (torch.float16, 0.8), (torch.float32, 0.8)])
def test_cache_stays_within_its_budget(cuda_device, dtype, temperature):
    model = small(dtype, cuda_device)
    dec = decode(model, 4, 64, 40, 200, PROMPTS, num_sink=2, num_recent=10, temperature=temperature)
    assert dec.evictions >= 4
    for s in dec.scores:  # accumulated weights are finite and not negative
        assert bool((s >= 0).all()) and bool(s.isfinite().all())
