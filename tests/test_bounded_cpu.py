"""Host side of the bounded speculative decoder: the operators are stubs that check what they are
given and answer with plain values, so that every window, slot and position can be looked at."""
import pytest
import torch

from vasr_paged_attn import _lib, bounded
from vasr_paged_attn.engine import DecoderConfig, RandomQwen3Decoder


class Stubs:
    """Stand-ins for the operators: they record the windows and check slots against the pages."""

    def __init__(self, accept=0):
        self.accept, self.windows, self.positions = accept, [], []

    def append(self, qkv, qw, kw, eps, cos, sin, positions, sections, kc, vc, slots, heads, score_cache=None, **kw_):
        bs = kc.shape[3]
        assert int(slots.min()) >= bs and int(slots.max()) < kc.shape[0] * bs  # never the null block
        assert len(set(slots.tolist())) == slots.numel()
        assert int(positions.min()) >= 0 and int(positions.max()) < cos.shape[0]
        self.positions.append(positions[0].tolist())
        return torch.zeros(qkv.shape[0], heads, 128)

    def attend(self, q, ks, vs, kc, vc, scores, tables, lens, longest, scale, score_rows=None):
        assert 1 <= q.shape[1] <= 64
        assert int(lens.max()) <= longest <= tables.shape[1] * kc.shape[3]
        self.windows.append(q.shape[1])
        return torch.zeros_like(q)

    def evict(self, kc, vc, scores, tables, lens, longest, budget, sink, recent):
        return None, lens.clamp(max=budget)

    def verify(self, logits, drafts, probs, uniform, race, temperature=0.0):
        b, k = drafts.shape
        n = min(self.accept, k)
        out = torch.full((b, k + 1), -1, dtype=torch.int32)
        out[:, :n], out[:, n] = drafts[:, :n], 7
        return out, torch.full((b,), n, dtype=torch.int32)


@pytest.fixture
def stubs(monkeypatch):
    s = Stubs()
    monkeypatch.setattr(bounded.fused, "qk_norm_mrope_append", s.append)
    monkeypatch.setattr(bounded.eviction, "paged_attention_scored", s.attend)
    monkeypatch.setattr(bounded.eviction, "evict_kv", s.evict)
    monkeypatch.setattr(bounded.speculative, "verify_draft_tokens", s.verify)
    return s


def decoder(k, capacity, budget, max_positions=512, seqs=2, **kw):
    cfg = DecoderConfig(hidden_size=32, num_layers=1, num_heads=2, num_kv_heads=1, intermediate_size=32,
                        vocab_size=50, max_positions=max_positions)
    model = RandomQwen3Decoder(cfg, "cpu", dtype=torch.float32, seed=1)
    return bounded.BoundedSpeculativeDecoder(model, seqs, k, capacity, budget, **kw)


def prompts(length, seqs=2):
    return [[(7 * i + j) % 50 for i in range(length)] for j in range(seqs)]


@pytest.mark.parametrize("capacity,budget,drafts,window", [(64, 60, 3, 16), (128, 120, 4, 16), (64, 62, 1, 64),
                                                           (64, 40, 3, 16), (64, 63, 0, 5), (256, 128, 4, 200)])
def test_a_prompt_stays_within_the_pages(stubs, capacity, budget, drafts, window):
    """Windows that are wider than the room an eviction leaves are cut to it."""
    dec = decoder(drafts, capacity, budget)
    dec.prefill(prompts(145), window)
    assert sum(stubs.windows) == 144 and max(stubs.windows) <= min(window, 64)
    assert int(dec.context_lens.max()) <= dec.capacity
    assert dec.next_positions.tolist() == [144, 144]
    assert sum(stubs.positions, []) == [p for at, w in zip(_starts(stubs.windows), stubs.windows)
                                        for _ in range(2) for p in range(at, at + w)]
    for _ in range(40):
        dec.step()
        assert int(dec.context_lens.max()) <= dec.capacity


def _starts(windows):
    return [sum(windows[:i]) for i in range(len(windows))]


def test_windows_that_fit_are_not_cut(stubs):
    dec = decoder(4, 64, 40)
    dec.prefill(prompts(100))
    assert stubs.windows == [16, 16, 16, 16, 16, 16, 3]
    assert dec.evictions == 2


def test_a_window_that_cannot_fit_is_refused_on_the_host(stubs):
    dec = decoder(3, 64, 60)
    dec.prefill(prompts(30))
    with pytest.raises(_lib.VasrPaError) as e:
        dec._make_room(5, 64)
    assert e.value.status == _lib.EINVAL_SHAPE
    with pytest.raises(_lib.VasrPaError):
        dec.prefill(prompts(30), 0)


def test_positions_stay_within_the_rotary_tables(stubs):
    """The cache is bounded, positions are not: a prompt that needs rows past the tables is refused,
    drafts are given up near their end, and a step past it is refused."""
    dec = decoder(4, 64, 40, max_positions=50)
    with pytest.raises(_lib.VasrPaError) as e:
        dec.prefill(prompts(51 + 1))
    assert e.value.status == _lib.EINVAL_SHAPE and not stubs.positions
    dec.prefill(prompts(44))
    for _ in range(7):  # first rows at 43 .. 49
        assert all(len(new) == 1 for new in dec.step())
    assert [len(w) // 2 for w in stubs.positions[-7:]] == [5, 5, 5, 4, 3, 2, 1]
    lens, tokens = dec.context_lens.tolist(), [list(t) for t in dec.tokens]
    with pytest.raises(_lib.VasrPaError) as e:
        dec.step()
    assert e.value.status == _lib.EINVAL_SHAPE
    assert dec.context_lens.tolist() == lens and dec.tokens == tokens


def test_the_longest_sequence_limits_the_drafts(stubs):
    dec = decoder(4, 64, 40, max_positions=50)
    dec.prefill(prompts(40))
    dec.tokens[1] += [1] * 6
    dec.next_positions[1] += 6
    dec.step()
    assert stubs.positions[-1] == list(range(39, 44)) + list(range(45, 50))
    stubs.accept = 4
    dec.step()
    assert stubs.positions[-1][-1] <= 49


def test_a_second_prompt_starts_afresh(stubs):
    dec = decoder(3, 64, 40)
    dec.prefill(prompts(100))
    for _ in range(10):
        dec.step()
    assert dec.evictions > 0
    del stubs.positions[:]
    dec.prefill(prompts(20))
    assert dec.context_lens.tolist() == [19, 19] and dec.next_positions.tolist() == [19, 19]
    assert dec.evictions == 0 and dec.tokens == prompts(20)
    assert [p[:16] for p in stubs.positions] == [list(range(16)), [16, 17, 18, 16, 17, 18]]
