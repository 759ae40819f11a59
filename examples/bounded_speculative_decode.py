"""Speculative decoding over a bounded cache with a random-init decoder (needs a B200).

    python examples/bounded_speculative_decode.py --seqs 8 --new 256 --budget 128

Prints how many drafts were accepted, how often the cache was shrunk, and the tokens per second.
"""
import argparse
import sys
import time
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "qwen3asr.rs_b200"))

import torch  # noqa: E402

from vasr_paged_attn.bounded import BoundedSpeculativeDecoder  # noqa: E402
from vasr_paged_attn.engine import DecoderConfig, RandomQwen3Decoder  # noqa: E402


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=96)
    ap.add_argument("--new", type=int, default=256)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--budget", type=int, default=128)
    ap.add_argument("--capacity", type=int, default=192)
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    cfg = DecoderConfig(num_layers=a.layers, vocab_size=32000)
    model = RandomQwen3Decoder(cfg, "cuda", seed=1)
    dec = BoundedSpeculativeDecoder(model, a.seqs, a.drafts, a.capacity, a.budget, temperature=a.temperature)
    gen = torch.Generator().manual_seed(2)
    dec.prefill(torch.randint(0, cfg.vocab_size, (a.seqs, a.prompt), generator=gen).tolist())
    torch.cuda.synchronize()
    began, steps, made = time.perf_counter(), 0, 0
    while min(len(t) for t in dec.tokens) < a.prompt + a.new:
        made += sum(len(t) for t in dec.step())
        steps += 1
    took = time.perf_counter() - began
    print(f"{made} tokens in {steps} steps: {made / (steps * a.seqs):.2f} a sequence and step "
          f"({a.drafts} drafts), {dec.evictions} evictions, longest context {int(dec.context_lens.max())} "
          f"of {dec.capacity}, {made / took:.0f} tokens/s, device error word {dec.device_error()}")


if __name__ == "__main__":
    main()
