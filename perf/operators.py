"""Benchmark cases of the operators around a bounded, speculatively decoded paged KV cache.

Four operators of one serving step, each in its plain torch form (``own = False``) and as the
framework's kernels (``own = True``):

* ``rotary``  per-head q/k RMSNorm, rotary embedding with several position axes (time, height,
  width) and the KV append; and the rotation alone, forwards and inverted (its gradient);
* ``scored``  attention of one new token, or of a short window of them, over the pages, which
  also adds every cached token's attention weight to a per-token score kept beside the pages;
* ``evict``   per kv head, keeps the tokens of the largest scores (and the first and last ones)
  and moves them to the front of a sequence's pages;
* ``verify``  accepts or rejects drafted tokens against the target's probabilities, with given
  random numbers, and draws the token that follows.

Cache layouts: key pages [blocks, kv heads, D / x, block, x] with x = 16 bytes of elements, value
pages [blocks, kv heads, D, block], scores [blocks, kv heads, block] in f32.
"""
import functools
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "fp8": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
SECTIONS = {128: (24, 20, 20), 64: (12, 10, 10), 256: (48, 40, 40)}  # time, height, width
MAX_POSITION = 65536
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def package():
    """The framework's modules (imported only where ``own`` is set)."""
    sys.path.insert(0, "qwen3asr.rs_b200")
    from vasr_paged_attn import eviction, fused, speculative

    return fused, eviction, speculative


# ------------------------------------------------------------------------------------ cases
def listed():
    heads = {"heads": 16, "kv_heads": 8, "dim": 128, "block": 16}
    return [
        # one decode step of 64 sequences: launch latency
        {"name": "rotary_step", "op": "rotary", "tokens": 64, "run": 1, "dtype": "bf16",
         "interleaved": True, **heads},
        # a prefill round: 32 prompts, 256 new tokens each
        {"name": "rotary_prompt", "op": "rotary", "tokens": 8192, "run": 256, "dtype": "bf16",
         "interleaved": True, **heads},
        # the gradient of the rotation of q and k rows in training, contiguous sections
        {"name": "rotary_inverse", "op": "rotate", "tokens": 4099, "heads": 24, "dim": 128,
         "dtype": "f16", "interleaved": False, "inverse": True},
        # a single sequence's decode step over a long context: split over its length
        {"name": "scored_single", "op": "scored", "seqs": 1, "lo": 16381, "hi": 16381, "rows": 1,
         "score_rows": 1, "dtype": "bf16", "cache": "bf16", **heads},
        # one decode step of a large batch, contexts from 64 to 4096 tokens
        {"name": "scored_batch", "op": "scored", "seqs": 512, "lo": 64, "hi": 4096, "rows": 1,
         "score_rows": 1, "dtype": "bf16", "cache": "bf16", **heads},
        # the same kind of step over one-byte pages
        {"name": "scored_fp8", "op": "scored", "seqs": 64, "lo": 200, "hi": 1500, "rows": 1,
         "score_rows": 1, "dtype": "bf16", "cache": "fp8", **heads},
        # a window of the last emitted token and four drafted ones, whose first row is scored
        {"name": "scored_window", "op": "scored", "seqs": 64, "lo": 200, "hi": 1500, "rows": 5,
         "score_rows": 1, "dtype": "f16", "cache": "f16", **heads},
        # a long sequence shrunk in place
        {"name": "evict_single", "op": "evict", "seqs": 1, "lo": 4099, "hi": 4099, "budget": 1024,
         "sink": 4, "recent": 256, "in_place": True, "dtype": "bf16", **heads},
        # a batch shrunk into fresh pages (the old ones stay, as a fork of a sequence needs)
        {"name": "evict_batch", "op": "evict", "seqs": 64, "lo": 700, "hi": 1500, "budget": 640,
         "sink": 4, "recent": 128, "in_place": False, "dtype": "bf16", **heads},
        # one sequence, four drafted tokens with the drafter's probabilities
        {"name": "verify_single", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936,
         "dtype": "bf16", "probs": "f32"},
        # a batch of such sequences
        {"name": "verify_batch", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 151936,
         "dtype": "bf16", "probs": "f32"},
        # drafts looked up in the prompt: no probabilities of a drafter
        {"name": "verify_lookup", "op": "verify", "seqs": 32, "drafts": 7, "vocab": 151936,
         "dtype": "f32", "probs": ""},
    ]


def spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    n = int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    n = min(max(n, lo), hi)
    return n + 1 if n == 3 * 1024 else n


def draw(rng):
    op = rng.choice(["rotary", "rotate", "scored", "scored", "evict", "verify"])
    kv = rng.choice([2, 4, 8])
    heads = {"heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": 128,
             "block": rng.choice([8, 16, 32])}
    dtype = rng.choice(["bf16", "f16", "bf16", "f32"])
    if op == "rotary":
        return {"op": op, "tokens": spread(rng, 1, 8192), "run": spread(rng, 1, 512),
                "dtype": dtype, "interleaved": rng.random() < 0.5, **heads}
    if op == "rotate":
        return {"op": op, "tokens": spread(rng, 1, 8192), "heads": rng.randint(1, 32),
                "dim": rng.choice([64, 128, 256]), "dtype": dtype,
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.5}
    if op == "scored":
        hi = spread(rng, 1, 20000)
        seqs = spread(rng, 1, max(1, min(512, 300000 // hi)))
        rows = rng.choice([1, 1, 2, 4, 5, 8])
        cache = dtype
        if dtype != "f32" and heads["block"] != 8 and rng.random() < 0.3:
            cache = "fp8"
        return {"op": op, "seqs": seqs, "lo": max(1, hi // rng.randint(1, 16)), "hi": hi,
                "rows": rows, "score_rows": rng.randint(1, rows), "dtype": dtype, "cache": cache,
                **heads}
    if op == "evict":
        hi = spread(rng, 16, 20000)
        budget = max(8, int(hi * rng.uniform(0.2, 0.9)))
        return {"op": op, "seqs": spread(rng, 1, max(1, min(256, 100000 // hi))),
                "lo": max(1, hi // rng.randint(1, 4)), "hi": hi, "budget": budget,
                "sink": rng.randint(0, 4), "recent": rng.randint(0, budget // 2),
                "in_place": rng.random() < 0.5, "dtype": dtype, **heads}
    return {"op": op, "seqs": spread(rng, 1, 64), "drafts": rng.randint(1, 8),
            "vocab": spread(rng, 1000, 151936), "dtype": dtype,
            "probs": rng.choice(["", "f32", "f32", "bf16"])}


def lengths(case):
    """The sequences' context lengths, spread over their logarithm (the last one the longest)."""
    rng = random.Random(17)
    lo, hi = case["lo"], case["hi"]
    return [spread(rng, lo, hi) for _ in range(case["seqs"] - 1)] + [hi]


def work(case):
    if case["op"] in ("rotary", "rotate"):
        t, d, es = case["tokens"], case["dim"], SIZES[case["dtype"]]
        rows = case["heads"] + 2 * case.get("kv_heads", 0)
        per_token = 2 * rows * d * es + 3 * 8 + 2 * (d // 2) * 4
        if case["op"] == "rotary":
            per_token += 8 + 4 * case["kv_heads"]  # slots, cleared scores
        return {"bytes": t * per_token, "flops": t * rows * d * 8}
    if case["op"] == "verify":
        b, k, v = case["seqs"], case["drafts"], case["vocab"]
        per_row = (k + 1) * SIZES[case["dtype"]] + 4  # every target row, the race's noise
        if case["probs"]:
            per_row += SIZES[case["probs"]]           # the drafter's row where a draft fails
        return {"bytes": b * v * per_row + b * (8 * k + 4 * (k + 2)), "flops": b * v * (4 * k + 8)}
    n = lengths(case)
    hk, d = case["kv_heads"], case["dim"]
    pages = sum(-(-x // case["block"]) for x in n)
    if case["op"] == "scored":
        rows = case["seqs"] * case["rows"] * case["heads"]
        return {"bytes": sum(n) * hk * (2 * d * SIZES[case["cache"]] + 8) + 4 * pages
                + 2 * rows * d * SIZES[case["dtype"]],
                "flops": 4 * sum(n) * case["rows"] * case["heads"] * d}
    moved = sum(case["budget"] for x in n if x > case["budget"])
    if not case["in_place"]:
        moved = sum(min(x, case["budget"]) for x in n)
    return {"bytes": sum(n) * hk * 4 + 2 * moved * hk * (2 * d * SIZES[case["dtype"]] + 4)
            + 4 * case["seqs"] * hk * case["budget"] + 4 * pages,
            "flops": sum(n) * hk}


# ----------------------------------------------------------------------------------- inputs
def axis_of_frequency(sections, interleaved):
    """Which position axis turns each frequency: sections one after another, or interleaved
    (axis a > 0 turns frequencies a, a + n, a + 2 n, ..., as many as its section says)."""
    n = len(sections)
    if not interleaved:
        return [a for a, s in enumerate(sections) for _ in range(s)]
    return [i % n if i // n < sections[i % n] else 0 for i in range(sum(sections))]


def tables(dim, device):
    inv = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    ang = torch.outer(torch.arange(MAX_POSITION, dtype=torch.float64, device=device), inv)
    return ang.cos().float(), ang.sin().float()


def grid_positions(tokens, device, gen):
    """Positions of text with pictures and video in it: runs of equal axes, and 12 x 20 grids."""
    i = torch.arange(tokens, device=device)
    at = i % 1000
    picture = at >= 400
    base = i // 1000 * 1000 + 400
    j = (at - 400).clamp(min=0)
    start = int(torch.randint(0, 4096, (1,), device=device, generator=gen))
    t = torch.where(picture, base + j // 240, i)
    h = torch.where(picture, base + j % 240 // 20, i)
    w = torch.where(picture, base + j % 20, i)
    return (torch.stack([t, h, w]) + start).contiguous()


def normal(shape, dtype, device, gen, scale=1.0):
    x = torch.empty(shape, dtype=dtype if dtype != DTYPES["fp8"] else torch.bfloat16, device=device)
    return x.normal_(0.0, scale, generator=gen).to(dtype)


def page_pool(case, blocks, cache, device, gen, scale=1.0):
    x = 16 // SIZES[cache]
    k = normal((blocks, case["kv_heads"], case["dim"] // x, case["block"], x), DTYPES[cache], device, gen, scale)
    v = normal((blocks, case["kv_heads"], case["dim"], case["block"]), DTYPES[cache], device, gen, scale)
    return k, v


def block_tables(case, n, device, gen, first=1):
    """Each sequence's pages, scattered over a pool (block 0 stays unused), and the pool's end."""
    need = torch.tensor([-(-x // case["block"]) for x in n], device=device)
    cols = int(need.max())
    total = int(need.sum())
    ids = torch.randperm(total, device=device, generator=gen).to(torch.int32) + first
    col = torch.arange(cols, device=device)
    at = (need.cumsum(0) - need)[:, None] + col
    used = col < need[:, None]
    return torch.where(used, ids[at.clamp(max=total - 1)], 0).contiguous(), first + total


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    st = {"case": case}
    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("rotary", "rotate"):
        t, d = case["tokens"], case["dim"]
        st["sections"] = SECTIONS[d]
        st["cos"], st["sin"] = tables(d, dev)
        st["positions"] = grid_positions(t, dev, gen)
        st["axes"] = torch.tensor(axis_of_frequency(SECTIONS[d], case["interleaved"]), device=dev)
        if case["op"] == "rotate":
            st["x"] = normal((t, case["heads"], d), dtype, dev, gen)
            return st
        bs = case["block"]
        st["qkv"] = normal((t, (case["heads"] + 2 * case["kv_heads"]) * d), dtype, dev, gen, 2.0)
        st["q_norm"] = 1 + normal((d,), dtype, dev, gen, 0.1)
        st["k_norm"] = 1 + normal((d,), dtype, dev, gen, 0.1)
        # tokens go to consecutive slots for `run` tokens at a time, each run on its own pages
        run = min(case["run"], t)
        per_run = -(-run // bs)
        runs = -(-t // run)
        ids = torch.randperm(runs * per_run, device=dev, generator=gen) + 1
        i = torch.arange(t, device=dev)
        at = i % run
        st["slots"] = ids[i // run * per_run + at // bs] * bs + at % bs
        blocks = runs * per_run + 1
        st["k"], st["v"] = (torch.zeros_like(c) for c in page_pool(case, blocks, case["dtype"], dev, gen))
        st["scores"] = torch.ones(blocks, case["kv_heads"], bs, device=dev)
        return st
    if case["op"] == "verify":
        b, k, v = case["seqs"], case["drafts"], case["vocab"]
        logits = normal((b, k + 1, v), torch.float32, dev, gen, 3.0)
        st["logits"] = logits.to(dtype)
        # the drafter is a noisier copy of the target, its drafts drawn from what it says
        q = (logits[:, :k] + normal((b, k, v), torch.float32, dev, gen, 0.7)).softmax(-1)
        del logits
        race = torch.empty((b, k, v), device=dev).exponential_(generator=gen)
        st["drafts"] = (q / race).argmax(-1).to(torch.int32)
        st["probs"] = q.to(DTYPES[case["probs"]]) if case["probs"] else None
        st["uniform"] = torch.rand((b, k), device=dev, generator=gen)
        st["race"] = torch.empty((b, v), device=dev).exponential_(generator=gen)
        st["temperature"] = 0.6 + 0.8 * torch.rand((b,), device=dev, generator=gen)
        return st
    n = lengths(case)
    st["tables"], blocks = block_tables(case, n, dev, gen)
    st["lens"] = torch.tensor(n, dtype=torch.int32, device=dev)
    st["longest"] = max(n)
    if case["op"] == "scored":
        st["k"], st["v"] = page_pool(case, blocks, case["cache"], dev, gen)
        st["q"] = normal((case["seqs"], case["rows"], case["heads"], case["dim"]), dtype, dev, gen, 1.5)
        fp8 = case["cache"] == "fp8"
        st["k_scale"] = torch.tensor([0.8], device=dev) if fp8 else None
        st["v_scale"] = torch.tensor([1.3], device=dev) if fp8 else None
        # weights of a few earlier steps
        st["scores"] = 0.01 * torch.rand((blocks, case["kv_heads"], case["block"]), device=dev, generator=gen)
        return st
    st["out_tables"] = None
    if not case["in_place"]:
        kept = [min(x, case["budget"]) for x in n]
        st["out_tables"], blocks = block_tables(case, kept, dev, gen, blocks)
    st["k"], st["v"] = page_pool(case, blocks, case["dtype"], dev, gen)
    # accumulated weights: a few heavy tokens, many light ones, some of no weight at all
    s = normal((blocks, case["kv_heads"], case["block"]), torch.float32, dev, gen, 2.0).exp()
    st["scores"] = torch.where(torch.rand(s.shape, device=dev, generator=gen) < 0.1, 0.0, s)
    return st


# ------------------------------------------------------------------------------ plain forms
def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def angles(st, dtype):
    rows = st["positions"][st["axes"]].t()
    return (st["cos"].gather(0, rows)[:, None].to(dtype), st["sin"].gather(0, rows)[:, None].to(dtype))


def plain_rotary(st):
    case = st["case"]
    hq, hk, d, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
    t = case["tokens"]
    x = st["qkv"].float().view(t, hq + 2 * hk, d)
    cos, sin = angles(st, torch.float32)
    qk = x[:, :hq + hk]
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    weight = torch.cat([st["q_norm"].float().expand(hq, d), st["k_norm"].float().expand(hk, d)])
    qk = rotate(qk * weight, cos, sin).to(st["qkv"].dtype)
    blk, off = st["slots"] // bs, st["slots"] % bs
    st["k"][blk, :, :, off] = qk[:, hq:].reshape(t, hk, *st["k"].shape[2::2])
    st["v"][blk, :, :, off] = st["qkv"].view(t, hq + 2 * hk, d)[:, hq + hk:]
    st["scores"][blk, :, off] = 0.0
    return qk[:, :hq].contiguous()


def plain_rotate(st):
    cos, sin = angles(st, torch.float32)
    return rotate(st["x"].float(), cos, -sin if st["case"]["inverse"] else sin).to(st["x"].dtype)


def rows_of(cache, blocks):
    """The given blocks of a cache (one-byte elements are indexed as bytes)."""
    if cache.element_size() == 1:
        return cache.view(torch.uint8)[blocks].view(cache.dtype)
    return cache[blocks]


def tokens_of(st, name):
    """Pages of every sequence as [seqs, kv heads, tokens, D] in f32."""
    x = rows_of(st[name], st["tables"].long()).float()
    if name == "k":  # [B, cols, H, D/x, bs, x]
        x = x.permute(0, 2, 1, 4, 3, 5).flatten(4)
    else:            # [B, cols, H, D, bs]
        x = x.permute(0, 2, 1, 4, 3)
    return x.flatten(2, 3)


def plain_scored(st):
    case = st["case"]
    b, rows, hq, d = st["q"].shape
    hk = case["kv_heads"]
    g = hq // hk
    tables = st["tables"].long()
    q = st["q"].float().view(b, rows, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, rows * g, d)
    k = tokens_of(st, "k")
    s = (q * d ** -0.5) @ k.transpose(2, 3)
    del k
    if st["k_scale"] is not None:
        s = s * st["k_scale"]
    j = torch.arange(s.shape[-1], device=s.device)
    last = st["lens"][:, None] - rows + torch.arange(rows, device=s.device)   # [B, rows]
    seen = (j <= last[:, :, None]).repeat_interleave(g, 1)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    del s
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = p @ tokens_of(st, "v")
    if st["v_scale"] is not None:
        out = out * st["v_scale"]
    out = out.view(b, hk, rows, g, d).permute(0, 2, 1, 3, 4).reshape(b, rows, hq, d)
    add = p[:, :, :case["score_rows"] * g].sum(2)
    add = add.view(b, hk, -1, case["block"]).transpose(1, 2)          # [B, cols, H, bs]
    live = (j < st["lens"][:, None]).view(b, -1, 1, case["block"])
    old = st["scores"][tables]
    st["scores"][tables] = torch.where(live, old + add, old)
    return {"out": out.to(st["q"].dtype), "scores": st["scores"]}


def kept_tokens(st):
    """[B, H, budget] indices of the tokens that stay, ascending, -1 past a sequence's own."""
    case, lens = st["case"], st["lens"].long()
    s = st["scores"][st["tables"].long()].transpose(1, 2).flatten(2)  # [B, H, tokens]
    j = torch.arange(s.shape[-1], device=s.device)
    n = lens[:, None]
    always = (j < case["sink"]) | (j >= n - case["recent"])
    s = torch.where(always[:, None], math.inf, s)
    s = torch.where((j < n)[:, None], s, -math.inf)
    order = s.sort(dim=-1, descending=True, stable=True).indices[..., :case["budget"]]
    kept = n.clamp(max=case["budget"])
    at = torch.arange(case["budget"], device=s.device)
    if order.shape[-1] < case["budget"]:
        order = torch.nn.functional.pad(order, (0, case["budget"] - order.shape[-1]))
    live = (at < kept)[:, None]
    ids = torch.where(live, order, s.shape[-1]).sort(-1).values
    return torch.where(live, ids, -1).to(torch.int32), kept[:, 0].to(torch.int32)


def places(tables, index, block):
    """Block and offset of each token index [B, H, N]."""
    cols = (index // block).clamp(max=tables.shape[1] - 1)
    blk = tables.long()[:, None].expand(-1, index.shape[1], -1).gather(2, cols)
    return blk, index % block


def plain_evict(st):
    case = st["case"]
    kept, lens = kept_tokens(st)
    live = kept >= 0
    head = torch.arange(case["kv_heads"], device=kept.device)[:, None]
    to = torch.arange(case["budget"], device=kept.device).expand(kept.shape)
    out_tables = st["tables"] if st["out_tables"] is None else st["out_tables"]
    sb, so = places(st["tables"], kept.clamp(min=0).long(), case["block"])
    db, do = places(out_tables, to, case["block"])
    # what is not a kept token's place gets its own value back (at block 0, where a table ends)
    db, do = torch.where(live, db, 0), torch.where(live, do, 0)
    sb, so = torch.where(live, sb, 0), torch.where(live, so, 0)
    st["k"][db, head, :, do] = st["k"][sb, head, :, so]
    st["v"][db, head, :, do] = st["v"][sb, head, :, so]
    st["scores"][db, head, do] = st["scores"][sb, head, so]
    return {"kept": kept, "lens": lens, "k": st["k"], "v": st["v"], "scores": st["scores"]}


def plain_verify(st, dtype=torch.float32):
    drafts = st["drafts"].long()
    b, k = drafts.shape
    x = st["logits"].to(dtype) / st["temperature"].to(dtype)[:, None, None]
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    px = p[:, :k].gather(2, drafts[..., None])[..., 0]
    row = torch.arange(b, device=p.device)
    if st["probs"] is not None:
        qx = st["probs"].gather(2, drafts[..., None])[..., 0].to(dtype)
    else:
        qx = torch.ones_like(px)
    ok = st["uniform"].to(dtype) * qx < px
    n = ok.long().cumprod(1).sum(1)
    pn = p[row, n]
    at = n.clamp(max=k - 1)
    if st["probs"] is not None:
        rest = (pn - st["probs"][row, at].to(dtype)).clamp(min=0)
    else:
        rest = pn.scatter(1, drafts[row, at][:, None], 0.0)
    rest = torch.where((n < k)[:, None], rest, pn)
    rest = torch.where((rest > 0).any(1, keepdim=True), rest, pn)
    nxt = (rest / st["race"].to(dtype)).argmax(1)
    at = torch.arange(k + 1, device=p.device)
    tokens = torch.nn.functional.pad(drafts, (0, 1))
    tokens = torch.where(at < n[:, None], tokens, torch.where(at == n[:, None], nxt[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "accepted": n.to(torch.int32)}


def run(st):
    case, op = st["case"], st["case"]["op"]
    if op == "rotary":
        if own:
            q = package()[0].qk_norm_mrope_append(
                st["qkv"], st["q_norm"], st["k_norm"], EPS, st["cos"], st["sin"], st["positions"],
                st["sections"], st["k"], st["v"], st["slots"], case["heads"],
                interleaved=case["interleaved"], score_cache=st["scores"])
        else:
            q = plain_rotary(st)
        return {"q": q, "k": st["k"], "v": st["v"], "scores": st["scores"]}
    if op == "rotate":
        if own:
            return package()[0].mrope(st["x"], st["cos"], st["sin"], st["positions"],
                                      st["sections"], interleaved=case["interleaved"],
                                      inverse=case["inverse"])
        return plain_rotate(st)
    if op == "scored":
        if own:
            out = package()[1].paged_attention_scored(
                st["q"], st["k_scale"], st["v_scale"], st["k"], st["v"], st["scores"],
                st["tables"], st["lens"], st["longest"], case["dim"] ** -0.5,
                score_rows=case["score_rows"])
            return {"out": out, "scores": st["scores"]}
        return plain_scored(st)
    if op == "evict":
        if own:
            kept, lens = package()[1].evict_kv(
                st["k"], st["v"], st["scores"], st["tables"], st["lens"], st["longest"],
                case["budget"], case["sink"], case["recent"], out_block_tables=st["out_tables"])
            return {"kept": kept, "lens": lens, "k": st["k"], "v": st["v"], "scores": st["scores"]}
        return plain_evict(st)
    if own:
        tokens, accepted = package()[2].verify_draft_tokens(
            st["logits"], st["drafts"], st["probs"], st["uniform"], st["race"],
            temperature=st["temperature"])
        return {"tokens": tokens, "accepted": accepted}
    return plain_verify(st)


# ---------------------------------------------------------------------------- in 64 bits
def exact_angles(st):
    """cos and sin [tokens, 1, D / 2] read off the tables, one frequency after another."""
    cos, sin = [], []
    for i, a in enumerate(st["axes"].tolist()):
        at = st["positions"][a]
        cos.append(st["cos"][:, i].double()[at])
        sin.append(st["sin"][:, i].double()[at])
    return torch.stack(cos, 1)[:, None], torch.stack(sin, 1)[:, None]


def exact_turn(x, cos, sin):
    """Each (i, i + D / 2) pair as a complex number times cos + i sin."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(*torch.broadcast_tensors(cos, sin))
    return torch.cat([z.real, z.imag], -1)


def exact_rotary(st):
    case = st["case"]
    hq, hk, d, bs, t = case["heads"], case["kv_heads"], case["dim"], case["block"], case["tokens"]
    rows = st["qkv"].double().view(t, -1, d)
    cos, sin = exact_angles(st)

    def head(x, w):
        return exact_turn(x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w.double(), cos, sin)

    # [blocks, H, token of the block, D], then the page layouts
    k = torch.zeros(st["k"].shape[0] * bs, hk, d, dtype=torch.float64, device=rows.device)
    v = torch.zeros_like(k)
    scores = torch.ones(st["k"].shape[0] * bs, hk, dtype=torch.float64, device=rows.device)
    k[st["slots"]] = head(rows[:, hq:hq + hk], st["k_norm"])
    v[st["slots"]] = rows[:, hq + hk:]
    scores[st["slots"]] = 0
    x = st["k"].shape[-1]
    k = k.view(-1, bs, hk, d // x, x).permute(0, 2, 3, 1, 4).contiguous()
    v = v.view(-1, bs, hk, d).permute(0, 2, 3, 1).contiguous()
    return {"q": head(rows[:, :hq], st["q_norm"]), "k": k, "v": v,
            "scores": scores.view(-1, bs, hk).transpose(1, 2).contiguous()}


def exact_scored(st):
    case = st["case"]
    hk, g, d, bs = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["block"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    scores = st["scores"].double()
    mul = float(st["k_scale"]) if st["k_scale"] is not None else 1.0
    out_mul = float(st["v_scale"]) if st["v_scale"] is not None else 1.0
    for b, n in enumerate(lengths(case)):
        blk = st["tables"][b, :-(-n // bs)].long()
        k = rows_of(st["k"], blk).double().transpose(3, 4).reshape(len(blk), hk, d, bs)
        k = k.permute(1, 2, 0, 3).reshape(hk, d, -1)[..., :n]          # [H, D, n]
        v = rows_of(st["v"], blk).double().permute(1, 2, 0, 3).reshape(hk, d, -1)[..., :n]
        add = torch.zeros(hk, n, dtype=torch.float64, device=k.device)
        for i in range(case["rows"]):
            m = n - case["rows"] + i + 1
            if m <= 0:
                continue
            q = st["q"][b, i].double().view(hk, g, d)
            w = torch.softmax(q @ k[..., :m] * (mul * d ** -0.5), -1)
            out[b, i] = (torch.einsum("hgn,hdn->hgd", w, v[..., :m]) * out_mul).reshape(-1, d)
            if i < case["score_rows"]:
                add[:, :m] += w.sum(1)
        j = torch.arange(n, device=k.device)
        scores[blk[j // bs], :, j % bs] += add.t()
    return {"out": out, "scores": scores}


def exact_evict(st):
    """Sequence by sequence, kv head by kv head, on the host."""
    case, bs = st["case"], st["case"]["block"]
    table = st["tables"].cpu()
    to = table if st["out_tables"] is None else st["out_tables"].cpu()
    old = st["scores"].cpu()
    kept = torch.full((case["seqs"], case["kv_heads"], case["budget"]), -1, dtype=torch.int32)
    sb, so, db, do, hh = [], [], [], [], []
    for b, n in enumerate(lengths(case)):
        for h in range(case["kv_heads"]):
            s = old[table[b].long(), h].flatten()[:n].tolist()
            mid = range(min(case["sink"], n), max(case["sink"], n - case["recent"]))
            mid = [j for j in mid if j < n]
            always = sorted(set(range(n)) - set(mid))
            best = sorted(mid, key=lambda j: (-s[j], j))
            ids = sorted(always + best[:max(0, case["budget"] - len(always))])[:case["budget"]]
            kept[b, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            i, j = torch.tensor(ids), torch.arange(len(ids))
            sb.append(table[b, i // bs].long())
            so.append(i % bs)
            db.append(to[b, j // bs].long())
            do.append(j % bs)
            hh.append(torch.full((len(ids),), h))
    dev = st["k"].device
    sb, so, db, do, hh = (torch.cat(x).to(dev) for x in (sb, so, db, do, hh))
    k, v, scores = st["k"].double(), st["v"].double(), st["scores"].double()
    k[db, hh, :, do] = st["k"].double()[sb, hh, :, so]
    v[db, hh, :, do] = st["v"].double()[sb, hh, :, so]
    scores[db, hh, do] = st["scores"].double()[sb, hh, so]
    lens = torch.tensor([min(n, case["budget"]) for n in lengths(case)], dtype=torch.int32)
    return {"kept": kept, "lens": lens, "k": k, "v": v, "scores": scores}


def exact_verify(st):
    """One sequence after another."""
    tokens, accepted = [], []
    for b in range(st["case"]["seqs"]):
        x = st["logits"][b].double() / st["temperature"][b].double()
        p = torch.softmax(x, -1)
        drafts = st["drafts"][b].tolist()
        rest, n = p[-1], len(drafts)
        for i, t in enumerate(drafts):
            q = torch.nn.functional.one_hot(torch.tensor(t), p.shape[-1]).to(p) if st["probs"] is None \
                else st["probs"][b, i].double()
            if not float(st["uniform"][b, i]) * float(q[t]) < float(p[i, t]):
                rest, n = (p[i] - q).clamp(min=0), i
                if not bool((rest > 0).any()):
                    rest = p[i]
                break
        nxt = int((rest / st["race"][b].double()).argmax())
        tokens.append(drafts[:n] + [nxt] + [-1] * (len(drafts) - n))
        accepted.append(n)
    return {"tokens": torch.tensor(tokens, dtype=torch.int32),
            "accepted": torch.tensor(accepted, dtype=torch.int32)}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        return exact_rotary(st)
    if op == "rotate":
        cos, sin = exact_angles(st)
        return exact_turn(st["x"].double(), cos, -sin if case["inverse"] else sin)
    return {"scored": exact_scored, "evict": exact_evict, "verify": exact_verify}[op](st)
