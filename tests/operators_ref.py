"""64-bit restatements (numpy) of the rotary, scored-attention, eviction and verification
operators, and the page plumbing their tests share.

Unit roundoffs: a value stored in a type with p significant bits is off by at most 2^-p of itself
(f32 24, f16 11, bf16 8, E4M3 4 bits), plus half the spacing of its subnormals.
"""
import numpy as np
import torch

ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
         torch.float8_e4m3fn: 2.0 ** -4}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float8_e4m3fn: 2.0 ** -10}


def f64(t):
    return t.detach().double().cpu().numpy() if t.element_size() > 1 else t.detach().float().double().cpu().numpy()


def axis_of(sections, interleaved):
    n, half = len(sections), sum(sections)
    if not interleaved:
        return np.repeat(np.arange(n), sections)
    axes = np.zeros(half, int)
    for a in range(1, n):
        for k in range(sections[a]):
            axes[a + k * n] = a
    return axes


def rotate(x, cos, sin, positions, sections, interleaved, inverse=False):
    """x [T, H, D], positions [A, T]; f64."""
    half = sum(sections)
    axes = axis_of(sections, interleaved)
    pos = positions[axes].T                                   # [T, half]
    i = np.arange(half)
    c, s = cos[pos, i][:, None], sin[pos, i][:, None] * (-1 if inverse else 1)
    y = x.copy()
    a, b = x[..., :half], x[..., half:2 * half]
    y[..., :half] = a * c - b * s
    y[..., half:2 * half] = b * c + a * s
    return y


def rms_norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def token_major(key_cache, value_cache):
    """[blocks * bs, H, D] views of K and V pages (f64)."""
    k, v = f64(key_cache), f64(value_cache)
    nb, h, dx, bs, x = k.shape
    return (k.transpose(0, 3, 1, 2, 4).reshape(nb * bs, h, dx * x),
            v.transpose(0, 3, 1, 2).reshape(nb * bs, h, -1))


def slots_of(table, n, bs):
    j = np.arange(n)
    return table[j // bs].astype(np.int64) * bs + j % bs


def scored(q, key_cache, value_cache, scores, tables, lens, scale, softcap=1.0, decay=1.0, score_rows=None,
           k_scale=1.0, v_scale=1.0):
    """q [B, W, Hq, D] -> (out, scores, weights' sums, largest sum |q k| scale); all f64."""
    kt, vt = token_major(key_cache, value_cache)
    kt, vt = kt * k_scale, vt * v_scale
    q, scores = f64(q), f64(scores)
    b, w, hq, d = q.shape
    nb, hkv, bs = scores.shape
    g = hq // hkv
    rows = w if score_rows is None else score_rows
    out = np.zeros_like(q)
    flat = scores.transpose(0, 2, 1).reshape(nb * bs, hkv).copy()
    added = np.zeros_like(flat)
    reach = 0.0
    for i in range(b):
        n = int(lens[i])
        sl = slots_of(tables[i], n, bs)
        for r in range(w):
            m = n - w + r + 1
            if m <= 0:
                continue
            for h in range(hq):
                k = kt[sl[:m], h // g]
                x = k @ q[i, r, h] * scale
                reach = max(reach, float(np.nanmax(np.abs(k) @ np.abs(q[i, r, h]) * scale)))
                if softcap != 1.0:
                    x = softcap * np.tanh(x / softcap)
                p = np.exp(x - x.max())
                p /= p.sum()
                out[i, r, h] = p @ vt[sl[:m], h // g]
                if r < rows:
                    added[sl[:m], h // g] += p
        flat[sl] = decay * flat[sl] + added[sl]
    return (out, flat.reshape(nb, bs, hkv).transpose(0, 2, 1), added.reshape(nb, bs, hkv).transpose(0, 2, 1), reach)


def evict_indices(scores, tables, lens, budgets, sink, recent):
    """[[ascending kept indices per head] per sequence] from f32 scores [nb, H, bs]."""
    nb, hkv, bs = scores.shape
    kept = []
    for i, n in enumerate(lens):
        n = int(n)
        per_head = []
        for h in range(hkv):
            j = np.arange(n)
            s = scores[tables[i][j // bs], h, j % bs].astype(np.float64)
            s = np.where(np.isnan(s), -np.inf, s)
            always = (j < sink) | (j >= n - recent)
            order = sorted(range(n), key=lambda t: (not always[t], -s[t] if not always[t] else 0.0, t))
            per_head.append(sorted(order[:min(int(budgets[i]), n)]))
        kept.append(per_head)
    return kept


def verify(logits, drafts, probs, uniform, race, temps, lens=None):
    """f64; logits [B, K + 1, V] -> (tokens [B, K + 1], accepted [B])."""
    b, k1, v = logits.shape
    tokens, accepted = np.full((b, k1), -1, np.int64), np.zeros(b, np.int64)
    x = np.where(np.isnan(logits), -np.inf, logits)
    for i in range(b):
        k = k1 - 1 if lens is None else int(lens[i])
        t = temps[i]

        def row(r):
            m = x[i, r].max()
            if m == -np.inf:
                return None
            if m == np.inf:
                p = (x[i, r] == m).astype(np.float64)
            else:
                p = np.exp((x[i, r] - m) / t)
            return p / p.sum()

        n = 0
        while n < k:
            d = int(drafts[i, n])
            if d < 0 or d >= v or x[i, n].max() == -np.inf:
                break
            if t > 0:
                qd = 1.0 if probs is None else float(probs[i, n, d])
                if not float(uniform[i, n]) * qd < row(n)[d]:
                    break
            elif d != int(x[i, n].argmax()):
                break
            n += 1
        if x[i, n].max() == -np.inf:
            nxt = 0
        elif t > 0:
            p = row(n)
            r = p
            if n < k:
                q = np.zeros(v)
                if probs is not None:
                    q = probs[i, n].astype(np.float64)
                    r = np.maximum(p - q, 0)
                else:
                    r = p.copy()
                    if 0 <= drafts[i, n] < v:
                        r[drafts[i, n]] = 0
            if not (r > 0).any():
                r = p
            with np.errstate(divide="ignore", invalid="ignore"):
                a = np.where(r > 0, r / race[i].astype(np.float64), -1.0)
            nxt = int(a.argmax())
        else:
            nxt = int(x[i, n].argmax())
        tokens[i, :n] = drafts[i, :n]
        tokens[i, n] = nxt
        accepted[i] = n
    return tokens, accepted


# ------------------------------------------------------------------------------- page pools
def make_pool(rng, lens, hkv, d, bs, dtype, device, extra_cols=0, spare=2, fill=True):
    """Pages with seeded values in every token below ``lens`` and NaN everywhere else."""
    cols = [max(1, -(-int(n) // bs)) for n in lens]
    nb = sum(cols) + 1 + spare
    ids = rng.permutation(np.arange(1, nb))[:sum(cols)]
    tables = np.zeros((len(lens), max(cols) + extra_cols), np.int32)
    at = 0
    for i, c in enumerate(cols):
        tables[i, :c] = ids[at:at + c]
        at += c
    es = torch.empty((), dtype=dtype).element_size()
    x = 16 // es
    k = torch.full((nb * bs, hkv, d), float("nan"))
    v = torch.full((nb * bs, hkv, d), float("nan"))
    if fill:
        for i, n in enumerate(lens):
            sl = slots_of(tables[i], int(n), bs)
            k[sl] = torch.from_numpy(rng.standard_normal((len(sl), hkv, d), np.float32))
            v[sl] = torch.from_numpy(rng.standard_normal((len(sl), hkv, d), np.float32))
    kc = k.view(nb, bs, hkv, d // x, x).permute(0, 2, 3, 1, 4).contiguous().to(dtype)
    vc = v.view(nb, bs, hkv, d).permute(0, 2, 3, 1).contiguous().to(dtype)
    return kc.to(device), vc.to(device), tables


def raw(t):
    """The bits of a tensor, as whole numbers on the host."""
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).cpu().numpy()
