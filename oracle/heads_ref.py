"""The head operators (dropout, layer norm, sampling) in 64 bits, on the CPU,
from their definitions: test infrastructure."""

import math

import numpy as np
import torch


def philox4x32(counter, key):
    """Philox4x32-10 (Salmon et al., 2011) of uint64 arrays holding 32-bit words:
    four counter words and two key words -> four output words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [np.uint64(int(key[0]) & 0xFFFFFFFF), np.uint64(int(key[1]) & 0xFFFFFFFF)]
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ k[0], b & low, (a >> sh) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def threshold(p):
    return round(65536 * p)


def drop_scale(p):
    t = threshold(p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def keep_mask(rows, d, p, seed, stream=0):
    """(len(rows), d) truth values: what dropout keeps in these rows."""
    rows = np.asarray(rows, dtype=np.uint64).reshape(-1, 1)
    nb = -(-d // 8)
    blk = np.broadcast_to(np.arange(nb, dtype=np.uint64), (rows.shape[0], nb))
    seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    words = philox4x32((blk, np.broadcast_to(rows & np.uint64(0xFFFFFFFF), blk.shape),
                        np.full(blk.shape, stream, np.uint64),
                        np.broadcast_to(rows >> np.uint64(32), blk.shape)),
                       (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    return torch.from_numpy(halves.reshape(rows.shape[0], nb * 8)[:, :d] >= np.uint64(threshold(p)))


def drop(x, p, keep):
    return torch.where(keep, x * drop_scale(p), torch.zeros_like(x))


def gelu(x):
    return x * 0.5 * torch.erfc(-x / math.sqrt(2.0))


def layernorm(x, w=None, b=None, eps=1e-5, use_gelu=False, p=0.0, keep=None):
    """fp64 rows in, fp64 rows out (differentiable)."""
    h = gelu(x) if use_gelu else x
    c = h - h.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return y if keep is None else drop(y, p, keep)


def sample_row(values, u, T=1.0, k=0, tp=1.0, mp=0.0):
    """(place, log-probability) of one row of float64 values; (-1, -inf) without
    a candidate."""
    values = np.asarray(values, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        pos = np.flatnonzero(values > -np.inf)
    if pos.size == 0:
        return -1, -math.inf
    order = pos[np.argsort(-values[pos], kind="stable")]
    top = values[order[0]]
    if not T > 0:
        return int(order[0]), 0.0
    if k > 0:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(values[order] == top, 1.0, np.exp((values[order] - top) / T))
    if top == np.inf:  # nothing else has a weight beside it, at T = inf either
        w[values[order] < top] = 0.0
    before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
    keep = (w >= mp) & ((tp >= 1.0) | (before < tp * w.sum()))
    keep[0] = True
    chosen = order[keep]
    w = w[keep]
    by = np.argsort(chosen)
    chosen, w = chosen[by], w[by]
    run = np.cumsum(w)
    i = min(int(np.searchsorted(run, u * run[-1], side="right")), len(w) - 1)
    while w[i] == 0.0 and i > 0:
        i -= 1
    return int(chosen[i]), float(math.log(w[i] / run[-1]))


def sample(logits, u, T=1.0, k=0, tp=1.0, mp=0.0, tokens=None):
    """(ids, logp) lists over rows; each setting a number or one a row."""
    R = len(logits)

    def of(v, r):
        return float(v[r]) if np.ndim(v) else float(v)

    ids, logp = [], []
    for r in range(R):
        row = np.asarray(logits[r], dtype=np.float64)
        if tokens is not None:
            t = np.asarray(tokens[r], dtype=np.int64)
            ok = (t >= 0) & (t < row.size)
            row = np.where(ok, row[np.where(ok, t, 0)], -np.inf)
        i, lp = sample_row(row, float(u[r]), of(T, r), int(of(k, r)), of(tp, r), of(mp, r))
        ids.append(i if i < 0 or tokens is None else int(tokens[r][i]))
        logp.append(lp)
    return ids, logp
