"""The training operators (embedding, rows in 8 bits, RMS norm with the residual's
addition, the gated recurrence) in 64 bits, on the CPU, from their definitions: test
infrastructure."""

import math

import numpy as np
import torch

BLOCK = 32


def embedding(ids, w, scale, dout=None, padding_idx=None):
    """scale w[ids] (zeros for ids outside the table), or with dout the table's
    gradient."""
    ids = ids.reshape(-1).tolist()
    V, d = w.shape
    if dout is None:
        out = torch.zeros(len(ids), d, dtype=torch.float64)
        for i, v in enumerate(ids):
            if 0 <= v < V:
                out[i] = scale * w[v].double()
        return out
    dw = torch.zeros(V, d, dtype=torch.float64)
    for i, v in enumerate(ids):
        if 0 <= v < V and v != padding_idx:
            dw[v] += dout.reshape(len(ids), d)[i].double()
    return scale * dw


def pack8(x):
    """(q int8, e uint8) of rows x, one block of 32 columns after another."""
    x = x.double().numpy()
    rows, d = x.shape
    nb = -(-d // BLOCK)
    q, e = np.zeros((rows, d), np.int8), np.zeros((rows, nb), np.uint8)
    for r in range(rows):
        for j in range(nb):
            v = x[r, j * BLOCK:(j + 1) * BLOCK]
            top = np.abs(v).max()
            if not np.isfinite(top):
                e[r, j] = 255
                continue
            E = -126
            if top > 0:
                # the least power that rounds the largest to at most 127
                E = max(-126, math.frexp(top)[1] - 9)
                while abs(np.rint(top / 2.0 ** E)) > 127:
                    E += 1
            e[r, j] = E + 127
            q[r, j * BLOCK:(j + 1) * BLOCK] = np.rint(v / 2.0 ** E).astype(np.int8)
    return torch.from_numpy(q), torch.from_numpy(e)


def unpack8(q, e):
    d = q.shape[1]
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127)
    step = torch.where(e == 255, torch.nan, step)
    return q.double() * step.repeat_interleave(BLOCK, dim=1)[:, :d]


def rmsnorm(s, w, eps):
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * r * w


def gated(x, z, h0=None, starts=None):
    """All states (B, L, D); differentiable."""
    B, L, D = x.shape
    h = torch.zeros(B, D, dtype=x.dtype) if h0 is None else h0
    ys = []
    for t in range(L):
        a = torch.sigmoid(z[:, t])
        if starts is not None:
            h = torch.where(starts[:, t, None], torch.zeros_like(h), h)
        h = a * h + torch.sigmoid(-z[:, t]) * x[:, t]
        ys.append(h)
    return torch.stack(ys, dim=1)
