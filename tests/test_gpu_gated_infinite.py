"""Infinite states and gradients of the gated recurrence.  a_t is above 0 for every
finite gate that fp32's exp does not round to 0, and an infinity times it stays one, for
as many steps as the sequence has and however these are split; 0 times an infinity, by a
gate of -inf, is NaN.  Compared with the formula in 64 bits: which values are infinite,
of which sign, and which are NaN."""

import pytest
import torch

from redpanda_amd.gated import hip_gated_scan

pytestmark = pytest.mark.gpu
dev = "cuda"
INF = float("inf")


def same_kind(name, got, want, sure=None):
    got = got.detach().double()
    if sure is not None:
        got, want = got[sure], want[sure]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), name


def make(B, L, D, t, level, seed):
    """Gates around `level`, so that a product over a stretch underflows or not."""
    g = torch.Generator(device=dev).manual_seed(seed)
    z = (level + 0.5 * torch.randn(B, L, D, generator=g, device=dev)).to(t)
    x, dy = (torch.randn(B, L, D, generator=g, device=dev).to(t) for _ in range(2))
    return x, z, torch.randn(B, D, generator=g, device=dev), dy, torch.randn(B, D, generator=g, device=dev)


def formula(x, z, h0, dy, dh, st):
    """(y, dx, dz, dh0) step by step in 64 bits, and where dz's two factors are not so near
    0 that fp32 may give another sign (a state of size 1 is within 1e-5 there)."""
    x, z, h, dy, l = (t.double() for t in (x, z, h0, dy, dh))
    B, L, D = x.shape
    a, na = torch.sigmoid(z), torch.sigmoid(-z)
    y, prev = torch.empty_like(x), torch.empty_like(x)
    for t in range(L):
        if st is not None:
            h = torch.where(st[:, t, None], 0.0, h)
        prev[:, t] = h
        h = a[:, t] * h + na[:, t] * x[:, t]
        y[:, t] = h
    dx, dz, sure = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x, dtype=torch.bool)
    for t in range(L - 1, -1, -1):
        s = dy[:, t] + l
        sure[:, t] = ~(((prev[:, t] - x[:, t]).abs() <= 1e-4) | (s.abs() <= 1e-4))
        dx[:, t], dz[:, t] = s * na[:, t], s * ((prev[:, t] - x[:, t]) * (a[:, t] * na[:, t]))
        l = a[:, t] * s
        if st is not None:
            l = torch.where(st[:, t, None], 0.0, l)
    return y, dx, dz, l, sure


# a lane a channel and all steps at once; split along time in one turn of 64 steps and in
# several; four waves over the whole sequence; one wave; a single step's kernel
SHAPES = [(2, 250, 40), (1, 700, 50), (200, 2501, 3), (300, 203, 66), (40, 12, 30), (3, 4, 8)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("level", [-9.0, -3.0, 3.0])
@pytest.mark.parametrize("starts", [False, True])
@pytest.mark.parametrize("B,L,D", SHAPES)
def test_an_infinity_stays_one(gpu_lib, B, L, D, starts, level, t):
    x, z, h0, dy, dh = make(B, L, D, t, level, L + D)
    h0[:, 0], dh[:, 1] = INF, -INF
    x[:, L // 3, 2], dy[:, L - 1 - L // 5, 2] = -INF, INF
    st = None
    if starts:
        st = torch.zeros(B, L, dtype=torch.bool, device=dev)
        st[:, L // 2] = True
        st[:, L - 1] = L > 100
    want = formula(x, z, h0, dy, dh, st)
    leaves = [v.clone().requires_grad_(True) for v in (x, z, h0)]
    y, last = hip_gated_scan(*leaves, starts=st)
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    assert bool(torch.isinf(want[0]).any()) and bool(torch.isinf(want[1]).any())
    same_kind("y", y, want[0])
    same_kind("last", last, want[0][:, -1])
    for name, got, w, sure in zip(("dx", "dz", "dh0"), grads, want[1:], (None, want[4], None)):
        same_kind(name, got, w, sure)


@pytest.mark.parametrize("B,L,D", SHAPES[:4])
def test_a_closed_gate_makes_it_nan(gpu_lib, B, L, D):
    x, z, h0, dy, dh = make(B, L, D, torch.float32, -3.0, 5)
    h0[:, 0], dh[:, 1] = INF, -INF
    z[:, L // 3] = -INF
    want = formula(x, z, h0, dy, dh, None)
    leaves = [v.clone().requires_grad_(True) for v in (x, z, h0)]
    y, last = hip_gated_scan(*leaves)
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    assert bool(torch.isnan(want[0]).any())
    same_kind("y", y, want[0])
    for name, got, w, sure in zip(("dx", "dz", "dh0"), grads, want[1:], (None, want[4], None)):
        same_kind(name, got, w, sure)
