"""Gated recurrences whose workgroups take several turns of steps: the state and the
gradient carried from turn to turn, both halves of the LDS, the steps loaded ahead in the
sums of a split, and more chunks than the fold's waves take at once.  The bounds are those
of tests/test_gpu_gated.py."""

import pytest
import torch

from redpanda_amd.gated import hip_gated_scan
from tests.test_gpu_gated import TYPES, U, check, make, to_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,L,D,starts", [
    (200, 2501, 3, 0.0),    # split into chunks of 256 steps, four turns each, the last of them cut
    (200, 2501, 3, 0.004),
    (300, 203, 66, 0.0),    # whole sequences by four waves: four turns, the last of them cut
    (300, 203, 66, 0.02),
    (1, 20000, 5, 0.0005),  # 313 chunks: a wave of the fold takes 20
])
def test_several_turns(gpu_lib, B, L, D, starts, t):
    check(*make(B, L, D, t, L + D, True, starts))


@pytest.mark.parametrize("t", TYPES)
def test_several_turns_of_wide_rows(gpu_lib, t):
    """The same bounds with the 64-bit side on the device: 20 million values."""
    x, z, h0, st, dy, dh = make(60, 2500, 130, t, 3, True, 0.002)
    leaves = [v.detach().requires_grad_(True) for v in (x, z, h0)]
    y, last = hip_gated_scan(leaves[0], leaves[1], leaves[2], st)
    got = torch.autograd.grad((y, last), leaves, (dy, dh))
    xd, zd, h, l = x.detach().double(), z.detach().double(), h0.double(), dh.double()
    a, na, go = torch.sigmoid(zd), torch.sigmoid(-zd), (~st).double()[..., None]
    eg = (2 * zd.abs() + 6) * U
    hs, prev, Es, Ep = (torch.empty_like(xd) for _ in range(4))
    E = torch.zeros_like(h)
    for k in range(x.shape[1]):
        prev[:, k], Ep[:, k] = h * go[:, k], E * go[:, k]
        kept, taken = a[:, k] * prev[:, k], na[:, k] * xd[:, k]
        E = a[:, k] * Ep[:, k] + (eg[:, k] + 3 * U) * (kept.abs() + taken.abs())
        h = kept + taken
        hs[:, k], Es[:, k] = h, E
    ls, Els = torch.empty_like(xd), torch.empty_like(xd)
    El = torch.zeros_like(h)
    for k in range(x.shape[1] - 1, -1, -1):
        l = dy[:, k].double() + l
        El = El + 2 * U * l.abs()
        ls[:, k], Els[:, k] = l, El
        El = (a[:, k] * El + (eg[:, k] + 3 * U) * (a[:, k] * l).abs()) * go[:, k]
        l = a[:, k] * l * go[:, k]
    Es, Ep, Els = 2 * Es, 2 * Ep, 2 * Els
    dx, dz = na * ls, (prev - xd) * a * na * ls
    tz = a * na * ((prev - xd).abs() * Els + ls.abs() * (Ep + 2 * U * (prev.abs() + xd.abs())))
    for name, g, want, tol in (("y", y, hs, to_type(hs, t, Es)), ("last", last, h, Es[:, -1]),
                               ("dx", got[0], dx, to_type(dx, t, na * Els + (eg + 2 * U) * dx.abs())),
                               ("dz", got[1], dz, to_type(dz, t, tz + (2 * eg + 6 * U) * dz.abs())),
                               ("dh0", got[2], l, 2 * El + 2 * U * l.abs())):
        assert bool(((g.detach().double() - want).abs() <= tol).all()), name


def test_long_memory_over_turns(gpu_lib):
    """Gates near 1: what enters a turn matters to the end."""
    for B, L, D in ((200, 1203, 5), (300, 203, 66)):
        x, z, h0, _, dy, dh = make(B, L, D, torch.float32, 5)
        check(x, (z.abs() + 5).detach(), 100 * h0, None, dy, dh)
