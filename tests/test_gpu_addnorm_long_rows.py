"""Rows of 8193 to 16384 columns, more of them than workgroups: each takes several, whose
columns' sums stand in LDS and whose weights are read again.  The bounds are those of
tests/test_gpu_addnorm.py."""

import pytest
import torch

from redpanda_amd.checkpoint8 import hip_pack8, hip_unpack8
from redpanda_amd.norm import hip_rmsnorm
from tests.test_gpu_addnorm import B, CHAIN, F, H, U, expect_sum, make, to_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("tx,ta,tout", [(F, B, B), (H, H, H), (B, None, F)])
@pytest.mark.parametrize("rows,d", [(700, 9000), (515, 16384)])
def test_several_rows_a_workgroup(gpu_lib, rows, d, tx, ta, tout, keep8):
    x, add, w, dy, ds = make(rows, d, tx, ta, tout, d + 2)
    total = expect_sum(x, add)
    leaves = [t.requires_grad_(True) for t in (x, w, add) if t is not None]
    outs = hip_rmsnorm(x, w, add=add, out_dtype=tout, keep8=keep8)
    out = outs if add is None else outs[1]
    got = torch.autograd.grad(outs, leaves, dy if add is None else (ds, dy))
    if add is not None:
        assert torch.equal(outs[0], total)
    f, wd = total.double(), w.detach().double()
    r = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-5)
    want = f * r * wd
    er = (CHAIN / 2 + 4) * U
    assert bool(((out.double() - want).abs() <= to_type(want, tout, want.abs() * (er + 2 * U))).all())
    if keep8:
        f = hip_unpack8(hip_pack8(total)).double()
        r = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-5)
    g = dy.double()
    q, xh = g * wd, f * r
    m = (q * xh).mean(-1, keepdim=True)
    dn = r * (q - xh * m)
    em = (CHAIN + 4) * U * (q * xh).abs().mean(-1, keepdim=True) + er * m.abs()
    tol = r * (3 * U * q.abs() + xh.abs() * em + (xh * m).abs() * (er + 3 * U)) + dn.abs() * er
    full = dn if add is None else dn + ds.double()
    tol = tol + U * full.abs()
    for i, t in ((0, tx), (2, ta)):
        if t is not None:
            assert got[i].dtype == t
            assert bool(((got[i].double() - full).abs() <= to_type(full, t, tol)).all())
    gx = g * xh
    assert bool(((got[1].double() - gx.sum(0)).abs() <= (er + (rows + 4) * U) * gx.abs().sum(0) + U * gx.sum(0).abs()).all())
