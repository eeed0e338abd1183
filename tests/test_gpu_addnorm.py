"""GPU parity of the RMS norm with the residual's addition, its backward, and rows in
8 bits, against the restatement in 64 bits (oracle/train_ref.py).

The sum is one fp32 addition rounded to its type, and 8 bits are exact by their
definition: both are compared bit for bit.  With U = 2^-24, a row's sums chains of at
most CHAIN additions, s the rows (or what 8 bits hold of them), r = 1 / sqrt(mean s^2 +
eps), xh = s r, q = g w:
    r:    er = (CHAIN / 2 + 4) U of it
    out:  |out| (er + 2 U), and its rounding
    m = mean(q xh):  em = (CHAIN + 4) U mean|q xh| + er |m|
    ds:   |r| (3 U |q| + |xh| em + |xh m| (er + 3 U)) + |norm's part| er + U |ds|, and its
          rounding
    dw:   (er + (rows + 4) U) sum |g xh|, and its rounding"""

import pytest
import torch

from oracle import train_ref as ref
from redpanda_amd.checkpoint8 import Packed8, hip_pack8, hip_unpack8
from redpanda_amd.norm import hip_add_rmsnorm, hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
CHAIN = 64
F, B, H = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F, None, F), (F, B, B), (F, F, F), (B, B, B), (H, H, H), (B, None, F), (H, B, H), (B, F, B)]


def to_type(v, t, bound):
    bound = bound + torch.finfo(t).eps / 2 * (v.abs() + bound)
    return bound + 2.0 ** -25 if t == H else bound


def within(name, got, want, tol):
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), (name, float((err / (tol + 1e-300)).max()))


def make(rows, d, tx, ta, tout, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = (randn(rows, d) * torch.exp(randn(rows, 1))).to(tx)
    add = None if ta is None else (0.5 * randn(rows, d)).to(ta)
    ts = tx if ta is None else torch.promote_types(tx, ta)
    return x, add, 1 + 0.1 * randn(d), randn(rows, d).to(tout), randn(rows, d).to(ts)


def expect_sum(x, add):
    if add is None:
        return x.detach()
    return (x.detach().float() + add.detach().float()).to(torch.promote_types(x.dtype, add.dtype))


def check(x, add, w, dy, ds, tout, eps=1e-5, keep8=False):
    rows, d = x.reshape(-1, x.shape[-1]).shape
    leaves = [t.requires_grad_(True) for t in (x, add, w) if t is not None]
    out = hip_rmsnorm(x, w, eps, add=add, out_dtype=tout, keep8=keep8)
    total = expect_sum(x, add)
    if add is None:
        outs, gouts = (out,), (dy,)
    else:
        assert torch.equal(out[0].detach(), total) and out[0].dtype == total.dtype
        outs, gouts = out, (ds, dy)
        out = out[1]
    assert out.dtype == tout and out.shape == x.shape
    s = total.cpu().double().reshape(rows, d)
    wd = torch.ones(d, dtype=torch.float64) if w is None else w.detach().cpu().double()
    want = ref.rmsnorm(s, wd, eps)
    er = (CHAIN / 2 + 4) * U
    within("out", out.reshape(rows, d), want, to_type(want, tout, want.abs() * (er + 2 * U)))
    grads = dict(zip(map(id, leaves), torch.autograd.grad(outs, leaves, gouts)))
    if keep8:
        s = ref.unpack8(*ref.pack8(s))
    s = s.requires_grad_(True)
    wl = wd.clone().requires_grad_(True)
    g = dy.cpu().double().reshape(rows, d)
    dn, dw = torch.autograd.grad(ref.rmsnorm(s, wl, eps), (s, wl), g)
    s = s.detach()
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    xh, q = s * r, g * wd
    m = (q * xh).mean(-1, keepdim=True)
    em = (CHAIN + 4) * U * (q * xh).abs().mean(-1, keepdim=True) + er * m.abs()
    tol = r * (3 * U * q.abs() + xh.abs() * em + (xh * m).abs() * (er + 3 * U)) + dn.abs() * er
    full = dn if add is None else dn + ds.cpu().double().reshape(rows, d)
    tol = tol + U * full.abs()
    for t, name in ((x, "dx"), (add, "dadd")):
        if t is not None:
            got = grads[id(t)]
            assert got.dtype == t.dtype and got.shape == t.shape
            within(name, got.reshape(rows, d), full, to_type(full, t.dtype, tol))
    if w is not None:
        tw = (er + (rows + 4) * U) * (g * xh).abs().sum(0)
        within("dw", grads[id(w)], dw, to_type(dw, w.dtype, tw))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("tx,ta,tout", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 5), (2, 64), (33, 100), (17, 384), (5, 768), (9, 1001),
                                    (130, 257)])
def test_forward_and_gradients(gpu_lib, rows, d, tx, ta, tout, keep8):
    x, add, w, dy, ds = make(rows, d, tx, ta, tout, rows * 1000 + d)
    check(x, add, w, dy, ds, tout, keep8=keep8)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("tx,ta,tout", [(F, B, B), (H, H, H), (B, None, F)])
@pytest.mark.parametrize("d", [127, 128, 129, 256, 257, 512, 513, 769, 1024, 1025, 1536, 1537, 2048, 2049,
                               4097, 8192, 8193, 16384, 16385, 20011])
def test_widths_of_every_shape(gpu_lib, d, tx, ta, tout, keep8):
    x, add, w, dy, ds = make(11, d, tx, ta, tout, d)
    check(x, add, w, dy, ds, tout, keep8=keep8)


@pytest.mark.parametrize("d", [40, 768, 1024, 5000])
def test_groups_that_walk_several_rows(gpu_lib, d):
    """More rows than the launch has groups, an uneven number for each."""
    rows = {40: 33000, 768: 9001, 1024: 9001, 5000: 2100}[d]
    x, add, w, dy, ds = make(rows, d, F, B, B, d + 1)
    out = hip_rmsnorm(x, w, add=add, out_dtype=B)
    total = expect_sum(x, add)
    assert torch.equal(out[0], total)
    f = total.double()
    r = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-5)
    want = f * r * w.double()
    er = (CHAIN / 2 + 4) * U
    assert bool(((out[1].double() - want).abs() <= to_type(want, B, want.abs() * (er + 2 * U))).all())
    for keep8 in (False, True):
        xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        got = torch.autograd.grad(hip_rmsnorm(xs, ws, add=add, out_dtype=B, keep8=keep8), (xs, ws), (ds, dy))
        f = total.double()
        if keep8:
            f = hip_unpack8(hip_pack8(total)).double()
        r = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-5)
        q, xh = dy.double() * w.double(), f * r
        m = (q * xh).mean(-1, keepdim=True)
        dn = r * (q - xh * m)
        em = (CHAIN + 4) * U * (q * xh).abs().mean(-1, keepdim=True) + er * m.abs()
        tol = r * (3 * U * q.abs() + xh.abs() * em + (xh * m).abs() * (er + 3 * U)) + dn.abs() * er
        full = dn + ds.double()
        assert bool(((got[0].double() - full).abs() <= (tol + 2 * U * full.abs())).all())
        gx = dy.double() * xh
        assert bool(((got[1].double() - gx.sum(0)).abs() <= (er + (rows + 4) * U) * gx.abs().sum(0)).all())


def test_without_weight_and_part_of_the_gradients(gpu_lib):
    x, add, w, dy, ds = make(37, 300, F, H, H, 5)
    check(x.clone(), add.clone(), None, dy, ds, H)
    full = hip_rmsnorm(x.requires_grad_(True), w.requires_grad_(True), add=add.requires_grad_(True), out_dtype=H)
    gx, ga, gw = torch.autograd.grad(full, (x, add, w), (ds, dy), retain_graph=True)
    for t, g in ((x, gx), (add, ga), (w, gw)):
        leaves = [p.detach() for p in (x, add, w)]
        i = [id(p) for p in (x, add, w)].index(id(t))
        leaves[i].requires_grad_(True)
        out = hip_rmsnorm(leaves[0], leaves[2], add=leaves[1], out_dtype=H)
        assert torch.equal(torch.autograd.grad(out, (leaves[i],), (ds, dy))[0], g)
    # only the sum, or only the norm, used
    (only,) = torch.autograd.grad(full[0], (x,), ds, retain_graph=True)
    assert torch.equal(only, ds)
    (both,) = torch.autograd.grad(full, (x,), (torch.zeros_like(ds), dy), retain_graph=True)
    (norm,) = torch.autograd.grad(full[1], (x,), dy)
    assert torch.equal(both, norm)


def test_the_step_norms_values(gpu_lib):
    """The same mathematics as the step's fp32 norm, to rounding."""
    x, add, w, _, _ = make(29, 384, F, F, F, 6)
    s0, o0 = hip_add_rmsnorm(x, add, w, 1e-5)
    s1, o1 = hip_rmsnorm(x, w, 1e-5, add=add)
    assert torch.equal(s0, s1)
    assert bool(((o0 - o1).abs() <= 2 * (CHAIN / 2 + 6) * U * o0.abs()).all())


def test_strides_and_leading_dimensions(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(3)
    big = torch.randn(21, 401, generator=g, device=dev)
    w = torch.randn(100, generator=g, device=dev)
    x, add = big[:, 1:101], big[:, 200:300]
    s, o = hip_rmsnorm(x, w, add=add)
    s2, o2 = hip_rmsnorm(x.contiguous(), w, add=add.contiguous())
    assert torch.equal(s, s2) and torch.equal(o, o2)
    t = torch.randn(4, 100, 5, generator=g, device=dev).transpose(1, 2)
    assert torch.equal(hip_rmsnorm(t, w), hip_rmsnorm(t.contiguous(), w))
    xl = x.detach().requires_grad_(True)
    o = hip_rmsnorm(xl, w)
    dy = torch.randn(21, 300, generator=g, device=dev)[:, 5:105]
    (a,) = torch.autograd.grad(o, (xl,), dy, retain_graph=True)
    (b,) = torch.autograd.grad(o, (xl,), dy.contiguous(), retain_graph=True)
    assert torch.equal(a, b)
    (c,) = torch.autograd.grad(o, (xl,), torch.ones((), device=dev).expand(21, 100))
    assert torch.isfinite(c).all()


def test_infinities_stay_in_their_rows(gpu_lib):
    x, add, w, dy, ds = make(8, 200, F, B, F, 7)
    s0, o0 = hip_rmsnorm(x, w, add=add)
    x2 = x.clone()
    x2[3, 10], x2[5, 199] = float("inf"), float("nan")
    s1, o1 = hip_rmsnorm(x2, w, add=add)
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(o0[keep], o1[keep]) and torch.equal(s0[keep], s1[keep])
    assert torch.isnan(o1[3, 10]) and o1[3, 11] == 0 and torch.isnan(o1[5]).all()
    # and in 8 bits, in their 32 columns
    p = hip_unpack8(hip_pack8(x2))
    assert torch.isnan(p[3, :32]).all() and torch.isfinite(p[3, 32:]).all()
    assert torch.isnan(p[5, 192:]).all() and torch.isfinite(p[5, :192]).all()


def test_zero_rows(gpu_lib):
    w = torch.ones(64, device=dev, requires_grad=True)
    x = torch.zeros(3, 64, device=dev, requires_grad=True)
    o = hip_rmsnorm(x, w, 1e-5, keep8=True)
    dx, dw = torch.autograd.grad(o, (x, w), torch.ones_like(o))
    # r = 1 / sqrt(eps), xh = 0
    assert o.abs().max() == 0 and dw.abs().max() == 0
    assert bool(((dx - 1e-5 ** -0.5).abs() <= 4e-7 * 1e-5 ** -0.5).all())
    e = torch.zeros(0, 64, device=dev, requires_grad=True)
    o = hip_rmsnorm(e, w)
    assert o.shape == (0, 64)
    assert torch.autograd.grad(o, (w,), o.detach())[0].abs().max() == 0


@pytest.mark.parametrize("t", [F, B, H])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 31), (5, 32), (4, 33), (7, 100), (6, 768), (3, 1001)])
def test_pack_bit_for_bit(gpu_lib, rows, d, t):
    g = torch.Generator(device=dev).manual_seed(rows * 37 + d)
    x = (torch.randn(rows, d, generator=g, device=dev) * torch.exp(4 * torch.randn(rows, 1, generator=g, device=dev))).to(t)
    x[0, 0] = 127.5
    p = hip_pack8(x)
    q, e = ref.pack8(x.cpu())
    assert torch.equal(p.q.cpu(), q) and torch.equal(p.e.cpu(), e)
    for out in (F, B, H):
        assert torch.equal(hip_unpack8(p, out).cpu(), ref.unpack8(q, e).to(out))
    assert hip_unpack8(p).dtype == t


def test_pack_ends_of_the_range(gpu_lib):
    big = torch.finfo(F).max
    x = torch.zeros(1, 256, device=dev)
    x[0, 0], x[0, 1] = big, -big / 3
    x[0, 32] = 2.0 ** -149
    x[0, 64] = 2.0 ** -126 * 127
    x[0, 96], x[0, 97] = 2.0 ** -120, -2.0 ** -127
    x[0, 128:160] = -0.0
    x[0, 160] = float("-inf")
    x[0, 192] = float("nan")
    x[0, 224] = 65504.0
    q, e = ref.pack8(x.cpu())
    p = hip_pack8(x)
    assert torch.equal(p.q.cpu(), q) and torch.equal(p.e.cpu(), e)
    got, want = hip_unpack8(p).cpu(), ref.unpack8(q, e).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_the_norm_packs_what_pack_packs(gpu_lib):
    from redpanda_amd.norm import norm_forward
    for d in (33, 100, 768, 1001, 3000, 20000):
        x, add, w, _, _ = make(9, d, F, B, B, d)
        total, _, kept, _, _ = norm_forward(x, add, w, 1e-5, B, True)
        p = hip_pack8(total)
        assert torch.equal(p.q, kept[0]) and torch.equal(p.e, kept[1])


def test_pack_shapes_and_strides(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(3, 5, 70, generator=g, device=dev)
    p = hip_pack8(x)
    assert p.shape == (3, 5, 70) and p.e.shape == (3, 5, 3)
    assert torch.equal(hip_unpack8(p), hip_unpack8(hip_pack8(x.reshape(15, 70))).reshape(3, 5, 70))
    v = torch.randn(6, 200, generator=g, device=dev)[:, 9:109]
    assert torch.equal(hip_pack8(v).q, hip_pack8(v.contiguous()).q)
    assert hip_unpack8(hip_pack8(x[:0])).shape == (0, 5, 70)
    assert hip_unpack8(hip_pack8(x[..., :0])).shape == (3, 5, 0)


def test_differences(gpu_lib):
    """dx along a direction against a central difference of the kernel's own values.
    f = sum dy out, about 300 values of unit size: each value is within (CHAIN / 2 + 6) U
    of it, so f(x + t v) - f(x - t v) within 2 sqrt(n) (the errors' signs vary; 4 times
    that is allowed) of it, over 2 t; the third derivative's part is t^2 / 6 of a few
    units."""
    g = torch.Generator(device=dev).manual_seed(9)
    x, v = torch.randn(4, 75, generator=g, device=dev), torch.randn(4, 75, generator=g, device=dev)
    w, dy = torch.randn(75, generator=g, device=dev), torch.randn(4, 75, generator=g, device=dev)
    xl = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(hip_rmsnorm(xl, w), (xl,), dy)
    t = 2.0 ** -7
    f = [(hip_rmsnorm(x + s * t * v, w).double() * dy.double()).sum() for s in (1, -1)]
    diff = (f[0] - f[1]) / (2 * t)
    slope = (dx.double() * v.double()).sum()
    noise = 4 * 2 * 300 ** 0.5 * (CHAIN / 2 + 6) * U * 4 / (2 * t)
    assert abs(float(diff - slope)) <= noise + t * t * 300


def test_captured_with_eager_work_between(gpu_lib):
    x, add, w, dy, ds = make(257, 768, F, B, B, 14)
    for t in (x, add, w):
        t.requires_grad_(True)
    for keep8 in (False, True):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(hip_rmsnorm(x, w, add=add, out_dtype=B, keep8=keep8), (x, add, w), (ds, dy))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = hip_rmsnorm(x, w, add=add, out_dtype=B, keep8=keep8)
            got = torch.autograd.grad(out, (x, add, w), (ds, dy))
        for seed in range(3):
            new = make(257, 768, F, B, B, 30 + seed)
            with torch.no_grad():
                for t, n in zip((x, add, w, dy, ds), new):
                    t.copy_(n)
            graph.replay()
            torch.cuda.synchronize()
            leaves = [t.detach().clone().requires_grad_(True) for t in (x, add, w)]
            want = hip_rmsnorm(leaves[0], leaves[2], add=leaves[1], out_dtype=B, keep8=keep8)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(want, leaves, (ds, dy))))


def test_refusals(gpu_lib):
    x, add, w, dy, _ = make(4, 50, F, B, F, 15)
    with pytest.raises(ValueError, match="last dimension"):
        hip_rmsnorm(x[:, :0])
    with pytest.raises(ValueError, match="add"):
        hip_rmsnorm(x, w, add=add[:3])
    with pytest.raises(ValueError, match="weight"):
        hip_rmsnorm(x, w[:49])
    with pytest.raises(ValueError, match="weight"):
        hip_rmsnorm(x, w.cpu())
    with pytest.raises(ValueError, match="eps"):
        hip_rmsnorm(x, w, -1.0)
    with pytest.raises(TypeError, match="dtype"):
        hip_rmsnorm(x.double(), w)
    with pytest.raises(TypeError, match="dtype"):
        hip_rmsnorm(x, w, add=add.double())
    with pytest.raises(TypeError, match="dtype"):
        hip_rmsnorm(x, w, out_dtype=torch.int8)
    with pytest.raises(TypeError, match="dtype"):
        hip_pack8(x.double())
    with pytest.raises(ValueError, match="dimension"):
        hip_pack8(x[0, 0])
    p = hip_pack8(x)
    with pytest.raises(ValueError, match="8 bits"):
        hip_unpack8(Packed8(p.q, p.e[:, :1], F))
    with pytest.raises(ValueError, match="8 bits"):
        hip_unpack8(Packed8(p.q.to(torch.uint8), p.e, F))
    with pytest.raises(TypeError, match="dtype"):
        hip_unpack8(p, torch.int32)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            hip_rmsnorm(dual, w)
    # a backward that would be differentiated again
    xl = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(hip_rmsnorm(xl, w), (xl,), dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
