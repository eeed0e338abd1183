"""GPU parity of the gated recurrence and its backward against the restatement in 64
bits (oracle/train_ref.py).

With U = 2^-24: a = 1 / (1 + exp(-z)) comes from exp2(|z| log2 e), whose argument is off
by 2 U of |z| log2 e, so that exp(-|z|) is off by (2 |z| + 2) U of it; each of a and 1 -
a is off by eg = (2 |z| + 6) U of it at most.  A state's error, E_t = a (E_{t-1}) +
(eg + 3 U) (|a h_{t-1}| + |(1 - a) x|), is carried along in the test; a sequence that is
split along time forms the same products in another order, for which the bound is
doubled.  The gradients' errors are carried the same way from the other end:
    l:   El_t = a_{t+1} (El_{t+1}) + (eg + 3 U) |a_{t+1} l_{t+1}| + U |l|
    dx:  |1 - a| El + (eg + 2 U) |dx|
    dz:  a (1 - a) (|h - x| El + |l| (E_{t-1} + 2 U (|h_{t-1}| + |x|))) + (2 eg + 6 U) |dz|
and the rounding to their type is added."""

import pytest
import torch

from oracle import train_ref as ref
from redpanda_amd.gated import hip_gated_scan, hip_gated_step

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def to_type(v, t, bound):
    bound = bound + torch.finfo(t).eps / 2 * (v.abs() + bound)
    return bound + 2.0 ** -25 if t == torch.float16 else bound


def within(name, got, want, tol):
    err = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= tol).all()), (name, float((err / (tol + 1e-300)).max()))


def make(B, L, D, t, seed, state=True, starts=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    both = randn(B, L, 2 * D)
    both[..., D:] = 2 * both[..., D:] + 4 * torch.rand(D, generator=g, device=dev)
    both = both.to(t)
    h0 = randn(B, D) if state else None
    st = torch.rand(B, L, generator=g, device=dev) < starts if starts else None
    return both[..., :D], both[..., D:], h0, st, randn(B, L, D).to(t), randn(B, D)


def check(x, z, h0, st, dy, dh):
    B, L, D = x.shape
    leaves = [t.detach().requires_grad_(True) for t in (x, z, h0) if t is not None]
    y, last = hip_gated_scan(leaves[0], leaves[1], h0=leaves[2] if h0 is not None else None, starts=st)
    assert y.dtype == x.dtype and last.dtype == torch.float32
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    xd, zd = cpu(x).double().requires_grad_(True), cpu(z).double().requires_grad_(True)
    hd = (torch.zeros(B, D, dtype=torch.float64) if h0 is None else cpu(h0).double()).requires_grad_(True)
    sd = cpu(st)
    h = ref.gated(xd, zd, hd, sd)
    want = torch.autograd.grad((h, h[:, -1]), (xd, zd, hd), (cpu(dy).double(), cpu(dh).double()))
    with torch.no_grad():
        a, na = torch.sigmoid(zd), torch.sigmoid(-zd)
        eg = (2 * zd.abs() + 6) * U
        go = torch.ones(B, L, 1, dtype=torch.float64) if sd is None else (~sd).double()[..., None]
        prev = torch.cat((hd[:, None], h[:, :-1]), 1) * go
        E, Es, Ep = torch.zeros(B, D, dtype=torch.float64), [], []
        for t in range(L):
            E = E * go[:, t]
            Ep.append(E)
            E = a[:, t] * E + (eg[:, t] + 3 * U) * ((a * prev)[:, t].abs() + (na * xd)[:, t].abs())
            Es.append(E)
        E, Ep = 2 * torch.stack(Es, 1), 2 * torch.stack(Ep, 1)
        within("y", y, h, to_type(h, y.dtype, E))
        within("last", last, h[:, -1], E[:, -1])
        l, El, ls, Els = cpu(dh).double(), torch.zeros(B, D, dtype=torch.float64), [], []
        for t in range(L - 1, -1, -1):
            l = cpu(dy).double()[:, t] + l
            El = El + 2 * U * l.abs()
            ls.append(l)
            Els.append(El)
            El = (a[:, t] * El + (eg[:, t] + 3 * U) * (a[:, t] * l).abs()) * go[:, t]
            l = a[:, t] * l * go[:, t]
        El0 = 2 * El
        ls, Els = torch.stack(ls[::-1], 1), 2 * torch.stack(Els[::-1], 1)
        within("dx", grads[0], want[0], to_type(want[0], x.dtype, na * Els + (eg + 2 * U) * want[0].abs()))
        tz = a * na * ((prev - xd).abs() * Els + ls.abs() * (Ep + 2 * U * (prev.abs() + xd.abs())))
        within("dz", grads[1], want[1], to_type(want[1], x.dtype, tz + (2 * eg + 6 * U) * want[1].abs()))
        if h0 is not None:
            within("dh0", grads[2], want[2], El0 + 2 * U * want[2].abs())
    return y, last, grads


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("state,starts", [(False, 0.0), (True, 0.0), (True, 0.1)])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (3, 1, 40), (2, 3, 5), (1, 7, 2), (3, 17, 64), (2, 33, 130),
                                   (1, 130, 257), (2, 16, 3), (5, 64, 100)])
def test_states_and_gradients(gpu_lib, B, L, D, state, starts, t):
    check(*make(B, L, D, t, B * 1000 + L * 10 + D, state, starts))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,L,D,starts", [(1, 1000, 66, 0.01), (2, 515, 33, 0.0), (1, 2049, 129, 0.002),
                                          (3, 128, 1, 0.05), (600, 20, 130, 0.1), (1200, 3, 64, 0.0)])
def test_split_along_time_and_many_rows(gpu_lib, B, L, D, starts, t):
    check(*make(B, L, D, t, L + D, True, starts))


def test_long_memory_across_chunks(gpu_lib):
    """Gates near 1: what enters a chunk matters to its end."""
    x, z, h0, _, dy, dh = make(1, 3000, 34, torch.float32, 5)
    check(x, (z.abs() + 5).detach(), 100 * h0, None, dy, dh)


def test_step_is_the_scan(gpu_lib):
    x, z, h0, _, _, _ = make(70, 9, 48, torch.bfloat16, 6)
    y, last = hip_gated_scan(x, z, h0)
    h = h0
    for t in range(9):
        yt, h = hip_gated_step(x[:, t], z[:, t], h)
        assert torch.equal(yt, y[:, t])
    assert torch.equal(h, last)
    y0, h = hip_gated_step(x[:, 0], z[:, 0])
    assert torch.equal(y0, hip_gated_scan(x[:, :1], z[:, :1])[0][:, 0])


def test_infinite_gates(gpu_lib):
    """+inf keeps the state (and passes no gradient to x and the gate), -inf takes x."""
    x, z, h0, _, dy, dh = make(2, 20, 37, torch.float32, 7)
    z = z.contiguous()
    z[:, 5] = float("inf")
    z[:, 9] = float("-inf")
    z[:, 15:] = float("inf")
    xl, zl, hl = (t.detach().clone().requires_grad_(True) for t in (x, z, h0))
    y, last = hip_gated_scan(xl, zl, hl)
    assert torch.equal(y[:, 5], y[:, 4]) and torch.equal(y[:, 9], x[:, 9])
    assert torch.equal(last, y[:, 14]) and torch.equal(y[:, 19], y[:, 14])
    gx, gz, gh = torch.autograd.grad((y, last), (xl, zl, hl), (dy, dh))
    assert gx[:, 5].abs().max() == 0 and gx[:, 15:].abs().max() == 0
    assert gz[:, [5, 9, 15, 19]].abs().max() == 0
    assert torch.isfinite(gx).all() and torch.isfinite(gz).all() and torch.isfinite(gh).all()
    # the padding's gradients reach the last real step
    z2, dy2 = z[:, :15], dy[:, :15].clone()
    dy2[:, 14] += dy[:, 15:].sum(1)
    xs = x[:, :15].detach().clone().requires_grad_(True)
    zs = z2.detach().clone().requires_grad_(True)
    y2, l2 = hip_gated_scan(xs, zs, h0)
    assert torch.equal(y2, y[:, :15])
    g2 = torch.autograd.grad((y2, l2), (xs,), (dy2, dh))[0]
    assert bool(((g2 - gx[:, :15]).abs() <= 64 * U * (1 + g2.abs()) * 8).all())


@pytest.mark.parametrize("L", [40, 700])
def test_a_start_passes_nothing_on(gpu_lib, L):
    """Sequences packed in one row are those sequences by themselves, whatever stands
    before them: infinities and NaN too."""
    x, z, h0, _, dy, dh = make(1, L, 50, torch.float32, 8)
    cuts = [0, 7, 8, L // 2, L - 3, L]
    st = torch.zeros(1, L, dtype=torch.bool, device=dev)
    st[0, cuts[1:-1]] = True
    x = x.detach().clone()
    x[0, 3, 5], x[0, 20, 6], x[0, 22, 7] = float("inf"), float("nan"), float("-inf")
    xl, zl = x.clone().requires_grad_(True), z.detach().clone().requires_grad_(True)
    y, last = hip_gated_scan(xl, zl, h0, st)
    g = torch.autograd.grad((y, last), (xl, zl), (dy, dh))
    for i in range(len(cuts) - 1):
        a, b = cuts[i], cuts[i + 1]
        xs, zs = (t.detach()[:, a:b].clone().requires_grad_(True) for t in (x, z))
        ys, ls = hip_gated_scan(xs, zs, h0 if i == 0 else None)
        gs = torch.autograd.grad((ys, ls), (xs, zs), (dy[:, a:b], dh if b == L else torch.zeros_like(dh)))
        for p, q in ((y[:, a:b], ys), (g[0][:, a:b], gs[0]), (g[1][:, a:b], gs[1])):
            assert torch.equal(torch.isnan(p), torch.isnan(q))
            assert torch.equal(torch.isinf(p), torch.isinf(q))
            fine = torch.isfinite(q)
            # (the splits along time differ: sums of up to L terms in another order)
            assert bool(((p - q)[fine].abs() <= 1e-5 * (1 + q[fine].abs())).all())


def test_every_step_a_start(gpu_lib):
    x, z, h0, _, dy, dh = make(2, 300, 20, torch.float32, 9)
    st = torch.ones(2, 300, dtype=torch.bool, device=dev)
    y, _, grads = check(x, z, h0, st, dy, dh)
    assert grads[2].abs().max() == 0


def test_strides(gpu_lib):
    x, z, h0, _, dy, dh = make(4, 30, 40, torch.bfloat16, 10)
    want = hip_gated_scan(x.contiguous(), z.contiguous(), h0)
    assert all(torch.equal(a, b) for a, b in zip(hip_gated_scan(x, z, h0), want))
    tx = x.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert all(torch.equal(a, b) for a, b in zip(hip_gated_scan(tx, z, h0), want))
    cx = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert all(torch.equal(a, b) for a, b in zip(hip_gated_scan(cx, z, h0), want))
    # an odd offset, a broadcast batch, a broadcast time
    buf = torch.empty(4 * 30 * 41 + 3, dtype=torch.bfloat16, device=dev)
    ox = buf[3:].view(4, 30, 41)[..., 1:]
    ox.copy_(x)
    assert all(torch.equal(a, b) for a, b in zip(hip_gated_scan(ox, z, h0), want))
    ex = x[:1].expand(4, 30, 40)
    assert all(torch.equal(a, b) for a, b in
               zip(hip_gated_scan(ex, z, h0), hip_gated_scan(ex.contiguous(), z, h0)))
    zl = z[:, :1].detach().clone().requires_grad_(True)
    y, last = hip_gated_scan(x, zl.expand(4, 30, 40), h0)
    (g,) = torch.autograd.grad((y, last), (zl,), (torch.ones((), dtype=torch.bfloat16, device=dev).expand(4, 30, 40), dh))
    assert g.shape == (4, 1, 40) and torch.isfinite(g).all()


def test_part_of_the_gradients(gpu_lib):
    x, z, h0, st, dy, dh = make(2, 50, 24, torch.float32, 11, True, 0.1)
    full = check(x, z, h0, st, dy, dh)[2]
    for i in range(3):
        ts = [t.detach().clone() for t in (x, z, h0)]
        ts[i].requires_grad_(True)
        out = hip_gated_scan(*ts, starts=st)
        assert torch.equal(torch.autograd.grad(out, (ts[i],), (dy, dh))[0], full[i])
    xl = x.detach().clone().requires_grad_(True)
    y, last = hip_gated_scan(xl, z, h0, st)
    a = torch.autograd.grad(y, (xl,), dy, retain_graph=True)[0]
    b = torch.autograd.grad(last, (xl,), dh, retain_graph=True)[0]
    both = torch.autograd.grad((y, last), (xl,), (dy, dh), retain_graph=True)[0]
    za = torch.autograd.grad((y, last), (xl,), (dy, torch.zeros_like(dh)), retain_graph=True)[0]
    zb = torch.autograd.grad((y, last), (xl,), (torch.zeros_like(dy), dh))[0]
    assert torch.equal(a, za) and torch.equal(b, zb)
    assert bool(((a + b - both).abs() <= 64 * U * (a.abs() + b.abs() + both.abs()) + 1e-12).all())


def test_nothing(gpu_lib):
    h0 = torch.randn(2, 6, device=dev, requires_grad=True)
    e = torch.zeros(2, 0, 6, device=dev)
    y, last = hip_gated_scan(e, e, h0)
    assert y.shape == (2, 0, 6) and torch.equal(last, h0)
    assert torch.equal(torch.autograd.grad(last.sum(), (h0,))[0], torch.ones_like(h0))
    assert hip_gated_scan(e, e)[1].abs().max() == 0
    assert hip_gated_scan(torch.zeros(0, 3, 6, device=dev), torch.zeros(0, 3, 6, device=dev))[1].shape == (0, 6)
    assert hip_gated_scan(torch.zeros(2, 3, 0, device=dev), torch.zeros(2, 3, 0, device=dev))[0].shape == (2, 3, 0)


def test_the_same_bits_each_time_and_captured(gpu_lib):
    x, z, h0, st, dy, dh = make(1, 1500, 66, torch.float32, 12, True, 0.01)
    x, z = x.contiguous(), z.contiguous()
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, z, h0)]

    def once():
        out = hip_gated_scan(*leaves, starts=st)
        return (*out, *torch.autograd.grad(out, leaves, (dy, dh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.detach().clone() for t in once()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for seed in range(3):
        new = make(1, 1500, 66, torch.float32, 40 + seed, True, 0.01)
        with torch.no_grad():
            for t, n in zip((*leaves, st, dy, dh), new):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        held = [t.detach().clone() for t in got]
        fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
        out = hip_gated_scan(*fresh, starts=st)
        want = (*out, *torch.autograd.grad(out, fresh, (dy, dh)))
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_differences(gpu_lib):
    """The gate's gradient along a direction against a central difference of the
    kernel's own states: f = sum dy y over 360 values of size 1, each within 20 U; the
    third derivative's part is t^2 / 6 of a few units a value."""
    x, z, h0, st, dy, _ = make(2, 9, 20, torch.float32, 13, True, 0.2)
    zl = z.detach().clone().requires_grad_(True)
    g = torch.Generator(device=dev).manual_seed(1)
    v = torch.randn(z.shape, generator=g, device=dev)
    (gz,) = torch.autograd.grad(hip_gated_scan(x, zl, h0, st)[0], (zl,), dy)
    t = 2.0 ** -7
    f = [(hip_gated_scan(x, z + s * t * v, h0, st)[0].double() * dy.double()).sum() for s in (1, -1)]
    diff = (f[0] - f[1]) / (2 * t)
    slope = (gz.double() * v.double()).sum()
    assert abs(float(diff - slope)) <= 4 * 2 * 360 ** 0.5 * 20 * U * 4 / (2 * t) + t * t * 360


def test_refusals(gpu_lib):
    x, z, h0, _, _, _ = make(2, 5, 8, torch.float32, 14)
    st = torch.zeros(2, 5, dtype=torch.bool, device=dev)
    with pytest.raises(ValueError, match="B, L, D"):
        hip_gated_scan(x[0], z[0])
    with pytest.raises(ValueError, match="gate"):
        hip_gated_scan(x, z[:, :4])
    with pytest.raises(TypeError, match="one dtype"):
        hip_gated_scan(x, z.bfloat16())
    with pytest.raises(TypeError, match="dtype"):
        hip_gated_scan(x.double(), z.double())
    with pytest.raises(ValueError, match="h0"):
        hip_gated_scan(x, z, h0[:1])
    with pytest.raises(TypeError, match="h0"):
        hip_gated_scan(x, z, h0.half())
    with pytest.raises(ValueError, match="starts"):
        hip_gated_scan(x, z, h0, st[:, :4])
    with pytest.raises(TypeError, match="starts"):
        hip_gated_scan(x, z, h0, st.int())
    with pytest.raises(ValueError, match="starts"):
        hip_gated_scan(x, z, h0, st.cpu())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h0, torch.ones_like(h0))
        with pytest.raises((RuntimeError, NotImplementedError)):
            hip_gated_scan(x, z, dual)
