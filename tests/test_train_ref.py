"""The 64-bit restatements behind the training operators' tests, against simple
properties and differences; and the argument checks of the entry points (nothing is
launched)."""

import ctypes

import pytest
import torch

from oracle import train_ref as ref
from redpanda_amd import _lib
from redpanda_amd.checkpoint8 import Packed8, hip_checkpoint8, hip_pack8, hip_unpack8
from redpanda_amd.embedding import hip_embedding
from redpanda_amd.gated import hip_gated_scan, hip_gated_step
from redpanda_amd.norm import hip_rmsnorm

FAKE = 0x100000  # never dereferenced: validation only


@pytest.fixture(scope="module")
def lib():
    return _lib.open_library()


def test_embedding_ref_is_torchs():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(11, 5, dtype=torch.float64, generator=g, requires_grad=True)
    ids = torch.randint(0, 11, (40,), generator=g)
    dy = torch.randn(40, 5, dtype=torch.float64, generator=g)
    y = torch.nn.functional.embedding(ids, w, padding_idx=3) * 1.5
    assert torch.equal(ref.embedding(ids, w.detach(), 1.5), y.detach())
    (dw,) = torch.autograd.grad(y, (w,), dy)
    assert torch.allclose(ref.embedding(ids, w.detach(), 1.5, dy, padding_idx=3), dw, rtol=1e-13)


def test_pack8_ref():
    x = torch.zeros(1, 96)
    x[0, 0] = 127.0      # step 1: kept as it is
    x[0, 1] = 0.5        # a tie, to the even 0
    x[0, 2] = 1.5        # to 2
    x[0, 32] = 127.49    # step 1
    x[0, 64] = 127.5     # would round to 128: step 2, a tie at 63.75 is none
    q, e = ref.pack8(x)
    assert e.tolist() == [[127, 127, 128]]
    assert q[0, [0, 1, 2, 32, 64]].tolist() == [127, 0, 2, 127, 64]
    assert ref.unpack8(q, e)[0, 64] == 128
    y = torch.tensor([[float("inf")] + [1.0] * 32])
    q, e = ref.pack8(y)
    assert e.tolist() == [[255, 121]] and torch.isnan(ref.unpack8(q, e)[0, :32]).all()
    assert ref.unpack8(q, e)[0, 32] == 1.0
    q, e = ref.pack8(torch.full((1, 3), 1e-40))
    assert e.tolist() == [[1]] and q.abs().max() == 0


def test_pack8_ref_is_half_a_step_off():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 70, generator=g) * torch.exp(3 * torch.randn(9, 1, generator=g))
    q, e = ref.pack8(x)
    step = torch.pow(2.0, e.double() - 127).repeat_interleave(32, dim=1)[:, :70]
    assert bool(((ref.unpack8(q, e) - x.double()).abs() <= step / 2).all())
    # and the step is the least one that may be taken
    top = torch.nn.functional.pad(x.abs(), (0, 26)).view(9, 3, 32).amax(-1).double()
    assert bool((torch.round(top / torch.pow(2.0, e.double() - 128)) > 127).all())


def test_gradients_of_the_refs_against_differences():
    g = torch.Generator().manual_seed(3)

    def randn(*s):
        return torch.randn(*s, dtype=torch.float64, generator=g).requires_grad_(True)

    assert torch.autograd.gradcheck(lambda s, w: ref.rmsnorm(s, w, 1e-5), (randn(3, 7), randn(7)))
    starts = torch.rand(2, 6, generator=g) < 0.3
    assert torch.autograd.gradcheck(lambda x, z, h: ref.gated(x, z, h, starts),
                                    (randn(2, 6, 3), randn(2, 6, 3), randn(2, 3)))


def _emb(**kw):
    a = dict(N=4, V=10, d=8, dtype_w=0, dtype_out=0, ids64=1, scale=1.0, padding=-1, ids=FAKE,
             w=2 * FAKE, w_sr=8, out=3 * FAKE)
    a.update(kw)
    return _lib.EmbeddingArgs(**a)


@pytest.mark.parametrize("bad,word", [
    (dict(N=-1), "N < 0"), (dict(V=0), "V < 1"), (dict(d=-1), "d < 0"), (dict(N=1 << 27), "2^26"),
    (dict(V=1 << 28), "2^27"), (dict(d=1 << 23), "2^22"), (dict(dtype_w=3), "dtype"),
    (dict(dtype_out=-1), "dtype"), (dict(ids64=2), "ids64"), (dict(ids=None), "ids"),
    (dict(ids=FAKE + 4), "ids"), (dict(w=None), "w"), (dict(w_sr=7), "row stride"),
    (dict(w=2 * FAKE + 2), "misaligned"), (dict(out=None), "out"), (dict(out=2 * FAKE + 64), "overlaps"),
    (dict(out=FAKE + 8), "overlaps")])
def test_embedding_refusals(lib, bad, word):
    assert lib.rp_embedding_fwd(ctypes.byref(_emb(**bad)), None) < 0
    assert word in lib.rp_last_error().decode()


def test_embedding_grad_refusals(lib):
    a = _emb()
    need = lib.rp_embedding_work_bytes(ctypes.byref(a))
    assert need > 0

    def grad(**kw):
        g = dict(dout=4 * FAKE, dout_sr=8, dw=5 * FAKE, work=6 * FAKE, work_bytes=need)
        g.update(kw)
        return lib.rp_embedding_bwd(ctypes.byref(a), ctypes.byref(_lib.EmbeddingGrad(**g)), None)

    for bad, word in ((dict(dout=None), "dout"), (dict(dout_sr=7), "row stride"), (dict(dw=None), "dw"),
                      (dict(work=None), "workspace"), (dict(work=6 * FAKE + 16), "workspace"),
                      (dict(work_bytes=need - 1), "workspace"), (dict(dw=4 * FAKE), "overlaps"),
                      (dict(dw=6 * FAKE), "overlap")):
        assert grad(**bad) < 0 and word in lib.rp_last_error().decode(), (bad, word)
    assert lib.rp_embedding_bwd(ctypes.byref(a), None, None) < 0
    assert lib.rp_embedding_fwd(None, None) < 0


def _pack(**kw):
    a = dict(rows=4, d=40, dtype=0, x=FAKE, x_sr=40, q=2 * FAKE, e=3 * FAKE)
    a.update(kw)
    return _lib.PackArgs(**a)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "negative"), (dict(x_sr=39), "stride"), (dict(dtype=4), "dtype"),
    (dict(x=None), "NULL"), (dict(q=None), "NULL"), (dict(e=None), "NULL"), (dict(x=FAKE + 1), "misaligned"),
    (dict(q=FAKE + 8), "overlap"), (dict(e=2 * FAKE + 159), "overlap")])
def test_pack_refusals(lib, bad, word):
    for fn in (lib.rp_pack, lib.rp_unpack):
        assert fn(ctypes.byref(_pack(**bad)), None) < 0
        assert word in lib.rp_last_error().decode()


def test_unpack_wants_contiguous_rows(lib):
    assert lib.rp_unpack(ctypes.byref(_pack(x_sr=48)), None) < 0
    assert "contiguous" in lib.rp_last_error().decode()
    assert lib.rp_pack(None, None) < 0


def _an(**kw):
    a = dict(rows=4, d=40, dtype_x=0, dtype_add=0, dtype_sum=0, dtype_out=0, x=FAKE, x_sr=40,
             add=2 * FAKE, add_sr=40, w=3 * FAKE, sum=4 * FAKE, out=5 * FAKE, q=6 * FAKE, e=7 * FAKE,
             eps=1e-5)
    a.update(kw)
    return _lib.AddNormArgs(**a)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "negative"), (dict(d=0, x_sr=0), "mean"), (dict(x_sr=39), "stride"),
    (dict(dtype_x=3), "dtype"), (dict(dtype_sum=9), "dtype"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q=None), "together"), (dict(e=None), "together"),
    (dict(w=3 * FAKE + 2), "misaligned"), (dict(x=None, q=None, e=None), "neither"),
    (dict(x=FAKE + 2), "misaligned"), (dict(sum=None), "together"), (dict(add=None), "together"),
    (dict(add=None, sum=None, dtype_sum=1), "type"), (dict(add_sr=8), "stride"),
    (dict(x=None), "no add"), (dict(x=None, add=None, sum=None, out=None), "NULL out"),
    (dict(out=FAKE + 16), "overlaps"), (dict(sum=2 * FAKE), "overlaps"), (dict(q=5 * FAKE), "overlap"),
    (dict(e=4 * FAKE), "overlap"), (dict(out=3 * FAKE), "overlaps")])
def test_addnorm_refusals(lib, bad, word):
    assert lib.rp_addnorm_fwd(ctypes.byref(_an(**bad)), None) < 0
    assert word in lib.rp_last_error().decode()


def test_addnorm_grad_refusals(lib):
    a = _an()
    need = lib.rp_addnorm_work_bytes(ctypes.byref(a))
    assert need > 0

    def grad(args=a, **kw):
        g = dict(dout=8 * FAKE, dout_sr=40, dsum=9 * FAKE, dsum_sr=40, dx=10 * FAKE, dadd=11 * FAKE,
                 dw=12 * FAKE, work=13 * FAKE, work_bytes=need)
        g.update(kw)
        return lib.rp_addnorm_bwd(ctypes.byref(args), ctypes.byref(_lib.AddNormGrad(**g)), None)

    for bad, word in ((dict(dout=None), "dout"), (dict(dout_sr=39), "stride"), (dict(dsum_sr=39), "stride"),
                      (dict(dx=10 * FAKE + 2), "misaligned"), (dict(dw=12 * FAKE + 1), "misaligned"),
                      (dict(work=None), "workspace"), (dict(work_bytes=need - 256), "workspace"),
                      (dict(dx=8 * FAKE), "overlaps"), (dict(dadd=FAKE), "overlaps"),
                      (dict(dw=10 * FAKE), "overlap"), (dict(dx=13 * FAKE), "overlap")):
        assert grad(**bad) < 0 and word in lib.rp_last_error().decode(), (bad, word)
    # rows beyond the register shapes need their scratch whatever is asked for
    wide = _an(d=20000, x_sr=20000)
    assert grad(wide, dout_sr=20000, dsum_sr=20000, dw=None, work=None) < 0
    assert "workspace" in lib.rp_last_error().decode()


def _gated(**kw):
    a = dict(B=2, L=6, D=40, dtype=0, x=FAKE, x_sb=240, x_sl=40, gate=2 * FAKE, gate_sb=240, gate_sl=40,
             h0=3 * FAKE, starts=4 * FAKE, starts_sb=6, y=5 * FAKE, h_last=6 * FAKE, ckpt=7 * FAKE)
    a.update(kw)
    return _lib.GatedArgs(**a)


@pytest.mark.parametrize("bad,word", [
    (dict(B=-1), "negative"), (dict(L=1 << 31), "int32"), (dict(B=1 << 25, D=65), "too many"),
    (dict(dtype=5), "dtype"), (dict(x=None), "NULL"), (dict(gate=None), "NULL"), (dict(x=FAKE + 2), "misaligned"),
    (dict(x_sl=39), "stride"), (dict(gate_sb=-1), "stride"), (dict(h0=3 * FAKE + 1), "misaligned"),
    (dict(starts_sb=-2), "starts"), (dict(y=None), "y"), (dict(y=FAKE), "overlaps"),
    (dict(h_last=3 * FAKE), "overlaps"), (dict(ckpt=5 * FAKE), "overlap")])
def test_gated_refusals(lib, bad, word):
    assert lib.rp_gated_fwd(ctypes.byref(_gated(**bad)), None) < 0
    assert word in lib.rp_last_error().decode()


def test_gated_grad_refusals(lib):
    def grad(args=None, **kw):
        g = dict(dy=8 * FAKE, dy_sb=240, dy_sl=40, dh_last=9 * FAKE, dx=10 * FAKE, dgate=11 * FAKE,
                 dh0=12 * FAKE)
        g.update(kw)
        return lib.rp_gated_bwd(ctypes.byref(args or _gated()), ctypes.byref(_lib.GatedGrad(**g)), None)

    for bad, word in ((dict(dx=None), "NULL"), (dict(dgate=None), "NULL"), (dict(dy_sl=3), "stride"),
                      (dict(dy=8 * FAKE + 1), "misaligned"), (dict(dx=FAKE), "overlaps"),
                      (dict(dgate=10 * FAKE), "overlap"), (dict(dh0=7 * FAKE), "overlaps")):
        assert grad(**bad) < 0 and word in lib.rp_last_error().decode(), (bad, word)
    assert grad(_gated(ckpt=None)) < 0 and "ckpt" in lib.rp_last_error().decode()
    # few channels of a long sequence are split along it, which takes a workspace
    long = _gated(B=1, L=4096, starts=None, x_sb=0, gate_sb=0)
    assert lib.rp_gated_work_bytes(ctypes.byref(long)) > 0
    assert lib.rp_gated_fwd(ctypes.byref(long), None) < 0
    assert "workspace" in lib.rp_last_error().decode()


def test_nothing_to_do_is_fine(lib):
    assert lib.rp_embedding_fwd(ctypes.byref(_emb(N=0, ids=None, w=None, out=None)), None) == 0
    assert lib.rp_pack(ctypes.byref(_pack(rows=0, x=None)), None) == 0
    assert lib.rp_addnorm_fwd(ctypes.byref(_an(rows=0, x=None, q=None, e=None)), None) == 0
    assert lib.rp_gated_fwd(ctypes.byref(_gated(L=0, x=None)), None) == 0
    assert lib.rp_gated_work_bytes(ctypes.byref(_gated(B=0))) == 0


@pytest.mark.parametrize("cname,pyname", [
    ("rp_embedding_args", "EmbeddingArgs"), ("rp_embedding_grad", "EmbeddingGrad"),
    ("rp_pack_args", "PackArgs"), ("rp_addnorm_args", "AddNormArgs"), ("rp_addnorm_grad", "AddNormGrad"),
    ("rp_gated_args", "GatedArgs"), ("rp_gated_grad", "GatedGrad")])
def test_structs_mirror_the_header(cname, pyname):
    from tests.test_capi import _header_struct_fields
    assert [f[0] for f in getattr(_lib, pyname)._fields_] == _header_struct_fields(cname)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="device"):
        hip_embedding(torch.zeros(3, dtype=torch.int64), x)
    with pytest.raises(RuntimeError, match="device"):
        hip_rmsnorm(x)
    with pytest.raises(RuntimeError, match="device"):
        hip_pack8(x)
    with pytest.raises(RuntimeError, match="device"):
        hip_unpack8(Packed8(x.to(torch.int8), torch.zeros(2, 1, dtype=torch.uint8), torch.float32))
    with pytest.raises(RuntimeError, match="device"):
        hip_checkpoint8(lambda t: t, x)
    with pytest.raises(RuntimeError, match="device"):
        hip_gated_scan(x[None], x[None])
    with pytest.raises(ValueError, match="R, D"):
        hip_gated_step(x[None], x[None])
