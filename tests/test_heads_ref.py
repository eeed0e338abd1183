"""The 64-bit restatements behind the head operators' tests, against published
values and simple properties; and the argument checks of the C entry points
(nothing is launched)."""

import ctypes

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import heads_ref as ref
from redpanda_amd import _lib
from redpanda_amd.dropout import hip_dropout
from redpanda_amd.layernorm import hip_layernorm
from redpanda_amd.sampling import hip_sample

FAKE = 0x10000  # never dereferenced: validation only


@pytest.fixture(scope="module")
def lib():
    return _lib.open_library()


# The known answers that the generator's authors publish with it.
@pytest.mark.parametrize("counter,key,out", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, out):
    got = ref.philox4x32([np.array([c]) for c in counter], key)
    assert [int(g[0]) for g in got] == list(out)


def test_mask_share_and_independence():
    a = ref.keep_mask(range(400), 500, 0.25, 11)
    b = ref.keep_mask(range(400), 500, 0.25, 11, stream=1)
    n = a.numel()
    # five standard deviations of a share and of a correlation
    assert abs(a.double().mean() - 0.75) < 5 * (0.75 * 0.25 / n) ** 0.5
    assert abs((a ^ b).double().mean() - 2 * 0.75 * 0.25) < 5 * 0.5 / n ** 0.5
    assert torch.equal(a, ref.keep_mask(range(400), 500, 0.25, 11))


def test_layernorm_and_gelu_are_torchs():
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, dtype=torch.float64, generator=g) for s in ((7, 33), (33,), (33,)))
    y = ref.layernorm(x, w, b, 1e-5, use_gelu=True)
    assert torch.allclose(y, F.layer_norm(F.gelu(x), (33,), w, b, 1e-5), rtol=1e-12, atol=1e-12)


def test_sample_row_cuts():
    v = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [ref.sample_row(v, u)[0] for u in (0.0, 0.0999, 0.1001, 0.4999, 0.5001, 0.701, 0.999)] == \
        [0, 0, 1, 1, 2, 3, 3]
    assert {ref.sample_row(v, u, k=2)[0] for u in np.linspace(0, 0.999, 50)} == {1, 3}
    assert {ref.sample_row(v, u, tp=0.75)[0] for u in np.linspace(0, 0.999, 50)} == {1, 2, 3}
    assert {ref.sample_row(v, u, mp=0.6)[0] for u in np.linspace(0, 0.999, 50)} == {1, 3}
    assert ref.sample_row(v, 0.9, T=0.0) == (1, 0.0)
    assert ref.sample_row([-np.inf, np.nan], 0.5) == (-1, -np.inf)
    assert ref.sample_row([1.0, 1.0, 1.0], 0.99, k=2)[0] == 1  # equal values: the first ones


def _dropout(**kw):
    a = _lib.DropoutArgs(rows=4, d=64, dtype_x=1, dtype_res=0, dtype_out=0, p=0.1, x=FAKE, x_sr=64,
                         res=FAKE + 0x10000, res_sr=64, out=FAKE + 0x20000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _norm(**kw):
    a = _lib.LayerNormArgs(rows=4, d=64, dtype_x=1, dtype_out=0, gelu=1, p=0.1, x=FAKE, x_sr=64,
                           out=FAKE + 0x20000, stats=FAKE + 0x30000, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _sample(**kw):
    a = _lib.SampleArgs(R=4, V=64, M=0, dtype_logits=1, logits=FAKE, logits_sr=64, u=FAKE + 0x10000,
                        temperature=1.0, top_p=0.9, min_p=0.0, ids=FAKE + 0x20000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,needle", [
    (dict(rows=-1), "negative"), (dict(d=1 << 31), "int32"), (dict(x_sr=63), "stride"),
    (dict(dtype_x=3), "dtype"), (dict(dtype_out=-1), "dtype"), (dict(dtype_res=9), "dtype"),
    (dict(p=1.5), "p must"), (dict(p=float("nan")), "p must"), (dict(x=None), "NULL"),
    (dict(out=None), "NULL"), (dict(x=FAKE + 1), "misaligned"), (dict(seed_ptr=FAKE + 4), "seed"),
    (dict(out=FAKE + 8), "overlaps x"), (dict(out=FAKE + 0x10008), "overlaps res"),
    (dict(res_sr=10), "res row stride"), (dict(rows=1 << 40, x_sr=1 << 40), "too many"),
])
def test_dropout_refusals(lib, kw, needle):
    assert lib.rp_dropout_check(ctypes.byref(_dropout())) == 0
    assert lib.rp_dropout_check(ctypes.byref(_dropout(**kw))) < 0
    assert needle in lib.rp_last_error().decode()
    assert lib.rp_dropout(ctypes.byref(_dropout(**kw)), None) < 0


@pytest.mark.parametrize("kw,needle", [
    (dict(rows=-1), "negative"), (dict(d=0), "no elements"), (dict(x_sr=63), "stride"),
    (dict(dtype_x=3), "dtype"), (dict(dtype_out=5), "dtype"), (dict(gelu=2), "gelu"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(p=-0.1), "p must"),
    (dict(x=None), "NULL"), (dict(x=FAKE + 1), "misaligned"), (dict(w=FAKE + 2), "misaligned"),
])
def test_layernorm_refusals(lib, kw, needle):
    assert lib.rp_layernorm_check(ctypes.byref(_norm())) == 0
    assert lib.rp_layernorm_check(ctypes.byref(_norm(**kw))) < 0
    assert needle in lib.rp_last_error().decode()
    assert lib.rp_layernorm_fwd(ctypes.byref(_norm(**kw)), None) < 0
    assert lib.rp_layernorm_work_bytes(ctypes.byref(_norm(**kw))) < 0


@pytest.mark.parametrize("kw,needle", [
    (dict(out=None), "out"), (dict(out=FAKE + 0x20002), "out"), (dict(out=FAKE + 16), "overlaps"),
    (dict(stats=FAKE + 0x20000), "overlaps"), (dict(w=FAKE + 0x20000), "overlaps"),
])
def test_layernorm_output_refusals(lib, kw, needle):
    assert lib.rp_layernorm_fwd(ctypes.byref(_norm(**kw)), None) < 0
    assert needle in lib.rp_last_error().decode()


@pytest.mark.parametrize("akw,kw,needle", [
    ({}, dict(dout=None), "dout"), ({}, dict(dout_sr=63), "dout"), ({}, dict(dw=None), "together"),
    (dict(stats=None), {}, "stats"), ({}, dict(dx=FAKE + 16), "overlaps"),
    ({}, dict(dw=FAKE + 0x50000), "outputs overlap"), ({}, dict(work=None), "workspace"),
    ({}, dict(work_bytes=16), "workspace"), ({}, dict(work=FAKE + 0x80004), "workspace"),
])
def test_layernorm_grad_refusals(lib, akw, kw, needle):
    a = _norm(**akw)
    g = _lib.LayerNormGrad(FAKE + 0x40000, 64, FAKE + 0x50000, FAKE + 0x60000, FAKE + 0x70000,
                           FAKE + 0x80000, 1 << 20)
    for k, v in kw.items():
        setattr(g, k, v)
    assert lib.rp_layernorm_bwd(ctypes.byref(a), ctypes.byref(g), None) < 0
    assert needle in lib.rp_last_error().decode()
    assert lib.rp_layernorm_bwd(ctypes.byref(a), None, None) < 0


@pytest.mark.parametrize("kw,needle", [
    (dict(R=-1), "R < 0"), (dict(V=0), "V < 1"), (dict(V=(1 << 30) + 1), "2^30"),
    (dict(dtype_logits=4), "dtype"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(top_p=-0.5), "top_p"),
    (dict(min_p=1.5), "min_p"), (dict(logits=None), "NULL"), (dict(u=None), "NULL"),
    (dict(ids=None), "NULL"), (dict(logits_sr=63), "stride"), (dict(ids=FAKE + 0x20004), "misaligned"),
    (dict(logits=FAKE + 1), "misaligned"), (dict(tokens=FAKE + 0x30000, M=8, tokens_sr=7), "stride"),
    (dict(ids=FAKE + 8), "overlaps"), (dict(logp=FAKE + 0x20010), "overlap"),
    (dict(top_k_row=FAKE + 2), "misaligned"),
])
def test_sample_refusals(lib, kw, needle):
    assert lib.rp_sample_check(ctypes.byref(_sample())) == 0
    assert lib.rp_sample_check(ctypes.byref(_sample(**kw))) < 0
    assert needle in lib.rp_last_error().decode()
    assert lib.rp_sample(ctypes.byref(_sample(**kw)), None) < 0


def test_empty_calls_launch_nothing(lib):
    assert lib.rp_dropout(ctypes.byref(_dropout(rows=0)), None) == 0
    assert lib.rp_dropout(ctypes.byref(_dropout(d=0, x_sr=0, res_sr=0)), None) == 0
    assert lib.rp_layernorm_fwd(ctypes.byref(_norm(rows=0, x=None, out=None)), None) == 0
    assert lib.rp_sample(ctypes.byref(_sample(R=0)), None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="ROCm"):
        hip_dropout(x, 0.1, 0)
    with pytest.raises(RuntimeError, match="ROCm"):
        hip_layernorm(x)
    with pytest.raises(ValueError, match="device tensor"):
        hip_sample(x, torch.zeros(2))


def test_sample_workspace(lib):
    """Few long rows have one, which may be left out; a short or unaligned one is
    refused."""
    assert lib.rp_sample_work_bytes(ctypes.byref(_sample())) == 0
    a = _sample(V=100003, logits_sr=100003, ids=FAKE + 0x1000000, u=FAKE + 0x2000000)
    need = lib.rp_sample_work_bytes(ctypes.byref(a))
    assert need > 0 and need % 256 == 0
    for work, nbytes in ((FAKE * 0x1000, need - 1), (FAKE * 0x1000 + 8, need)):
        a.work, a.work_bytes = work, nbytes
        assert lib.rp_sample(ctypes.byref(a), None) < 0
        assert "workspace" in lib.rp_last_error().decode()
    assert lib.rp_sample_work_bytes(ctypes.byref(_sample(R=-1))) < 0
