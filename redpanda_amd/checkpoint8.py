"""Activation checkpoints in 8 bits on the HIP kernels.

hip_pack8 / hip_unpack8 put a tensor into 8 bits and back: 32 columns share a power
of two, so that a value is off by half of a 127th to a 64th of the largest among its
32.  hip_checkpoint8 runs a pre-norm layer's branch and keeps of it, until the
backward, only the layer's input in 8 bits: 33 bytes for 32 values, where a
checkpoint of the stream takes 128 in fp32.
"""

import ctypes

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import dtype_code, once, recorded, rows_of
from redpanda_amd.norm import (check_norm, norm_again, norm_backward, norm_forward, pack_buffers)


class Packed8:
    """A tensor in 8 bits: q (int8, its shape), e (uint8, an exponent for each 32
    columns) and the dtype it had.  Its values are q * 2^(e - 127), cut to the dtype's
    finite range; NaN where e is 255."""

    __slots__ = ("q", "e", "dtype")

    def __init__(self, q, e, dtype):
        self.q, self.e, self.dtype = q, e, dtype

    @property
    def shape(self):
        return self.q.shape


def hip_pack8(x):
    """x (..., d) fp32 / bf16 / fp16 on the device in 8 bits, as a Packed8.

    Each 32 columns of a row (the last ones what is left) share the least power of two
    (2^-126 or more) that takes the largest of them to at most 127; values are rounded to
    nearest, ties to even.  Finite values come back finite (those nearest to the end of
    x's type as its largest value); 32 columns with an infinity or a NaN come back as NaN.
    Not differentiable."""
    if not x.is_cuda:
        raise RuntimeError("redpanda_amd pack8: inputs must be ROCm device tensors")
    if x.dim() == 0:
        raise ValueError("pack8: x must have at least one dimension")
    code = dtype_code(x.dtype, "pack8")
    d = x.shape[-1]
    q, e = pack_buffers(x)
    if q.numel() > 0:
        xr, rows, sr = rows_of(x, d)
        a = _lib.PackArgs(rows, d, code, code, xr.data_ptr(), sr, q.data_ptr(), e.data_ptr())
        _lib.call(_lib.load().rp_pack, x.device, ctypes.byref(a))
    return Packed8(q, e, x.dtype)


def hip_unpack8(packed, dtype=None):
    """The tensor that a Packed8 holds, in its own dtype or rounded to another."""
    q, e = packed.q, packed.e
    if not q.is_cuda:
        raise RuntimeError("redpanda_amd unpack8: inputs must be ROCm device tensors")
    dtype = packed.dtype if dtype is None else dtype
    code, held = dtype_code(dtype, "unpack8"), dtype_code(packed.dtype, "unpack8")
    d = q.shape[-1]
    if (q.dtype is not torch.int8 or e.dtype is not torch.uint8 or e.device != q.device or
            e.shape != (*q.shape[:-1], (d + 31) // 32)):
        raise ValueError(f"unpack8: q {tuple(q.shape)} {q.dtype} on {q.device} and e {tuple(e.shape)} "
                         f"{e.dtype} on {e.device} are not a tensor's 8 bits")
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel() > 0:
        q, e = q.contiguous(), e.contiguous()
        a = _lib.PackArgs(out.numel() // d, d, code, held, out.data_ptr(), d, q.data_ptr(), e.data_ptr())
        _lib.call(_lib.load().rp_unpack, out.device, ctypes.byref(a))
    return out


def _versions(params):
    return [None if p.is_inference() else p._version for p in params]


def _one_tensor(out):
    if not isinstance(out, torch.Tensor):
        raise TypeError(f"redpanda_amd checkpoint8: fn must give one tensor, got {type(out).__name__}")


class _HipCheckpoint8(torch.autograd.Function):

    @staticmethod
    def forward(ctx, fn, x, add, w, eps, out_dtype, *params):
        total, normed, kept, wc, a = norm_forward(x, add, w, eps, out_dtype, True)
        try:
            out = fn(normed)
        finally:
            # (a weight cast here, where nothing is recorded, must not be found in
            # autocast's cache by a later use that is; fn may turn the cache on itself, so
            # that it is emptied, not kept off)
            if torch.is_autocast_enabled("cuda"):
                torch.clear_autocast_cache()
        _one_tensor(out)
        ctx.save_for_backward(wc, *kept)
        # (not saved: their gradients are asked for by identity, and hooks on saved tensors,
        # such as another checkpoint's around this one, give others back)
        ctx.params, ctx.versions = params, _versions(params)
        ctx.fn, ctx.args, ctx.out_dtype = fn, a, out_dtype
        ctx.dtypes = (x.dtype, None if add is None else add.dtype, None if w is None else w.dtype)
        ctx.autocast = (torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda"),
                        torch.is_autocast_cache_enabled())
        ctx.set_materialize_grads(False)
        return out if add is None else (total, out)

    @staticmethod
    @once
    def backward(ctx, *grads):
        dsum, dout = grads if len(grads) == 2 else (None, grads[0])
        w, q, e = ctx.saved_tensors
        if _versions(ctx.params) != ctx.versions:
            raise RuntimeError("redpanda_amd checkpoint8: one of the params has been modified by an "
                               "inplace operation since the forward")
        need = ctx.needs_input_grad
        wanted = [p for p, n in zip(ctx.params, need[6:]) if n]
        got = [None] * len(wanted)
        dnorm = None
        if dout is not None:
            normed = norm_again((q, e), w, ctx.args, ctx.out_dtype).requires_grad_(True)
            on, dtype, cache = ctx.autocast
            with torch.enable_grad(), torch.autocast("cuda", dtype=dtype, enabled=on,
                                                     cache_enabled=cache):
                out = ctx.fn(normed)
            if out.requires_grad:  # (fn may detach)
                dnorm, *got = torch.autograd.grad(out, (normed, *wanted), dout, allow_unused=True)
        dx, dadd, dw = norm_backward(None, (q, e), w, ctx.args, ctx.dtypes, dsum, dnorm, need[1:4])
        it = iter(got)
        return (None, dx, dadd, dw, None, None, *(next(it) if n else None for n in need[6:]))


def hip_checkpoint8(fn, x, weight=None, eps=1e-5, add=None, out_dtype=None, params=()):
    """fn(RMSNorm(x) * weight), or with add (x + add, fn(RMSNorm(x + add) * weight)), of
    which only x + add in 8 bits is kept until the backward.

    x, add, weight, eps, out_dtype: as in hip_rmsnorm.  fn: a function of the normed rows
    that gives one tensor; it runs again in the backward, on the norm of the values that
    8 bits hold, and must then do the same (no random numbers but from seeds of its own);
    its argument may not be changed in place.
    params: the tensors it reads whose gradients are wanted, as a module's
    parameters().  The results are those of the plain layer; its gradients are the exact
    ones at the kept values.  Differentiable once and in reverse mode."""
    eps, out_dtype, grad = check_norm(x, weight, eps, add, out_dtype, "checkpoint8")
    params = tuple(dict.fromkeys(params))  # (one given twice has its gradient once)
    if recorded(grad or any(p.requires_grad for p in params)):
        return _HipCheckpoint8.apply(fn, x, add, weight, eps, out_dtype, *params)
    total, normed, _, _, _ = norm_forward(x, add, weight, eps, out_dtype, False)
    out = fn(normed)
    _one_tensor(out)
    return out if add is None else (total, out)
