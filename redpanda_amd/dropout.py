"""Dropout on the HIP kernel, with a mask that is never stored.

The mask comes from a counter-based generator (Philox4x32-10, see
include/redpanda_hip.h), so the backward pass draws it again from the seed: no
tensor is kept for it.  A residual is added in the same pass, as the
pre-norm layers' x + dropout(branch) needs it.
"""

import ctypes

import torch
from torch.autograd.function import once_differentiable

from redpanda_amd import _lib


def dtype_code(dtype, what):
    try:
        return _lib.DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"redpanda_amd {what}: unsupported dtype {dtype}") from None


def rows_of(t, d):
    """(rows, d) view of t with unit inner stride and rows that do not overlap,
    or a contiguous copy of it."""
    if not t.is_contiguous():
        if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < d:
            t = t.contiguous()
    return t if t.dim() == 2 else t.view(-1, d)


def row_stride(t):
    """A row view's stride (of a single row, which may carry any, its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def check_p(p, what):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be in [0, 1], got {p}")
    return p


def seed_arg(seed, device, what):
    """(value, tensor or None) of a seed: an int, or an int64 tensor of one
    element on the device, which the kernels read when they run."""
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"{what}: a seed tensor must be one int64 on {device}, got "
                             f"{tuple(seed.shape)} {seed.dtype} on {seed.device}")
        return 0, seed
    if seed is None:
        raise ValueError(f"{what}: dropout needs a seed (an int or an int64 tensor)")
    return int(seed) & 0xFFFFFFFFFFFFFFFF, None


def _run(x, res, p, seed, seed_t, stream, out_dtype):
    lib = _lib.load()
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    if out.numel() == 0:
        return out
    d = x.shape[-1]
    xr = rows_of(x, d)
    a = _lib.DropoutArgs(xr.shape[0], d, _lib.DTYPE_CODES[x.dtype], 0, _lib.DTYPE_CODES[out_dtype],
                         stream, p, seed, _lib.ptr(seed_t), xr.data_ptr(), row_stride(xr), None, 0,
                         out.data_ptr())
    if res is not None:
        rr = rows_of(res, d)
        a.dtype_res, a.res, a.res_sr = _lib.DTYPE_CODES[res.dtype], rr.data_ptr(), row_stride(rr)
    _lib.check(lib.rp_dropout(ctypes.byref(a), _lib.stream_of(x.device)), lib)
    return out


class _HipDropout(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, res, p, seed, seed_t, stream, out_dtype):
        ctx.args = (p, seed, stream)
        ctx.dtypes = (x.dtype, None if res is None else res.dtype)
        if seed_t is not None:
            ctx.save_for_backward(seed_t)
        return _run(x, res, p, seed, seed_t, stream, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, stream = ctx.args
        seed_t = ctx.saved_tensors[0] if ctx.saved_tensors else None
        dx = dres = None
        if ctx.needs_input_grad[0]:
            dx = _run(dy, None, p, seed, seed_t, stream, ctx.dtypes[0])
        if ctx.needs_input_grad[1]:
            dres = dy.to(ctx.dtypes[1])
        return dx, dres, None, None, None, None, None


def hip_dropout(x, p, seed, residual=None, stream=0):
    """[residual +] dropout(x, p): kept elements scaled by the inverse of the
    share that is kept, (round(65536 p) of 65536 are dropped).

    x: (..., d) fp32 / bf16 / fp16 on the device; residual: None or a tensor of
    x's shape, any of these dtypes.  The result has x's dtype, or with a
    residual the one torch promotes the two to; the sum is rounded once.  seed:
    an int, or an int64 tensor of one element on x's device, read when the
    kernel runs (a captured graph draws anew when it changes between replays;
    between a forward and its backward it must not change, which autograd
    checks).  The mask depends on the seed, `stream` (give each place of a model
    that drops its own, 0 .. 2^32 - 1), the row and the column only.
    Differentiable in x and residual."""
    if not x.is_cuda:
        raise RuntimeError("redpanda_amd dropout: inputs must be ROCm device tensors")
    if x.dim() == 0:
        raise ValueError("dropout: x must have at least one dimension")
    dtype_code(x.dtype, "dropout")
    out_dtype = x.dtype
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"dropout: residual {tuple(residual.shape)} on {residual.device} must be "
                             f"{tuple(x.shape)} on {x.device}")
        dtype_code(residual.dtype, "dropout")
        out_dtype = torch.promote_types(x.dtype, residual.dtype)
    p = check_p(p, "dropout")
    if not 0 <= stream < 1 << 32:
        raise ValueError(f"dropout: stream must be in [0, 2^32), got {stream}")
    seed, seed_t = seed_arg(seed, x.device, "dropout")
    if torch.is_grad_enabled() and (x.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _HipDropout.apply(x, residual, p, seed, seed_t, stream, out_dtype)
    return _run(x, residual, p, seed, seed_t, stream, out_dtype)
