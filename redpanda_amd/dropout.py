"""Dropout on the HIP kernel, with a mask that is never stored.

The mask comes from a counter-based generator (Philox4x32-10, see
include/redpanda_hip.h), so the backward pass draws it again from the seed: no
tensor is kept for it.  A residual is added in the same pass, as the
pre-norm layers' x + dropout(branch) needs it.
"""

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from redpanda_amd import _lib


def dtype_code(dtype, what):
    try:
        return _lib.DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"redpanda_amd {what}: unsupported dtype {dtype}") from None


def rows_of(t, d):
    """t as rows of d elements with unit inner stride that do not overlap: (t or a
    contiguous copy of it, the number of rows, their stride)."""
    if t.is_contiguous():
        return t, t.numel() // d, d
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= d:
        return t, t.shape[0], t.stride(0)
    return t.contiguous(), t.numel() // d, d


def empty_rows(t, dtype):
    """A contiguous tensor of t's shape."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def check_p(p, what):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be in [0, 1], got {p}")
    return p


def seed_arg(seed, device, what):
    """(value, tensor or None) of a seed: an int, or an int64 tensor of one
    element on the device, which the kernels read when they run."""
    if isinstance(seed, torch.Tensor):
        if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"{what}: a seed tensor must be one int64 on {device}, got "
                             f"{tuple(seed.shape)} {seed.dtype} on {seed.device}")
        return 0, seed
    if seed is None:
        raise ValueError(f"{what}: dropout needs a seed (an int or an int64 tensor)")
    return int(seed) & 0xFFFFFFFFFFFFFFFF, None


def _run(x, res, p, seed, seed_t, stream, out_dtype):
    lib = _lib.load()
    out = empty_rows(x, out_dtype)
    if out.numel() == 0:
        return out
    d = x.shape[-1]
    x, rows, sr = rows_of(x, d)
    a = _lib.DropoutArgs(rows, d, _lib.DTYPE_CODES[x.dtype], 0, _lib.DTYPE_CODES[out_dtype], stream, p,
                         seed, None if seed_t is None else seed_t.data_ptr(), x.data_ptr(), sr, None,
                         0, out.data_ptr())
    if res is not None:
        res, _, rsr = rows_of(res, d)
        a.dtype_res, a.res, a.res_sr = _lib.DTYPE_CODES[res.dtype], res.data_ptr(), rsr
    _lib.check(lib.rp_dropout(ctypes.byref(a), _lib.stream_of(out.device)), lib)
    return out


def recorded(grad):
    """Whether a call goes through its autograd Function: where an input requires a
    gradient, and within a forward-mode level, whose tangents (they do not show in
    requires_grad) the Function refuses and the plain call would lose."""
    return (grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0


def once(backward):
    """A backward that may not be differentiated again: once_differentiable's
    marks where a graph of it is being recorded, and the function itself (5 us
    less of a small call) where not."""
    marked = once_differentiable(backward)

    def run(ctx, *grads):
        return marked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


class _HipDropout(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, res, p, seed, seed_t, stream, out_dtype):
        ctx.args = (p, seed, stream, x.dtype, None if res is None else res.dtype)
        ctx.save_for_backward(seed_t)
        return _run(x, res, p, seed, seed_t, stream, out_dtype)

    @staticmethod
    @once
    def backward(ctx, dy):
        p, seed, stream, x_dtype, res_dtype = ctx.args
        (seed_t,) = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = _run(dy, None, p, seed, seed_t, stream, x_dtype) if need[0] else None
        dres = dy.to(res_dtype) if need[1] else None
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
    Differentiable in x and residual, once and in reverse mode (a tangent is
    refused)."""
    if not x.is_cuda:
        raise RuntimeError("redpanda_amd dropout: inputs must be ROCm device tensors")
    if x.dim() == 0:
        raise ValueError("dropout: x must have at least one dimension")
    out_dtype = x.dtype
    dtype_code(out_dtype, "dropout")
    grad = x.requires_grad
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"dropout: residual {tuple(residual.shape)} on {residual.device} must be "
                             f"{tuple(x.shape)} on {x.device}")
        dtype_code(residual.dtype, "dropout")
        out_dtype = torch.promote_types(out_dtype, residual.dtype)
        grad = grad or residual.requires_grad
    p = check_p(p, "dropout")
    if not 0 <= stream < 1 << 32:
        raise ValueError(f"dropout: stream must be in [0, 2^32), got {stream}")
    seed, seed_t = seed_arg(seed, x.device, "dropout")
    if recorded(grad):
        return _HipDropout.apply(x, residual, p, seed, seed_t, stream, out_dtype)
    return _run(x, residual, p, seed, seed_t, stream, out_dtype)
