"""Layer norm on the HIP kernels, with GELU before it and dropout behind it.

The middle of a search model's head (engine/search_mamba.py:52-72: Linear, GELU,
LayerNorm, Linear) in one pass over its rows, forward and backward: GELU's value
and slope are formed again from the input in the backward, the dropout's mask is
drawn again from its seed, and of the rows only the mean and the inverse of the
standard deviation are kept.
"""

import ctypes

import torch
from torch.autograd.function import once_differentiable

from redpanda_amd import _lib
from redpanda_amd.dropout import check_p, dtype_code, row_stride, rows_of, seed_arg


def _f32c(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def _args(xr, w, b, eps, gelu, p, seed, seed_t, stream, out_code, out, stats):
    return _lib.LayerNormArgs(xr.shape[0], xr.shape[1], _lib.DTYPE_CODES[xr.dtype], out_code, gelu,
                              stream, p, seed, _lib.ptr(seed_t), xr.data_ptr(), row_stride(xr),
                              _lib.ptr(w), _lib.ptr(b), _lib.ptr(out), _lib.ptr(stats), eps, 0)


def _forward(x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype, keep):
    """(out, x as rows, w in fp32, the rows' stats or None)."""
    lib = _lib.load()
    xr = rows_of(x, x.shape[-1])
    wc = _f32c(w)
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    stats = torch.empty((xr.shape[0], 2), dtype=torch.float32, device=x.device) if keep else None
    a = _args(xr, wc, _f32c(b), eps, gelu, p, seed, seed_t, stream, _lib.DTYPE_CODES[out_dtype],
              out, stats)
    _lib.check(lib.rp_layernorm_fwd(ctypes.byref(a), _lib.stream_of(x.device)), lib)
    return out, xr, wc, stats


class _HipLayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype):
        out, xr, wc, stats = _forward(x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype, True)
        ctx.save_for_backward(x, wc, stats, seed_t)
        ctx.args = (eps, gelu, p, seed, stream)
        ctx.out_dtype = out_dtype
        ctx.wdtypes = (None if w is None else w.dtype, None if b is None else b.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        lib = _lib.load()
        x, w, stats, seed_t = ctx.saved_tensors
        eps, gelu, p, seed, stream = ctx.args
        d = x.shape[-1]
        xr, dr = rows_of(x, d), rows_of(dout, d)
        need = ctx.needs_input_grad
        a = _args(xr, w, None, eps, gelu, p, seed, seed_t, stream, _lib.DTYPE_CODES[ctx.out_dtype],
                  None, stats)
        g = _lib.LayerNormGrad(dr.data_ptr(), row_stride(dr))
        dx = dwb = None
        if need[0]:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            g.dx = dx.data_ptr()
        if need[1] or need[2]:
            dwb = torch.empty((2, d), dtype=torch.float32, device=x.device)
            g.dw, g.db = dwb.data_ptr(), dwb.data_ptr() + 4 * d
            g.work_bytes = lib.rp_layernorm_work_bytes(ctypes.byref(a))
            work = torch.empty(max(g.work_bytes, 256), dtype=torch.uint8, device=x.device)
            g.work = work.data_ptr()
        _lib.check(lib.rp_layernorm_bwd(ctypes.byref(a), ctypes.byref(g), _lib.stream_of(x.device)),
                   lib)
        dw = dwb[0].to(ctx.wdtypes[0]) if need[1] else None
        db = dwb[1].to(ctx.wdtypes[1]) if need[2] else None
        return dx, dw, db, None, None, None, None, None, None, None


def hip_layernorm(x, weight=None, bias=None, eps=1e-5, gelu=False, p=0.0, seed=None, stream=0,
                  out_dtype=None):
    """dropout(layer_norm([gelu](x)) * weight + bias, p) over the last dimension.

    x: (..., d) fp32 / bf16 / fp16 on the device, d >= 1; weight, bias: (d,) or
    None (1 and 0); gelu: the exact GELU on x first; p, seed, stream: dropout on
    the result, as hip_dropout draws it (seed may be None where p is 0);
    out_dtype: the result's dtype, x's by default (torch's layer norm under
    autocast gives fp32).  Everything between is fp32.  Differentiable in x,
    weight and bias; the weights' gradients are summed in a fixed order."""
    if not x.is_cuda:
        raise RuntimeError("redpanda_amd layernorm: inputs must be ROCm device tensors")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layernorm: x {tuple(x.shape)} must have a last dimension of at least 1")
    dtype_code(x.dtype, "layernorm")
    if out_dtype is None:
        out_dtype = x.dtype
    else:
        dtype_code(out_dtype, "layernorm")
    grad = x.requires_grad
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.shape != x.shape[-1:] or t.device != x.device:
            raise ValueError(f"layernorm: {name} {tuple(t.shape)} on {t.device} must be "
                             f"({x.shape[-1]},) on {x.device}")
        dtype_code(t.dtype, "layernorm")
        grad = grad or t.requires_grad
    p = check_p(p, "layernorm")
    if not 0 <= stream < 1 << 32:
        raise ValueError(f"layernorm: stream must be in [0, 2^32), got {stream}")
    seed, seed_t = (0, None) if p == 0.0 else seed_arg(seed, x.device, "layernorm")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"layernorm: eps must be >= 0, got {eps}")
    gelu = 1 if gelu else 0
    if grad and torch.is_grad_enabled():
        return _HipLayerNorm.apply(x, weight, bias, eps, gelu, p, seed, seed_t, stream, out_dtype)
    return _forward(x, weight, bias, eps, gelu, p, seed, seed_t, stream, out_dtype, False)[0]
