"""Layer norm on the HIP kernels, with GELU before it and dropout behind it.

The middle of a search model's head (engine/search_mamba.py:52-72: Linear, GELU,
LayerNorm, Linear) in one pass over its rows, forward and backward: GELU's value
and slope are formed again from the input in the backward, the dropout's mask is
drawn again from its seed, and of the rows only the mean and the inverse of the
standard deviation are kept.
"""

import ctypes

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import check_p, dtype_code, empty_rows, once, recorded, rows_of, seed_arg


def _f32c(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def _forward(x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype, keep):
    """(out, w in fp32, the rows' stats or None, the arguments)."""
    lib = _lib.load()
    d = x.shape[-1]
    xr, rows, sr = rows_of(x, d)
    w, b = _f32c(w), _f32c(b)
    out = empty_rows(x, out_dtype)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=out.device) if keep else None
    a = _lib.LayerNormArgs(rows, d, _lib.DTYPE_CODES[x.dtype], _lib.DTYPE_CODES[out_dtype], gelu,
                           stream, p, seed, None if seed_t is None else seed_t.data_ptr(),
                           xr.data_ptr(), sr, None if w is None else w.data_ptr(),
                           None if b is None else b.data_ptr(), out.data_ptr(),
                           None if stats is None else stats.data_ptr(), eps, 0)
    _lib.check(lib.rp_layernorm_fwd(ctypes.byref(a), _lib.stream_of(out.device)), lib)
    return out, w, stats, a


class _HipLayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype):
        out, wc, stats, a = _forward(x, w, b, eps, gelu, p, seed, seed_t, stream, out_dtype, True)
        ctx.save_for_backward(x, wc, stats, seed_t)
        # the forward's settings; its pointers are set anew from the saved tensors
        ctx.args = a
        ctx.dtypes = (None if w is None else w.dtype, None if b is None else b.dtype)
        return out

    @staticmethod
    @once
    def backward(ctx, dout):
        lib = _lib.load()
        x, w, stats, seed_t = ctx.saved_tensors
        a = _lib.LayerNormArgs.from_buffer_copy(ctx.args)
        d = a.d
        xr, _, a.x_sr = rows_of(x, d)
        a.x, a.out, a.stats = xr.data_ptr(), None, stats.data_ptr()
        a.w = None if w is None else w.data_ptr()
        a.seed_ptr = None if seed_t is None else seed_t.data_ptr()
        dr, _, dsr = rows_of(dout, d)
        g = _lib.LayerNormGrad(dr.data_ptr(), dsr)
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0]:
            dx = empty_rows(x, x.dtype)
            g.dx = dx.data_ptr()
        if need[1] or need[2]:
            dw = torch.empty(d, dtype=torch.float32, device=stats.device)
            db = torch.empty_like(dw)
            nbytes = lib.rp_layernorm_work_bytes(ctypes.byref(a))
            work = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=stats.device)
            g.dw, g.db, g.work, g.work_bytes = dw.data_ptr(), db.data_ptr(), work.data_ptr(), nbytes
        _lib.check(lib.rp_layernorm_bwd(ctypes.byref(a), ctypes.byref(g), _lib.stream_of(stats.device)),
                   lib)
        wt, bt = ctx.dtypes
        dw = None if not need[1] else dw if wt is torch.float32 else dw.to(wt)
        db = None if not need[2] else db if bt is torch.float32 else db.to(bt)
        return dx, dw, db, None, None, None, None, None, None, None


def hip_layernorm(x, weight=None, bias=None, eps=1e-5, gelu=False, p=0.0, seed=None, stream=0,
                  out_dtype=None):
    """dropout(layer_norm([gelu](x)) * weight + bias, p) over the last dimension.

    x: (..., d) fp32 / bf16 / fp16 on the device, d >= 1; weight, bias: (d,) or
    None (1 and 0); gelu: the exact GELU on x first; p, seed, stream: dropout on
    the result, as hip_dropout draws it (seed may be None where p is 0);
    out_dtype: the result's dtype, x's by default (torch's layer norm under
    autocast gives fp32).  Everything between is fp32.  Differentiable in x,
    weight and bias, once and in reverse mode (a tangent is refused); the weights'
    gradients are summed in a fixed order."""
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
    for t in (weight, bias):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != x.shape[-1] or t.device != x.device:
                raise ValueError(f"layernorm: {'weight' if t is weight else 'bias'} {tuple(t.shape)} "
                                 f"on {t.device} must be ({x.shape[-1]},) on {x.device}")
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
    if recorded(grad):
        return _HipLayerNorm.apply(x, weight, bias, eps, gelu, p, seed, seed_t, stream, out_dtype)
    return _forward(x, weight, bias, eps, gelu, p, seed, seed_t, stream, out_dtype, False)[0]
