"""Residual add + RMSNorm on the HIP kernels (engine/mamba.py:82-89 RMSNorm; the
pre-norm loop of Mamba.step, :592-597).

hip_add_rmsnorm: the batched step's residual stream, fp32 and forward only, used
by the inference loop of Mamba.step when no autograd graph is being recorded.

hip_rmsnorm: for training, in every type and both ways, in one pass each; the
backward reads the stream, or with keep8 the stream in 8 bits, which the forward
writes beside the rest.
"""

import ctypes

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import dtype_code, empty_rows, once, recorded, rows_of


def hip_add_rmsnorm(x, add, w, eps):
    """(x + add, RMSNorm(x + add) * w) for fp32 rows x (R, d); add: None or
    (R, d) in fp32 / bf16 / fp16 (x itself is normalised then, and returned
    as the first element).  Torch's op order: (x' * rsqrt(mean(x'^2) + eps))
    * w, the mean as the sum times the fp32 reciprocal of d."""
    if x.dim() != 2 or x.dtype != torch.float32 or not x.is_cuda:
        raise ValueError("add_rmsnorm: x must be a (R, d) fp32 device tensor")
    R, d = x.shape
    if w.shape != (d,):
        raise ValueError(f"add_rmsnorm: weight {tuple(w.shape)} must be ({d},)")
    lib = _lib.load()
    if x.stride(-1) != 1:
        x = x.contiguous()
    wc = w  # only its data pointer is used
    if w.dtype is not torch.float32 or not w.is_contiguous():
        wc = w.detach().to(torch.float32).contiguous()
    a = _lib.RmsNormArgs()
    a.rows, a.d, a.eps = R, d, float(eps)
    a.x, a.x_sr = x.data_ptr(), x.stride(0)
    a.w = wc.data_ptr()
    out = torch.empty((R, d), dtype=torch.float32, device=x.device)
    a.out = out.data_ptr()
    x_new = x
    if add is not None:
        if add.shape != (R, d):
            raise ValueError(f"add_rmsnorm: add {tuple(add.shape)} must be {(R, d)}")
        if add.stride(-1) != 1:
            add = add.contiguous()
        try:
            a.dtype_add = _lib.DTYPE_CODES[add.dtype]
        except KeyError:
            raise TypeError(f"add_rmsnorm: unsupported dtype {add.dtype}") from None
        a.add, a.add_sr = add.data_ptr(), add.stride(0)
        x_new = torch.empty((R, d), dtype=torch.float32, device=x.device)
        a.x_out = x_new.data_ptr()
    _lib.check(lib.rp_rmsnorm_fwd(ctypes.byref(a), _lib.stream_of(x.device)), lib)
    return x_new, out


def _f32c(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def pack_buffers(t):
    """(q, e) for the rows of t in 8 bits: int8 of its shape, and an exponent for
    each 32 columns."""
    d = t.shape[-1]
    return (empty_rows(t, torch.int8),
            torch.empty((*t.shape[:-1], (d + 31) // 32), dtype=torch.uint8, device=t.device))


def norm_forward(x, add, w, eps, out_dtype, pack):
    """(sum or x, out, (q, e) or None, w in fp32, the arguments)."""
    lib = _lib.load()
    d = x.shape[-1]
    xr, rows, sr = rows_of(x, d)
    w = _f32c(w)
    out = empty_rows(x, out_dtype)
    code = _lib.DTYPE_CODES[x.dtype]
    a = _lib.AddNormArgs(rows, d, code, code, code, _lib.DTYPE_CODES[out_dtype], xr.data_ptr(), sr,
                         None, 0, None if w is None else w.data_ptr(), None, out.data_ptr(), None,
                         None, eps, 0)
    total = x
    if add is not None:
        ar, _, asr = rows_of(add, d)
        total = empty_rows(x, torch.promote_types(x.dtype, add.dtype))
        a.dtype_add, a.dtype_sum = _lib.DTYPE_CODES[add.dtype], _lib.DTYPE_CODES[total.dtype]
        a.add, a.add_sr, a.sum = ar.data_ptr(), asr, total.data_ptr()
    kept = None
    if pack:
        kept = pack_buffers(x)
        a.q, a.e = kept[0].data_ptr(), kept[1].data_ptr()
    _lib.call(lib.rp_addnorm_fwd, out.device, ctypes.byref(a))
    return total, out, kept, w, a


def norm_again(kept, w, args, out_dtype):
    """The norm's result for the rows that `kept` holds."""
    out = empty_rows(kept[0], out_dtype)
    a = _lib.AddNormArgs.from_buffer_copy(args)
    a.x = a.add = a.sum = None
    a.w = None if w is None else w.data_ptr()
    a.out, a.q, a.e = out.data_ptr(), kept[0].data_ptr(), kept[1].data_ptr()
    _lib.call(_lib.load().rp_addnorm_fwd, out.device, ctypes.byref(a))
    return out


def norm_backward(total, kept, w, args, dtypes, dsum, dout, need):
    """(dx, dadd, dw) of the norm, those that `need` (x, add, w) asks for.

    total: the rows, or None where `kept` holds them; args: the forward's; dtypes:
    those of x, add and w (None for one that was not given)."""
    lib = _lib.load()
    xt, at, wt = dtypes
    rows = total if total is not None else kept[0]
    d = args.d
    if dout is None:  # (nothing came through the norm)
        gx = None if dsum is None or not need[0] else dsum.to(xt)
        ga = None if dsum is None or not need[1] else dsum.to(at)
        return gx, ga, None
    a = _lib.AddNormArgs.from_buffer_copy(args)
    a.w = None if w is None else w.data_ptr()
    a.add = a.sum = a.out = None
    if total is not None:
        xr, _, a.x_sr = rows_of(total, d)
        a.x, a.q, a.e = xr.data_ptr(), None, None
    else:
        a.x, a.q, a.e = None, kept[0].data_ptr(), kept[1].data_ptr()
    dr, _, dsr = rows_of(dout, d)
    g = _lib.AddNormGrad(dr.data_ptr(), dsr)
    if dsum is not None:
        sr, _, ssr = rows_of(dsum, d)
        g.dsum, g.dsum_sr = sr.data_ptr(), ssr
    dx = dadd = dw = work = None
    same = at is xt and need[0]
    if need[0]:
        dx = empty_rows(rows, xt)
        g.dx = dx.data_ptr()
    if need[1] and not same:
        dadd = empty_rows(rows, at)
        g.dadd = dadd.data_ptr()
    nbytes = 0
    if need[2]:
        dw = torch.empty(d, dtype=torch.float32, device=rows.device)
        g.dw = dw.data_ptr()
    if need[2] or d > 16384:
        nbytes = lib.rp_addnorm_work_bytes(ctypes.byref(a))
        work = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=rows.device)
        g.work, g.work_bytes = work.data_ptr(), nbytes
    _lib.call(lib.rp_addnorm_bwd, rows.device, ctypes.byref(a), ctypes.byref(g))
    if need[1] and same:
        dadd = dx
    return dx, dadd, dw if dw is None or wt is torch.float32 else dw.to(wt)


class _HipRmsNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, add, w, eps, out_dtype, keep8):
        total, out, kept, wc, a = norm_forward(x, add, w, eps, out_dtype, keep8)
        if keep8:
            ctx.save_for_backward(wc, *kept)
        else:
            ctx.save_for_backward(wc, total)
        ctx.args = a
        ctx.keep8 = keep8
        ctx.dtypes = (x.dtype, None if add is None else add.dtype, None if w is None else w.dtype)
        ctx.set_materialize_grads(False)
        return out if add is None else (total, out)

    @staticmethod
    @once
    def backward(ctx, *grads):
        dsum, dout = grads if len(grads) == 2 else (None, grads[0])
        w, *rest = ctx.saved_tensors
        total, kept = (None, rest) if ctx.keep8 else (rest[0], None)
        dx, dadd, dw = norm_backward(total, kept, w, ctx.args, ctx.dtypes, dsum, dout,
                                     ctx.needs_input_grad)
        return dx, dadd, dw, None, None, None


def check_norm(x, weight, eps, add, out_dtype, what):
    """(eps, out_dtype, whether an input requires a gradient) after the checks."""
    if not x.is_cuda:
        raise RuntimeError(f"redpanda_amd {what}: inputs must be ROCm device tensors")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} must have a last dimension of at least 1")
    dtype_code(x.dtype, what)
    grad = x.requires_grad
    if out_dtype is None:
        out_dtype = x.dtype
    else:
        dtype_code(out_dtype, what)
    if add is not None:
        if add.shape != x.shape or add.device != x.device:
            raise ValueError(f"{what}: add {tuple(add.shape)} on {add.device} must be "
                             f"{tuple(x.shape)} on {x.device}")
        dtype_code(add.dtype, what)
        grad = grad or add.requires_grad
    if weight is not None:
        if weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.device != x.device:
            raise ValueError(f"{what}: weight {tuple(weight.shape)} on {weight.device} must be "
                             f"({x.shape[-1]},) on {x.device}")
        dtype_code(weight.dtype, what)
        grad = grad or weight.requires_grad
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must be >= 0, got {eps}")
    return eps, out_dtype, grad


def hip_rmsnorm(x, weight=None, eps=1e-5, add=None, out_dtype=None, keep8=False):
    """RMSNorm(x) * weight over the last dimension; with add, (x + add, RMSNorm(x +
    add) * weight).

    x, add: (..., d) fp32 / bf16 / fp16 on the device, d >= 1; the sum has the type
    torch promotes the two to, and is rounded to it before it is normed; weight: (d,)
    or None (1); out_dtype: the norm's, x's by default.  Everything between is fp32.
    keep8: the backward keeps the sum (x without add) in 8 bits, as hip_pack8 holds it,
    and gives the gradient at those values; the results are the same.  Differentiable in
    x, add and weight, once and in reverse mode (a tangent is refused); the weight's
    gradient is summed in a fixed order."""
    eps, out_dtype, grad = check_norm(x, weight, eps, add, out_dtype, "rmsnorm")
    if recorded(grad):
        return _HipRmsNorm.apply(x, add, weight, eps, out_dtype, bool(keep8))
    total, out, _, _, _ = norm_forward(x, add, weight, eps, out_dtype, False)
    return out if add is None else (total, out)
