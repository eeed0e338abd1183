"""Embedding lookup on the HIP kernels, with the table's gradient by sorted tokens.

torch's nn.Embedding adds the rows' gradients by atomics, whose order (and with it
the last bits) changes from run to run, and which wait for each other where a few
tokens are frequent, as a board's empty squares are.  Here the places are sorted by
their ids and each id's rows are added in order.
"""

import ctypes

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import dtype_code, once, recorded, rows_of


def _args(ids, V, d, wt, out_dtype, scale, padding):
    return _lib.EmbeddingArgs(ids.numel(), V, d, _lib.DTYPE_CODES[wt], _lib.DTYPE_CODES[out_dtype],
                              ids.dtype is torch.int64, scale, padding, ids.data_ptr())


def _forward(ids, w, scale, padding, out_dtype):
    lib = _lib.load()
    V, d = w.shape
    out = torch.empty((*ids.shape, d), dtype=out_dtype, device=w.device)
    if out.numel() == 0:
        return out
    ids = ids.contiguous()
    wr, _, wsr = rows_of(w, d)
    a = _args(ids, V, d, w.dtype, out_dtype, scale, padding)
    a.w, a.w_sr, a.out = wr.data_ptr(), wsr, out.data_ptr()
    _lib.call(lib.rp_embedding_fwd, out.device, ctypes.byref(a))
    return out


class _HipEmbedding(torch.autograd.Function):

    @staticmethod
    def forward(ctx, ids, w, scale, padding, out_dtype):
        ctx.save_for_backward(ids)
        ctx.args = (w.shape, w.dtype, scale, padding, out_dtype)
        return _forward(ids, w, scale, padding, out_dtype)

    @staticmethod
    @once
    def backward(ctx, dout):
        lib = _lib.load()
        (ids,) = ctx.saved_tensors
        (V, d), wt, scale, padding, out_dtype = ctx.args
        dw = torch.empty((V, d), dtype=wt, device=dout.device)
        if d == 0:
            return None, dw, None, None, None
        ids = ids.contiguous()
        a = _args(ids, V, d, wt, out_dtype, scale, padding)
        dr, _, dsr = rows_of(dout, d)
        nbytes = lib.rp_embedding_work_bytes(ctypes.byref(a))
        work = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dout.device)
        g = _lib.EmbeddingGrad(dr.data_ptr(), dsr, dw.data_ptr(), work.data_ptr(), nbytes)
        _lib.call(lib.rp_embedding_bwd, dw.device, ctypes.byref(a), ctypes.byref(g))
        return None, dw, None, None, None


def hip_embedding(ids, weight, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * weight[ids], rounded once.

    ids: int32 or int64 of any shape; an id outside [0, V), like -1, is padding: its
    row is zeros, and it takes no gradient (nothing is checked on the host).  weight:
    (V, d) fp32 / bf16 / fp16 on the device; the result is (*ids.shape, d) in out_dtype,
    weight's by default.  padding_idx: as torch's, an id whose row of the table gets no
    gradient.  Differentiable in weight, once and in reverse mode (a tangent is
    refused): a dense (V, d) gradient, each row an fp32 sum in the order of the
    places."""
    if not weight.is_cuda:
        raise RuntimeError("redpanda_amd embedding: inputs must be ROCm device tensors")
    if weight.dim() != 2 or weight.shape[0] < 1:
        raise ValueError(f"embedding: weight {tuple(weight.shape)} must be (V, d) with V >= 1")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"redpanda_amd embedding: ids must be int32 or int64, got {ids.dtype}")
    if ids.device != weight.device:
        raise ValueError(f"embedding: ids on {ids.device} must be on {weight.device}")
    dtype_code(weight.dtype, "embedding")
    if out_dtype is None:
        out_dtype = weight.dtype
    else:
        dtype_code(out_dtype, "embedding")
    padding = -1
    if padding_idx is not None:
        V = weight.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} must be in [-{V}, {V})")
        padding = padding_idx % V
    scale = float(scale)
    if recorded(weight.requires_grad):
        return _HipEmbedding.apply(ids, weight, scale, padding, out_dtype)
    return _forward(ids, weight, scale, padding, out_dtype)
