"""A gated linear recurrence on the HIP kernels, beside the selective scan.

    a_t = sigmoid(gate_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t

each channel by itself: one state a channel where the selective scan has N, for
mixers that need no more, at the price of reading their inputs.  Long sequences of
few channels are split along time; the step for single tokens is the same kernel.
"""

import ctypes

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import dtype_code, once, recorded


def _seq(t):
    """(t or a copy of it whose channels are adjacent, its batch and time strides)."""
    B, L, D = t.shape
    if t.is_contiguous():
        return t, L * D, D
    sb, sl, sd = t.stride()
    if (sd == 1 or D == 1) and (sl >= D or L == 1):
        # (a stride along a dimension of one is any number)
        return t, sb if B > 1 else 0, sl if L > 1 else D
    return t.contiguous(), L * D, D


def _args(x, gate, starts):
    B, L, D = x.shape
    a = _lib.GatedArgs(B, L, D, _lib.DTYPE_CODES[x.dtype], 0)
    x, a.x_sb, a.x_sl = _seq(x)
    gate, a.gate_sb, a.gate_sl = _seq(gate)
    a.x, a.gate = x.data_ptr(), gate.data_ptr()
    if starts is not None:
        a.starts, a.starts_sb = starts.data_ptr(), L
    return a, (x, gate, starts)  # (copies live as long as the call)


def _work(lib, a, device):
    a.work_bytes = lib.rp_gated_work_bytes(ctypes.byref(a))
    if a.work_bytes <= 0:
        return None
    work = torch.empty(a.work_bytes, dtype=torch.uint8, device=device)
    a.work = work.data_ptr()
    return work


def _forward(x, gate, h0, starts, keep):
    lib = _lib.load()
    B, L, D = x.shape
    if x.numel() == 0:  # the last state is the first
        last = torch.zeros((B, D), dtype=torch.float32, device=x.device)
        return torch.empty((B, L, D), dtype=x.dtype, device=x.device), last if h0 is None else last.copy_(h0), None
    a, hold = _args(x, gate, starts)
    y = torch.empty((B, L, D), dtype=x.dtype, device=x.device)
    last = torch.empty((B, D), dtype=torch.float32, device=x.device)
    if h0 is not None:
        h0 = h0.contiguous()
        a.h0 = h0.data_ptr()
    ckpt = None
    if keep:
        nbytes = lib.rp_gated_ckpt_bytes(ctypes.byref(a))
        if nbytes < 0:
            _lib.check(lib.rp_gated_check(ctypes.byref(a)), lib)
        ckpt = torch.empty(nbytes // 4, dtype=torch.float32, device=x.device)
        a.ckpt = ckpt.data_ptr()
    work = _work(lib, a, x.device)  # noqa: F841  (held until the launch)
    a.y, a.h_last = y.data_ptr(), last.data_ptr()
    _lib.call(lib.rp_gated_fwd, x.device, ctypes.byref(a))
    return y, last, ckpt


class _HipGatedScan(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, gate, h0, starts):
        y, last, ckpt = _forward(x, gate, h0, starts, True)
        ctx.save_for_backward(x, gate, starts, ckpt)
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return None, None, None, None
        lib = _lib.load()
        x, gate, starts, ckpt = ctx.saved_tensors
        B, L, D = x.shape
        need = ctx.needs_input_grad
        if x.numel() == 0:
            return (torch.zeros_like(x) if need[0] else None, torch.zeros_like(gate) if need[1] else None,
                    dlast if need[2] else None, None)
        a, hold = _args(x, gate, starts)
        a.ckpt = ckpt.data_ptr()
        work = _work(lib, a, x.device)  # noqa: F841  (held until the launch)
        dx = torch.empty((B, L, D), dtype=x.dtype, device=x.device)
        dgate = torch.empty_like(dx)
        g = _lib.GatedGrad(dx=dx.data_ptr(), dgate=dgate.data_ptr())
        if dy is not None:
            dy, g.dy_sb, g.dy_sl = _seq(dy)
            g.dy = dy.data_ptr()
        if dlast is not None:
            dlast = dlast.contiguous()
            g.dh_last = dlast.data_ptr()
        dh0 = None
        if need[2]:
            dh0 = torch.empty((B, D), dtype=torch.float32, device=x.device)
            g.dh0 = dh0.data_ptr()
        _lib.call(lib.rp_gated_bwd, x.device, ctypes.byref(a), ctypes.byref(g))
        return dx if need[0] else None, dgate if need[1] else None, dh0, None


def hip_gated_scan(x, gate, h0=None, starts=None):
    """(y, h_last): the states of h_t = a_t h_{t-1} + (1 - a_t) x_t, a_t =
    sigmoid(gate_t), along dimension 1.

    x, gate: (B, L, D) of one dtype (fp32 / bf16 / fp16) on the device, any strides (the
    halves of one projection are read in place); h0: (B, D) fp32 or None (0).  starts:
    None, or (B, L) bool: where it is True a sequence begins anew, h_{t-1} counting as 0
    (packed sequences).  A gate of +inf keeps the state as it is where x_t is
    finite (padding behind a sequence's end), of -inf takes x_t where the state is finite
    (and so beyond about +-87, where fp32's exp is 0): 0 times an infinity or a NaN is NaN,
    as in the formula; an infinite state stays one through all other gates.  y: (B, L, D)
    in x's dtype; h_last: (B, D) fp32, the last state (h0 where L is 0).  The state is fp32 throughout.  Differentiable in x,
    gate and h0, once and in reverse mode (a tangent is refused)."""
    if not x.is_cuda:
        raise RuntimeError("redpanda_amd gated_scan: inputs must be ROCm device tensors")
    if x.dim() != 3:
        raise ValueError(f"gated_scan: x {tuple(x.shape)} must be (B, L, D)")
    dev = x.device
    if gate.shape != x.shape or gate.device != dev:
        raise ValueError(f"gated_scan: gate {tuple(gate.shape)} on {gate.device} must be "
                         f"{tuple(x.shape)} on {dev}")
    dtype_code(x.dtype, "gated_scan")
    if gate.dtype is not x.dtype:
        raise TypeError(f"redpanda_amd gated_scan: gate is {gate.dtype} and x {x.dtype}: one dtype is "
                        "wanted")
    B, L, D = x.shape
    grad = x.requires_grad or gate.requires_grad
    if h0 is not None:
        if h0.shape != (B, D) or h0.device != dev:
            raise ValueError(f"gated_scan: h0 {tuple(h0.shape)} on {h0.device} must be ({B}, {D}) on {dev}")
        if h0.dtype is not torch.float32:
            raise TypeError(f"redpanda_amd gated_scan: h0 must be float32, got {h0.dtype}")
        grad = grad or h0.requires_grad
    if starts is not None:
        if starts.shape != (B, L) or starts.device != dev:
            raise ValueError(f"gated_scan: starts {tuple(starts.shape)} on {starts.device} must be "
                             f"({B}, {L}) on {dev}")
        if starts.dtype is not torch.bool:
            raise TypeError(f"redpanda_amd gated_scan: starts must be bool, got {starts.dtype}")
        starts = starts.contiguous()
    if recorded(grad):
        return _HipGatedScan.apply(x, gate, h0, starts)
    return _forward(x, gate, h0, starts, False)[:2]


def hip_gated_step(x, gate, h=None):
    """(y, h) of one token a row: x, gate (R, D), h (R, D) fp32 or None (0); as
    hip_gated_scan with L = 1."""
    if x.dim() != 2:
        raise ValueError(f"gated_step: x {tuple(x.shape)} must be (R, D)")
    y, last = hip_gated_scan(x.unsqueeze(1), gate.unsqueeze(1), h)
    return y.squeeze(1), last
