"""Sampling of a rollout's next move on the HIP kernel: temperature, top-k, top-p
and min-p over the continuation head's logits, or over each rollout's list of
legal moves, from given uniform numbers.

The reference draws on the host from a rollout's top candidates
(engine/mars_search.py:261-276); here a ply's moves are drawn on the device, so
the next step's token ids never leave it.
"""

import ctypes
import math

import torch

from redpanda_amd import _lib
from redpanda_amd.dropout import dtype_code


_WIDE = 8192  # (no row up to it takes a workspace)


def _setting(v, R, dtype, device, name):
    """(value, None) of a number, (0, (R,) tensor) of a setting per row."""
    if not isinstance(v, torch.Tensor):
        return v, None
    if v.shape != (R,) or v.device != device:
        raise ValueError(f"sample: {name} {tuple(v.shape)} on {v.device} must be a number or "
                         f"({R},) on {device}")
    if dtype is torch.int32 and v.dtype is torch.int64:
        v = v.clamp(0, 2**31 - 1)
    if v.dtype is not dtype or not v.is_contiguous():
        v = v.to(dtype).contiguous()
    return 0, v


def _rows(t, n):
    """(t or a contiguous copy with unit inner stride, its row stride)."""
    if t.is_contiguous():
        return t, n
    if t.stride(1) == 1 and t.stride(0) >= n:
        return t, t.stride(0)
    return t.contiguous(), n


def hip_sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, tokens=None,
               logprob=False):
    """One token id a row, (R,) int64; with logprob, (ids, (R,) fp32).

    logits: (R, V) fp32 / bf16 / fp16, unit inner stride; u: (R,) uniform
    numbers in [0, 1).  A row's candidates are its logits above -inf (a NaN is
    none).  In order of value, equal ones by place, those are kept that are among
    the first top_k (0 or less: all), that have less weight before them than
    top_p of these candidates' weight (1 or more: all), and whose weight exp((l -
    max) / temperature) is at least min_p; the first is always kept, and alone
    where the temperature is 0.  The token is the first kept one, in order of its
    place, at which the running sum of weights exceeds u times the total of the
    kept ones.  tokens: None, or (R, M) ids in whose order the candidates stand
    instead of the vocabulary's (ids outside [0, V), like -1, are padding).  Each
    setting is a number or an (R,) tensor, taken in fp32 and not looked at on the
    host: there a temperature of 0 or less, a top_p of 0 or less, a min_p above 1
    or a NaN keeps the first alone, and an infinite temperature gives every
    candidate the same weight (beside +inf only other +inf have one).  A row
    without candidates gives -1 (and -inf); logprob is the logarithm of the token's
    share of the kept weights.  Neither result is differentiable: the logits' gradient
    or tangent ends here, and a loss that needs the log-probability's forms it
    from the logits."""
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError(f"sample: logits must be a (R, V) device tensor, got {tuple(logits.shape)} on "
                         f"{logits.device}")
    R, V = logits.shape
    dev = logits.device
    code = dtype_code(logits.dtype, "sample")
    if V < 1:
        raise ValueError("sample: the vocabulary is empty")
    if u.shape != (R,) or u.device != dev:
        raise ValueError(f"sample: u {tuple(u.shape)} on {u.device} must be ({R},) on {dev}")
    logits, lsr = _rows(logits, V)
    if u.dtype is not torch.float32 or not u.is_contiguous():
        u = u.to(torch.float32).contiguous()
    T, T_row = _setting(temperature, R, torch.float32, dev, "temperature")
    k, k_row = _setting(top_k, R, torch.int32, dev, "top_k")
    tp, tp_row = _setting(top_p, R, torch.float32, dev, "top_p")
    mp, mp_row = _setting(min_p, R, torch.float32, dev, "min_p")
    if not T >= 0 or math.isinf(T):
        raise ValueError(f"sample: temperature must be finite and >= 0, got {T}")
    if not tp >= 0 or not 0 <= mp <= 1:
        raise ValueError(f"sample: top_p must be >= 0 and min_p in [0, 1], got {tp} and {mp}")
    ids = torch.empty(R, dtype=torch.int64, device=dev)
    logp = torch.empty(R, dtype=torch.float32, device=dev) if logprob else None
    a = _lib.SampleArgs(R, V, 0, code, 0, logits.data_ptr(), lsr, u.data_ptr(), None, 0,
                        T, tp, mp, min(max(int(k), 0), 1 << 31), _lib.ptr(T_row), _lib.ptr(tp_row),
                        _lib.ptr(mp_row), _lib.ptr(k_row), ids.data_ptr(), _lib.ptr(logp))
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != R or tokens.device != dev:
            raise ValueError(f"sample: tokens {tuple(tokens.shape)} on {tokens.device} must be "
                             f"({R}, M) on {dev}")
        if tokens.dtype is not torch.int32:
            if tokens.dtype is not torch.int64:
                raise TypeError(f"sample: tokens must be int32 or int64, got {tokens.dtype}")
            # an id beyond int32 is none of the vocabulary's either way
            tokens = tokens.clamp(-1, 2**31 - 1).to(torch.int32)
        if tokens.shape[1] == 0:
            tokens = tokens.new_full((R, 1), -1)  # (a list without storage would read as none)
        M = tokens.shape[1]
        tokens, a.tokens_sr = _rows(tokens, M)
        a.M, a.tokens = M, tokens.data_ptr()
    lib = _lib.load()
    if V > _WIDE and tokens is None:
        a.work_bytes = lib.rp_sample_work_bytes(ctypes.byref(a))
        if a.work_bytes > 0:
            work = torch.empty(a.work_bytes, dtype=torch.uint8, device=dev)
            a.work = work.data_ptr()
    _lib.check(lib.rp_sample(ctypes.byref(a), _lib.stream_of(dev)), lib)
    return (ids, logp) if logprob else ids
