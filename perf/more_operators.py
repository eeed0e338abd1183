"""The training operators' workloads: embedding, RMS norm with the residual's
addition, checkpoints in 8 bits, and a gated linear recurrence.

What a recurrent backbone runs beside its matrix products: tokens become rows of
the residual stream, each layer's branch is added to it and normed for the next
layer, a checkpointed layer keeps its input until the backward, and a diagonal
recurrence carries a state along the sequence.  Each case is one call of one of
these operators, or one training step (outputs and gradients), at the sizes of
this repository's configurations (the model defaults, bench.py, perf/cases.py)
and odd ones between them.

With `own` false, `run` computes the operators from elementary torch operations;
with `own` true it calls redpanda_amd.
"""

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
BLOCK = 32  # values that share a scale in an 8-bit checkpoint


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The token of one search node.  Launches and latency are all of it.
        dict(name="embed_one_node", kind="embed", N=1, V=8192, d=768, wtype="fp32", out="fp32",
             scale=1.0, train=False),
        # The evaluation model's tokens: 256 boards of 64 squares, whose piece
        # tokens are a dozen ids of the vocabulary's 8192.
        dict(name="embed_eval_train", kind="embed", N=16384, V=8192, d=768, wtype="fp32", out="fp32",
             scale=1.0, train=True),
        # A long-sequence batch (64 games of 2048 tokens), the table in bf16, rows
        # scaled by the root of the width.
        dict(name="embed_long_train", kind="embed", N=131072, V=8192, d=1024, wtype="bf16",
             out="bf16", scale=32.0, train=True),
        # One layer boundary of a search node: a bf16 branch on an fp32 stream.
        dict(name="norm_one_node", kind="norm", rows=1, d=768, dtype="fp32", add="bf16", out="bf16",
             keep8=False, train=False),
        # A layer boundary of the evaluation model under bf16 autocast.
        dict(name="norm_eval_train", kind="norm", rows=16384, d=768, dtype="fp32", add="bf16",
             out="bf16", keep8=False, train=True),
        # Odd rows of an odd width in fp16: no row starts on a vector boundary.
        dict(name="norm_odd_train", kind="norm", rows=1037, d=1001, dtype="fp16", add="fp16",
             out="fp16", keep8=False, train=True),
        # The evaluation model's layer boundary with the stream held in 8 bits
        # until the backward.
        dict(name="keep_eval_train", kind="norm", rows=16384, d=768, dtype="fp32", add="bf16",
             out="bf16", keep8=True, train=True),
        # An activation of the long-sequence batch put into 8 bits and back.
        dict(name="pack_long", kind="pack", rows=131072, d=1024, dtype="bf16"),
        # A ply of 4096 rollouts: one step of the recurrence from given states.
        dict(name="gated_step", kind="gated", B=4096, L=1, D=1024, dtype="fp32", state=True,
             starts=False, train=False),
        # The evaluation model's batch at its inner width.
        dict(name="gated_eval_train", kind="gated", B=256, L=64, D=1536, dtype="bf16", state=False,
             starts=False, train=True),
        # An odd batch with given states and sequences that begin anew inside.
        dict(name="gated_mid_train", kind="gated", B=12, L=250, D=1000, dtype="fp16", state=True,
             starts=True, train=True),
        # 64 games of about 2048 tokens in one row.  The largest.
        dict(name="gated_packed_train", kind="gated", B=1, L=131072, D=1024, dtype="bf16",
             state=False, starts=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    return rng.choice([384, 512, 768, 1024, 1536, _log(rng, 33, 9000), _log(rng, 33, 9000)])


def draw(rng):
    kind = rng.choice(["embed", "embed", "norm", "norm", "norm", "pack", "gated", "gated", "gated"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.7
    d = _width(rng)
    if kind == "embed":
        V = rng.choice([8192, 8192, _log(rng, 20, 131072), _log(rng, 20, 131072)])
        V = max(1, min(V, int(6e7 / d)))
        return dict(kind=kind, N=max(1, min(131072, int(_log(rng, d, 6e7) / d))), V=V, d=d,
                    wtype=dtype, out=rng.choice(["fp32", dtype]),
                    scale=rng.choice([1.0, math.sqrt(d), 0.5]), train=train)
    if kind in ("norm", "pack"):
        rows = max(1, min(131072, int(_log(rng, d, 6e7) / d)))
        if kind == "pack":
            return dict(kind=kind, rows=rows, d=d, dtype=dtype)
        return dict(kind=kind, rows=rows, d=d, dtype=dtype, add=rng.choice(["none", "bf16", dtype]),
                    out=rng.choice(["fp32", dtype]), keep8=rng.random() < 0.4, train=train)
    L = rng.choice([1, 64, _log(rng, 1, 65536), _log(rng, 1, 65536), _log(rng, 1, 65536)])
    B = max(1, min(4096, int(_log(rng, d * L, max(6e7, d * L + 1)) / (d * L))))
    return dict(kind=kind, B=B, L=max(1, min(L, int(6e7 / d))), D=d, dtype=dtype,
                state=rng.random() < 0.5, starts=rng.random() < 0.4, train=train)


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    kind, s, train = case["kind"], dict(case=case), case.get("train", False)
    if kind == "embed":
        N, V, d = case["N"], case["V"], case["d"]
        s["w"] = (0.02 * randn(V, d)).to(DTYPES[case["wtype"]])
        # half of the tokens are squares (13 ids, half of those empty ones), the
        # rest moves, few of them frequent; and some places are padding
        kinds = torch.where(rand(N) < 0.5, 0, (13 * rand(N)).long()).clamp(max=V - 1)
        moves = (V * rand(N) ** 3).long().clamp(max=V - 1)
        ids = torch.where(rand(N) < 0.5, kinds, moves)
        s["ids"] = torch.where(rand(N) < 0.02, -1, ids)
        if train:
            s["dy"] = randn(N, d).to(DTYPES[case["out"]])
            s["w"].requires_grad_(True)
    elif kind in ("norm", "pack"):
        rows, d, dt = case["rows"], case["d"], DTYPES[case["dtype"]]
        # a stream whose rows have levels of their own and a few loud channels
        loud = torch.where(rand(d) < 0.01, 20.0, 1.0)
        s["x"] = (randn(rows, d) * loud * torch.exp(randn(rows, 1))).to(dt)
        if kind == "norm":
            s["add"] = None if case["add"] == "none" else (0.5 * randn(rows, d)).to(DTYPES[case["add"]])
            s["w"] = 1.0 + 0.1 * randn(d)
            if train:
                s["dy"] = randn(rows, d).to(DTYPES[case["out"]])
                leaves = ["x", "w"]
                if s["add"] is not None:
                    leaves.append("add")
                    s["ds"] = randn(rows, d).to(torch.promote_types(dt, s["add"].dtype))
                for k in leaves:
                    s[k].requires_grad_(True)
    else:
        B, L, D, dt = case["B"], case["L"], case["D"], DTYPES[case["dtype"]]
        # the halves of one projection; gates that hold a state for a few steps or
        # for hundreds, each channel around a level of its own
        both = randn(B, L, 2 * D)
        both[..., D:] += 6 * rand(D) - 1
        both = both.to(dt)
        s["x"], s["gate"] = both[..., :D], both[..., D:]
        s["h0"] = randn(B, D) if case["state"] else None
        s["starts"] = None
        if case["starts"]:
            s["starts"] = rand(B, L) < max(1 / 2048, 1.5 / L)
        if train:
            s["dy"], s["dh"] = randn(B, L, D).to(dt), randn(B, D)
            for k in ("x", "gate", "h0"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_embed(s):
    case = s["case"]
    w, ids = s["w"].detach(), s["ids"]
    V = w.shape[0]
    fine = (ids >= 0) & (ids < V)
    at = torch.where(fine, ids, 0)
    y = torch.where(fine[:, None], w[at].float() * case["scale"], 0.0).to(DTYPES[case["out"]])
    if not case["train"]:
        return y
    g = torch.where(fine[:, None], s["dy"].float(), 0.0)
    dw = torch.zeros(V, w.shape[1], device=DEV).index_add_(0, at, g)
    return [y, (dw * case["scale"]).to(w.dtype)]


def _plain_pack(x):
    """The values that x holds in 8 bits: blocks of 32 along a row share a power of
    two, the least that takes the block's largest magnitude to 127 at most after
    rounding (2^-126 for a block of less), and each value is an integer times it."""
    rows, d = x.shape
    f = torch.nn.functional.pad(x.float(), (0, -d % BLOCK)).view(rows, -1, BLOCK)
    m, e = torch.frexp(f.abs().amax(-1, keepdim=True))
    e = torch.where(m * 128 >= 127.5, e - 6, e - 7)
    e = torch.where(m == 0, -126, e.clamp(min=-126))
    # the powers from their exponent fields: a library's power need not be exact
    up, down = ((127 + e) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)
    return (torch.round(f * down) * up).view(rows, -1)[:, :d]


def _plain_norm(s):
    case = s["case"]
    x, w = s["x"].detach(), s["w"].detach().float()
    add = None if s["add"] is None else s["add"].detach()
    stream = x if add is None else (x.float() + add.float()).to(torch.promote_types(x.dtype, add.dtype))
    f = stream.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    y = (f * r * w).to(DTYPES[case["out"]])
    outs = [y] if add is None else [stream, y]
    if not case["train"]:
        return outs
    if case["keep8"]:  # the gradient at the values that were kept
        f = _plain_pack(stream)
        r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    g, xh = s["dy"].float(), f * r
    # a sum over many rows, in 64 bits
    dw = (g * xh).sum(0, dtype=torch.float64).float()
    q = g * w
    dx = r * (q - xh * (q * xh).mean(-1, keepdim=True))
    if add is None:
        return outs + [dx.to(x.dtype), dw]
    dx = dx + s["ds"].float()
    return outs + [dx.to(x.dtype), dx.to(add.dtype), dw]


def _along(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from 0, by doubling."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat((b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]), dim=1)
        a = torch.cat((a[:, :n], a[:, n:] * a[:, :-n]), dim=1)
        n *= 2
    return b


def _plain_gated(s):
    case = s["case"]
    x, gate = s["x"].detach().float(), s["gate"].detach().float()
    h0 = torch.zeros(case["B"], case["D"], device=DEV) if s["h0"] is None else s["h0"].detach()
    keep = 1 / (1 + torch.exp(-gate))
    take = 1 / (1 + torch.exp(gate))
    a = keep if s["starts"] is None else torch.where(s["starts"][..., None], 0.0, keep)
    b = take * x
    b[:, 0] += a[:, 0] * h0
    h = _along(a, b)
    y, last = h.to(s["x"].dtype), h[:, -1].clone()
    if not case["train"]:
        return [y, last]
    g = s["dy"].float()
    g[:, -1] += s["dh"]
    after = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), dim=1)
    adj = _along(after.flip(1), g.flip(1)).flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), dim=1)
    if s["starts"] is not None:
        before = torch.where(s["starts"][..., None], 0.0, before)
    outs = [y, last, (adj * take).to(s["x"].dtype), (adj * (before - x) * keep * take).to(s["x"].dtype)]
    return outs if s["h0"] is None else outs + [adj[:, 0] * a[:, 0]]


# ---------------------------------------------------------------- one pass

def _own_embed(s):
    from redpanda_amd.embedding import hip_embedding
    case = s["case"]
    y = hip_embedding(s["ids"], s["w"], scale=case["scale"], out_dtype=DTYPES[case["out"]])
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (s["w"],), s["dy"])]


def _own_norm(s):
    from redpanda_amd.norm import hip_rmsnorm
    case = s["case"]
    out = hip_rmsnorm(s["x"], s["w"], EPS, add=s["add"], out_dtype=DTYPES[case["out"]],
                      keep8=case["keep8"])
    outs, gouts, ins = (out,), (s.get("dy"),), (s["x"], s["w"])
    if s["add"] is not None:
        outs, gouts, ins = out, (s.get("ds"), s.get("dy")), (s["x"], s["add"], s["w"])
    if not case["train"]:
        return list(outs)
    return [*(t.detach() for t in outs), *torch.autograd.grad(outs, ins, gouts)]


def _own_pack(s):
    from redpanda_amd.checkpoint8 import hip_pack8, hip_unpack8
    return hip_unpack8(hip_pack8(s["x"]))


def _own_gated(s):
    from redpanda_amd.gated import hip_gated_scan
    y, last = hip_gated_scan(s["x"], s["gate"], h0=s["h0"], starts=s["starts"])
    if not s["case"]["train"]:
        return [y, last]
    ins = (s["x"], s["gate"]) if s["h0"] is None else (s["x"], s["gate"], s["h0"])
    return [y.detach(), last.detach(), *torch.autograd.grad((y, last), ins, (s["dy"], s["dh"]))]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"embed": _own_embed, "norm": _own_norm, "pack": _own_pack,
                "gated": _own_gated}[kind](state)
    with torch.no_grad():
        if kind == "pack":
            return _plain_pack(state["x"]).to(state["x"].dtype)
        return {"embed": _plain_embed, "norm": _plain_norm, "gated": _plain_gated}[kind](state)


# ---------------------------------------------------------------- the work

def work(case):
    kind, train = case["kind"], case.get("train", False)
    if kind == "embed":
        N, d, b, o = (case["N"], case["d"], DTYPES[case["wtype"]].itemsize, DTYPES[case["out"]].itemsize)
        # the ids and the rows they name in, the rows out
        nbytes = N * (8 + d * o) + min(N, case["V"]) * d * b
        if train:  # the rows' gradients in, the table's out
            nbytes += N * (8 + d * o) + case["V"] * d * b
        return dict(bytes=nbytes, flops=N * d * (2 if train else 1))
    if kind == "gated":
        n, b, m = case["B"] * case["L"] * case["D"], DTYPES[case["dtype"]].itemsize, case["B"] * case["D"]
        nbytes, flops = 3 * n * b + 4 * m * (2 if case["state"] else 1), 9 * n
        if train:  # x, the gate and dy in, their gradients out; dh, and dh0
            nbytes += 5 * n * b + 4 * m * (2 if case["state"] else 1)
            flops += 20 * n
        return dict(bytes=nbytes, flops=flops)
    n, b = case["rows"] * case["d"], DTYPES[case["dtype"]].itemsize
    if kind == "pack":  # in, the 8 bits and their scales out and in again, out
        return dict(bytes=2 * n * b + 2 * n + 2 * n // BLOCK, flops=4 * n)
    o, e = DTYPES[case["out"]].itemsize, 0
    nbytes = n * (b + o) + 4 * case["d"]
    if case["add"] != "none":
        e = DTYPES[case["add"]].itemsize
        nbytes += n * (e + max(b, e))
    flops = 6 * n
    if train:
        kept = 1 + 1 / BLOCK if case["keep8"] else max(b, e)
        nbytes += n * (kept * (2 if case["keep8"] else 1) + o + b + (max(b, e) + e if e else 0)) + 8 * case["d"]
        flops += 12 * n
    return dict(bytes=int(nbytes), flops=flops)


# ---------------------------------------------------------------- in 64 bits

def _held64(t):
    """What 8 bits hold of an fp32 tensor, from its exponent fields."""
    rows, d = t.shape
    wide = torch.zeros(rows, -(-d // BLOCK) * BLOCK, device=t.device)
    wide[:, :d] = t
    top = wide.abs().view(rows, -1, BLOCK).max(dim=2).values
    bits = top.view(torch.int32)
    # 1.mantissa 2^(field - 127): seven bits up to the half step over 127
    power = (bits >> 23) - 127 - 6 + ((bits & 0x7FFFFF) >= 0x7F0000).int()
    step = ((power.clamp(min=-126).long() + 1023) << 52).view(torch.float64)
    step = step.repeat_interleave(BLOCK, dim=1)
    return (torch.round(wide.double() / step) * step)[:, :d]


def _norm64(case, s):
    x, w = s["x"].detach(), s["w"].detach().double()
    outs, stream = [], x
    if s["add"] is not None:
        kind = torch.promote_types(x.dtype, s["add"].dtype)
        stream = (x.double() + s["add"].detach().double()).to(kind)
        outs.append(stream.double())

    def norm(t, weight):
        return t / torch.sqrt(torch.mean(t ** 2, dim=1, keepdim=True) + EPS) * weight

    outs.append(norm(stream.double(), w))
    if case["train"]:
        kept = _held64(stream.float()) if case["keep8"] else stream.double()
        kept, w = kept.requires_grad_(True), w.requires_grad_(True)
        dx, dw = torch.autograd.grad(norm(kept, w), (kept, w), s["dy"].double())
        if s["add"] is not None:
            dx = dx + s["ds"].double()
            outs.append(dx)
        outs += [dx, dw]
    return outs


def _gated64(case, s):
    B, L, D = case["B"], case["L"], case["D"]
    x, z = s["x"].detach().double(), s["gate"].detach().double()
    h = torch.zeros(B, D, dtype=torch.float64, device=DEV) if s["h0"] is None else s["h0"].detach().double()
    keep = torch.sigmoid(z)
    go = torch.ones(B, L, 1, dtype=torch.float64, device=DEV)
    if s["starts"] is not None:
        go[s["starts"]] = 0
    pull = go * keep
    prev, y = torch.empty_like(x), torch.sigmoid(-z).mul_(x)
    for t in range(L):
        prev[:, t] = h * go[:, t]
        h = torch.addcmul(y[:, t], pull[:, t], h)
        y[:, t] = h
    outs = [y, h]
    if case["train"]:
        adj, lam = s["dy"].double(), s["dh"].double()
        for t in range(L - 1, -1, -1):
            lam = adj[:, t].add_(lam)
            lam = lam * pull[:, t]
        outs += [adj * torch.sigmoid(-z), adj * (prev - x) * keep * torch.sigmoid(-z)]
        if s["h0"] is not None:
            outs.append(lam)
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pack":
        return _held64(s["x"].float())
    if case["kind"] == "norm":
        return _norm64(case, s)
    if case["kind"] == "gated":
        return _gated64(case, s)
    w, ids = s["w"].detach().double(), s["ids"]
    V = w.shape[0]
    # a row of zeros behind the table for the ids that are none of it
    table = torch.cat((w * case["scale"], w.new_zeros(1, w.shape[1])))
    at = torch.where((ids < 0) | (ids >= V), V, ids)
    y = table.index_select(0, at)
    if not case["train"]:
        return y
    order = torch.argsort(at, stable=True)
    run = torch.cumsum(s["dy"].double()[order], dim=0)
    run = torch.cat((torch.zeros_like(run[:1]), run))
    end = torch.searchsorted(at[order].contiguous(), torch.arange(V, device=DEV), right=True)
    sums = run[end]
    sums[1:] -= run[end[:-1]]
    return [y, sums * case["scale"]]
