"""The head operators' workloads: layer norm, dropout and sampling.

A search model's heads are Linear -> GELU -> LayerNorm -> Linear; training puts
dropout behind the norm and on the layers' residual branches, and a rollout
draws its next move from the continuation head's logits.  Each case is one call
of one of these operators, or one training step (output and gradients), at the
sizes of this repository's configurations (the model defaults, bench.py,
perf/cases.py) and odd ones between them.

With `own` false, `run` computes the operators from elementary torch operations;
with `own` true it calls redpanda_amd.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
U32 = 0xFFFFFFFF


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One node of a search: the value head's GELU and norm for one row.
        # Launches and latency are all of it.
        dict(name="norm_one_node", kind="norm", rows=1, d=384, dtype="fp32", out="fp32", gelu=True,
             p=0.0, train=False),
        # The continuation head of a ply of 4096 rollouts, fp32, no gradients.
        dict(name="norm_rollouts", kind="norm", rows=4096, d=768, dtype="fp32", out="fp32",
             gelu=True, p=0.0, train=False),
        # Training the continuation head on 64 boards of 8 plies, with dropout.
        dict(name="norm_dynamics_train", kind="norm", rows=512, d=768, dtype="fp32", out="fp32",
             gelu=True, p=0.1, train=True),
        # A plain norm of the evaluation model's tokens (256 boards of 64) under
        # bf16 autocast: 16-bit rows in, fp32 out, as torch's own norm gives.
        dict(name="norm_eval_train", kind="norm", rows=16384, d=768, dtype="bf16", out="fp32",
             gelu=False, p=0.0, train=True),
        # Odd rows of an odd width in fp16: no row starts on a vector boundary.
        dict(name="norm_odd_train", kind="norm", rows=1037, d=1001, dtype="fp16", out="fp16",
             gelu=True, p=0.1, train=True),
        # Heads over every token of a long-sequence batch (64 games of 2048
        # tokens), bf16 both ways.  The largest.
        dict(name="norm_long_train", kind="norm", rows=131072, d=1024, dtype="bf16", out="bf16",
             gelu=True, p=0.2, train=True),
        # The residual branch of a small fp32 training batch (9 x 71 tokens).
        dict(name="drop_small_train", kind="drop", rows=639, d=384, dtype="fp32", res="fp32", p=0.1,
             train=True),
        # The evaluation model's residual branch: a bf16 branch on an fp32 stream.
        dict(name="drop_eval_train", kind="drop", rows=16384, d=768, dtype="bf16", res="fp32",
             p=0.1, train=True),
        # The move of one search node: one row of the vocabulary.
        dict(name="sample_one", kind="sample", R=1, V=8192, M=0, dtype="fp32", each=False, T=0.8,
             k=40, tp=0.95, mp=0.0),
        # A ply of 4096 rollouts under bf16 autocast, nucleus sampling.
        dict(name="sample_rollouts", kind="sample", R=4096, V=8192, M=0, dtype="bf16", each=False,
             T=1.0, k=0, tp=0.9, mp=0.0),
        # The same for an odd number of rollouts over their legal-move lists.
        dict(name="sample_legal", kind="sample", R=777, V=8192, M=218, dtype="fp32", each=False,
             T=0.7, k=0, tp=1.0, mp=0.05),
        # A served batch over a wide odd vocabulary, each row with settings of
        # its own.
        dict(name="sample_wide", kind="sample", R=64, V=100003, M=0, dtype="fp32", each=True, T=1.0,
             k=50, tp=0.92, mp=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "drop", "drop", "sample", "sample", "sample"])
    p = rng.choice([0.0, 0.05, 0.1, 0.2, 0.5])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "norm":
        d = rng.choice([384, 512, 768, 1024, 1536, _log(rng, 33, 9000), _log(rng, 33, 9000)])
        rows = max(1, min(131072, int(_log(rng, 400, 1.3e8) / d)))
        return dict(kind=kind, rows=rows, d=d, dtype=dtype, out=rng.choice(["fp32", dtype]),
                    gelu=rng.random() < 0.6, p=p, train=rng.random() < 0.7)
    if kind == "drop":
        d = rng.choice([384, 512, 768, 1024, 1536, _log(rng, 33, 9000), _log(rng, 33, 9000)])
        rows = max(1, min(65536, int(_log(rng, 400, 3e7) / d)))
        return dict(kind=kind, rows=rows, d=d, dtype=dtype, res=rng.choice(["none", "fp32", dtype]),
                    p=max(p, 0.05), train=rng.random() < 0.7)
    V = rng.choice([8192, 8192, _log(rng, 20, 131072), _log(rng, 20, 131072)])
    R = max(1, min(4096, int(_log(rng, V, 3.3e7) / V)))
    M = rng.randint(1, min(V, 256)) if rng.random() < 0.3 else 0
    return dict(kind=kind, R=R, V=V, M=M, dtype=dtype, each=rng.random() < 0.4,
                T=rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]), k=rng.choice([0, 0, 1, 8, 40, 200, 1000]),
                tp=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95]), mp=rng.choice([0.0, 0.0, 0.02, 0.1]))


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    kind, s = case["kind"], dict(case=case)
    if kind in ("norm", "drop"):
        rows, d, dt = case["rows"], case["d"], DTYPES[case["dtype"]]
        # the training loop's seed, on the device so that a graph can read it
        s["seed"] = torch.randint(0, 2**62, (1,), generator=g, device=DEV)
        # rows as a projection gives them, each with a level of its own
        s["x"] = (randn(rows, d) + 0.3 * randn(rows, 1)).to(dt)
    if kind == "norm":
        s["w"], s["b"] = 1.0 + 0.1 * randn(d), 0.1 * randn(d)
        if case["train"]:
            s["dy"] = randn(rows, d).to(DTYPES[case["out"]])
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
    elif kind == "drop":
        s["res"] = None if case["res"] == "none" else (2 * randn(rows, d)).to(DTYPES[case["res"]])
        if case["train"]:
            s["dy"] = randn(rows, d).to(dt if s["res"] is None else torch.promote_types(dt, s["res"].dtype))
            s["x"].requires_grad_(True)
    else:
        R, V, M = case["R"], case["V"], case["M"]
        lg = 2.5 * randn(R, V)
        # ids that are never moves, and in some batches a row with nothing left
        lg.masked_fill_(rand(1, V) < 0.02, -math.inf)
        if R > 2 and seed % 2:
            lg[R // 2] = -math.inf
        s["logits"], s["u"] = lg.to(DTYPES[case["dtype"]]), rand(R)
        s["tokens"] = None
        if M:
            # distinct ids in ascending order, as a move generator lists them,
            # from none at all to M of them, padded with -1
            ids = torch.sort(torch.argsort(rand(R, V), dim=1)[:, :M], dim=1).values
            n = (rand(R, 1) * (M + 1)).long()
            s["tokens"] = torch.where(torch.arange(M, device=DEV) < n, ids, -1).to(torch.int32)
        s["T"], s["k"], s["tp"], s["mp"] = case["T"], case["k"], case["tp"], case["mp"]
        if case["each"]:
            # one setting a row around the case's
            s["T"] = case["T"] * (0.5 + rand(R))
            s["k"] = (case["k"] * 2 * rand(R)).to(torch.int32)
            s["tp"] = torch.where(rand(R) < 0.3, torch.ones(R, device=DEV), case["tp"] * rand(R).sqrt())
            s["mp"] = case["mp"] * 2 * rand(R)
    return s


# ---------------------------------------------------------------- the plain forms

def _mulhilo(a, m):
    p = a * m  # modulo 2^64, the low and the high word of the product
    return (p >> 32) & U32, p & U32


def _plain_keep(seed, rows, d, p):
    """(rows, d) truth values: the elements that dropout keeps.

    Philox4x32-10 (Salmon et al., 2011) with the seed as its key and (column / 8,
    low word of the row, stream 0, high word of the row) as its counter; column
    8 b + 2 j + i takes half i of word j, and is kept from round(65536 p) on."""
    nb = (d + 7) // 8
    c0 = torch.arange(nb, device=DEV).expand(rows, nb)
    c1 = torch.arange(rows, device=DEV)[:, None].expand(rows, nb)
    c2 = torch.zeros_like(c0)
    c3 = torch.zeros_like(c0)
    k0, k1 = seed & U32, (seed >> 32) & U32
    for r in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & U32, (k1 + 0xBB67AE85) & U32
    words = torch.stack((c0, c1, c2, c3), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, nb * 8)[:, :d]
    return halves >= round(65536 * p)


def _scale(p):
    t = round(65536 * p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def _plain_norm(s):
    case = s["case"]
    x, w, b = (s[k].detach().float() for k in ("x", "w", "b"))
    h = x
    if case["gelu"]:
        cdf = 0.5 * torch.erfc(-x * math.sqrt(0.5))
        h = x * cdf
    c = h - h.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xh = c * r
    y = xh * w + b
    if case["p"]:
        keep = _plain_keep(s["seed"], case["rows"], case["d"], case["p"])
        y = torch.where(keep, y * _scale(case["p"]), 0.0)
    y = y.to(DTYPES[case["out"]])
    if not case["train"]:
        return y
    g = s["dy"].float()
    if case["p"]:
        g = torch.where(keep, g * _scale(case["p"]), 0.0)
    # sums over many rows in 64 bits
    db = g.sum(0, dtype=torch.float64).float()
    dw = (g * xh).sum(0, dtype=torch.float64).float()
    q = g * w
    dx = r * (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True))
    if case["gelu"]:
        dx = dx * (cdf + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi)))
    return [y, dx.to(s["x"].dtype), dw, db]


def _plain_drop(s):
    case = s["case"]
    keep = _plain_keep(s["seed"], case["rows"], case["d"], case["p"])
    y = torch.where(keep, s["x"].detach().float() * _scale(case["p"]), 0.0)
    dt = s["x"].dtype
    if s["res"] is not None:
        y = y + s["res"].float()
        dt = torch.promote_types(dt, s["res"].dtype)
    y = y.to(dt)
    if not case["train"]:
        return y
    return [y, torch.where(keep, s["dy"].float() * _scale(case["p"]), 0.0).to(s["x"].dtype)]


def _plain_sample(s):
    # in 64 bits: a draw next to the border of two tokens turns on the last bits
    lg, V = s["logits"].double(), s["logits"].shape[1]
    tok = s["tokens"]
    if tok is not None:
        lg = lg.gather(1, tok.long().clamp(0, V - 1)).masked_fill((tok < 0) | (tok >= V), -math.inf)
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    R, n = lg.shape

    def col(v):
        return v.double()[:, None] if torch.is_tensor(v) else torch.full((R, 1), float(v), dtype=torch.float64, device=DEV)

    T, k, tp, mp = (col(s[q]) for q in ("T", "k", "tp", "mp"))
    val, order = torch.sort(lg, dim=1, descending=True, stable=True)
    rank = torch.arange(n, device=DEV)[None]
    top = val[:, :1]
    w = torch.where(val == top, 1.0, torch.exp((val - top) / torch.where(T > 0, T, 1.0)))
    w = torch.where(val == -math.inf, 0.0, w)
    w = torch.where((T > 0) | (rank == 0), w, 0.0)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    cum = w.cumsum(1)
    before = torch.cat((torch.zeros_like(top), cum[:, :-1]), dim=1)
    keep = (rank == 0) | (((tp >= 1) | (before < tp * cum[:, -1:])) & (w >= mp))
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))
    cum = w.cumsum(1)
    total = cum[:, -1:]
    last = torch.where(w > 0, rank, 0).amax(1, keepdim=True)
    at = torch.minimum((cum <= s["u"].double()[:, None] * total).sum(1, keepdim=True), last)
    some = total > 0
    logp = torch.where(some, torch.log(w.gather(1, at) / total), -math.inf).float()
    ids = at if tok is None else tok.long().gather(1, at)
    return [torch.where(some, ids, -1).squeeze(1), logp.squeeze(1)]


# ---------------------------------------------------------------- one pass

def _own_norm(s):
    from redpanda_amd.layernorm import hip_layernorm
    case = s["case"]
    y = hip_layernorm(s["x"], s["w"], s["b"], EPS, gelu=case["gelu"], p=case["p"], seed=s["seed"],
                      out_dtype=DTYPES[case["out"]])
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])]


def _own_drop(s):
    from redpanda_amd.dropout import hip_dropout
    case = s["case"]
    y = hip_dropout(s["x"], case["p"], s["seed"], residual=s["res"])
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (s["x"],), s["dy"])]


def _own_sample(s):
    from redpanda_amd.sampling import hip_sample
    return list(hip_sample(s["logits"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["tp"],
                           min_p=s["mp"], tokens=s["tokens"], logprob=True))


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "drop": _own_drop, "sample": _own_sample}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "drop": _plain_drop, "sample": _plain_sample}[kind](state)


# ---------------------------------------------------------------- the work

def work(case):
    if case["kind"] == "sample":
        R, V, M = case["R"], case["V"], case["M"]
        b = DTYPES[case["dtype"]].itemsize
        # the row (or the list and its logits), u in; the token and its log-probability out
        n = M or V
        return dict(bytes=R * (n * (b + (4 if M else 0)) + 4 + 12 + (16 if case["each"] else 0)),
                    flops=R * n * 16)
    n, b, p = case["rows"] * case["d"], DTYPES[case["dtype"]].itemsize, case["p"] > 0
    # 10 rounds of 2 products and 4 exclusive ors per 8 elements
    mask = 8 if p else 0
    if case["kind"] == "norm":
        o, gelu = DTYPES[case["out"]].itemsize, 18 if case["gelu"] else 0
        nbytes, flops = n * (b + o) + 8 * case["d"], n * (8 + gelu + mask)
        if case["train"]:  # dy in, dx and the weights' gradients out; the input stays in hand
            nbytes, flops = nbytes + n * (b + o) + 8 * case["d"], flops + n * (16 + gelu + mask)
        return dict(bytes=nbytes, flops=flops)
    r = 0 if case["res"] == "none" else DTYPES[case["res"]].itemsize
    o = max(b, r)
    nbytes, flops = n * (b + r + o), n * (2 + mask)
    if case["train"]:
        nbytes, flops = nbytes + n * (o + b), flops + n * (1 + mask)
    return dict(bytes=nbytes, flops=flops)


# ---------------------------------------------------------------- in 64 bits

def _mask64(seed, rows, d, p):
    """The same mask, its products from 16-bit limbs."""
    key = int(seed.item())
    nb = -(-d // 8)
    blk = torch.arange(rows * nb, device=DEV)
    x = [blk % nb, blk // nb, 0 * blk, 0 * blk]

    def high(v, m):
        return ((v >> 16) * m + (((v & 0xFFFF) * m) >> 16)) >> 16

    def low(v, m):
        return ((((v >> 16) * m & 0xFFFF) << 16) + (v & 0xFFFF) * m) & U32

    for r in range(10):
        ka = ((key & U32) + r * 0x9E3779B9) & U32
        kb = ((key >> 32 & U32) + r * 0xBB67AE85) & U32
        x = [high(x[2], 0xCD9E8D57) ^ x[1] ^ ka, low(x[2], 0xCD9E8D57),
             high(x[0], 0xD2511F53) ^ x[3] ^ kb, low(x[0], 0xD2511F53)]
    out = torch.empty(rows * nb, 8, dtype=torch.bool, device=DEV)
    for j in range(8):
        out[:, j] = (x[j // 2] >> (16 * (j % 2))) % 65536 >= round(p * 65536)
    return out.view(rows, nb * 8)[:, :d]


def _sample64(s):
    lg = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    toks = None if s["tokens"] is None else s["tokens"].cpu().numpy()
    R, V = lg.shape

    def per_row(v):
        return v.double().cpu().numpy() if torch.is_tensor(v) else np.full(R, float(v))

    T, k, tp, mp = (per_row(s[q]) for q in ("T", "k", "tp", "mp"))
    ids, logp = np.full(R, -1, dtype=np.int64), np.full(R, -np.inf)
    for r in range(R):
        name = np.arange(V) if toks is None else toks[r].astype(np.int64)
        pos = np.flatnonzero((name >= 0) & (name < V))
        val = lg[r][name[pos]]
        fine = val > -np.inf  # false for NaN too
        pos, val = pos[fine], val[fine]
        if not len(pos):
            continue
        first = np.argsort(-val, kind="stable")
        if T[r] <= 0:
            ids[r], logp[r] = name[pos[first[0]]], 0.0
            continue
        if k[r] > 0:
            first = first[:int(k[r])]
        with np.errstate(invalid="ignore"):
            w = np.exp((val[first] - val[first[0]]) / T[r])
        w[val[first] == val[first[0]]] = 1.0
        n = len(w)
        if tp[r] < 1:
            run = np.cumsum(w)
            n = max(1, int(np.searchsorted(np.concatenate(([0.0], run[:-1])), tp[r] * run[-1], side="left")))
        n = max(1, min(n, int((w >= mp[r]).sum())))
        by_id = np.argsort(first[:n])
        w, at = w[:n][by_id], first[:n][by_id]
        run = np.cumsum(w)
        i = min(int(np.searchsorted(run, u[r] * run[-1], side="right")), n - 1)
        ids[r], logp[r] = name[pos[at[i]]], np.log(w[i] / run[-1])
    return [torch.from_numpy(ids), torch.from_numpy(logp)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _sample64(s)
    keep = _mask64(s["seed"], case["rows"], case["d"], case["p"]) if case["p"] else None
    up = 65536.0 / (65536 - round(case["p"] * 65536))
    x = s["x"].detach().double().requires_grad_(case["train"])
    if case["kind"] == "drop":
        y = torch.where(keep, x * up, torch.zeros_like(x))
        if s["res"] is not None:
            y = y + s["res"].double()
        ins = (x,)
    else:
        w, b = (s[k].detach().double().requires_grad_(case["train"]) for k in ("w", "b"))
        h = torch.nn.functional.gelu(x) if case["gelu"] else x
        y = torch.nn.functional.layer_norm(h, (case["d"],), w, b, EPS)
        if keep is not None:
            y = torch.where(keep, y * up, torch.zeros_like(y))
        ins = (x, w, b)
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, ins, s["dy"].double())]
