"""The head operators in the search model: training with dropout, and rollouts
drawn on the device, against the same steps from torch's ops and the
restatements in 64 bits."""

import pytest
import torch
import torch.nn.functional as F

from oracle import heads_ref as ref
from redpanda_amd.mamba import MambaConfig
from redpanda_amd.search_mamba import SearchMamba

pytestmark = pytest.mark.gpu
dev = "cuda"


def model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = MambaConfig(d_model=64, n_layer=2, d_state=12, n_track_state=4, vocab_size=96, mimo_p=2, **kw)
    return SearchMamba(cfg, vocab_size=96, eval_dim=32).to(dev)


def nrel(a, b):
    return float((a.double() - b.double()).abs().max() / (b.double().abs().max() + 1e-30))


def plain_head(head, h, p, seed, stream):
    x = F.gelu(head[0](h))
    x = F.layer_norm(x, x.shape[-1:], head[2].weight, head[2].bias, head[2].eps)
    keep = ref.keep_mask(range(x.shape[0]), x.shape[1], p, seed, stream).to(x.device)
    x = torch.where(keep, x * ref.drop_scale(p), torch.zeros_like(x))
    for m in head[3:]:
        x = m(x)
    return x


@pytest.mark.parametrize("seed_on_device", [False, True])
def test_dynamics_rollout_with_dropout(gpu_lib, seed_on_device):
    m = model()
    g = torch.Generator().manual_seed(1)
    board = torch.randint(0, 96, (5, 9), generator=g).to(dev)
    moves = torch.randint(0, 96, (5, 3), generator=g).to(dev)
    seed = torch.tensor([31], device=dev) if seed_on_device else 31
    v, c, f = m.dynamics_rollout(board, moves, dropout=0.25, seed=seed)
    (v.sum() + (c * c).mean() + f.sum()).backward()
    grads = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    m.zero_grad()
    # the same from torch's ops with the masks of the restatement
    _, cache = m.backbone.prime_cache(board)
    vs, cs, fs = [], [], []
    for t in range(3):
        h, cache = m.backbone.step(token_id=moves[:, t], cache=cache)
        vs.append(torch.tanh(plain_head(m.value_head, h, 0.25, 31, 2 * t)).squeeze(-1))
        cs.append(plain_head(m.continuation_head, h, 0.25, 31, 2 * t + 1))
        fs.append(m.consistency_proj(h))
    v2, c2, f2 = torch.stack(vs, 1), torch.stack(cs, 1), torch.stack(fs, 1)
    (v2.sum() + (c2 * c2).mean() + f2.sum()).backward()
    # a head's GELU and norm are a few hundred fp32 roundings either way
    assert nrel(v, v2) <= 1e-5 and nrel(c, c2) <= 1e-5 and torch.equal(f, f2)
    for n, p in m.named_parameters():
        if p.grad is not None:
            assert nrel(grads[n], p.grad) <= 1e-4, n


def test_without_dropout_nothing_changes(gpu_lib):
    m = model()
    board = torch.arange(8, device=dev).view(1, 8)
    moves = torch.arange(3, device=dev).view(1, 3)
    a = m.dynamics_rollout(board, moves)
    _, cache = m.backbone.prime_cache(board)
    for t in range(3):
        h, cache = m.backbone.step(token_id=moves[:, t], cache=cache)
        assert torch.equal(a[0][:, t], torch.tanh(m.value_head(h)).squeeze(-1))
        assert torch.equal(a[1][:, t], m.continuation_head(h))
    ids = torch.arange(12, device=dev).view(2, 6)
    assert torch.equal(m.backbone(ids), m.backbone(ids, dropout=0.0))


@pytest.mark.parametrize("checkpoint", [False, True])
def test_residual_dropout(gpu_lib, checkpoint):
    m = model(grad_checkpoint=checkpoint).backbone.train()
    ids = torch.arange(12, device=dev).view(2, 6)
    y = m(ids, dropout=0.2, seed=5)
    y.square().mean().backward()
    got = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    x = m.embedding(ids)
    for i, layer in enumerate(m.layers):
        keep = ref.keep_mask(range(12), 64, 0.2, 5, i).view(2, 6, 64).to(dev)
        out = layer["mixer"](layer["norm"](x))
        x = x + torch.where(keep, out * ref.drop_scale(0.2), torch.zeros_like(out))
    y2 = m.norm_f(x)
    y2.square().mean().backward()
    assert nrel(y, y2) <= 1e-6
    for n, p in m.named_parameters():
        assert nrel(got[n], p.grad) <= 1e-4, n


def test_sample_rollout(gpu_lib):
    """Tokens, log-probabilities and values of rollouts drawn on the device, ply by
    ply against the restatement on the same logits."""
    m = model(3)
    board = torch.arange(10)
    K, T = 7, 4
    u = torch.rand(T, K, generator=torch.Generator().manual_seed(2)).to(dev)
    g = torch.Generator().manual_seed(4)
    lists = [torch.stack([torch.randperm(96, generator=g)[:20].sort().values for _ in range(K)]).int().to(dev)
             for _ in range(T)]
    for t in range(T):
        lists[t][5, 3:] = -1
    lists[2][1] = -1  # rollout 1 ends at the third ply
    kw = dict(temperature=0.8, top_k=12, top_p=0.9, min_p=0.01)
    tok, logp, val = m.sample_rollout(board, u, legal=lambda t, last: lists[t], **kw)
    hidden, cache = m.prime_board(board.to(dev), compact=True)
    hidden, cache = hidden.expand(K, -1).contiguous(), m._expand_cache(cache, K)
    alive = [True] * K
    with torch.no_grad():
        for t in range(T):
            logits = m._fused_head(m.continuation_head, hidden)
            assert nrel(logits, m.continuation_head(hidden)) <= 1e-5
            ids, lp = ref.sample(logits.cpu().double().numpy(), u[t].cpu().double().numpy(), 0.8, 12, 0.9, 0.01,
                                 tokens=lists[t].cpu().numpy())
            alive = [a and i >= 0 for a, i in zip(alive, ids)]
            want = [i if a else -1 for a, i in zip(alive, ids)]
            assert tok[t].tolist() == want
            for a, x, y in zip(alive, logp[t].tolist(), lp):
                assert abs(x - y) <= 2.0 ** -24 * abs(y) + 1e-9 if a else x == -float("inf")
            hidden, cache = m.backbone.step(token_id=tok[t].clamp(min=0), cache=cache)
            v = torch.tanh(m.value_head(hidden)).squeeze(-1)
            live = torch.tensor(alive, device=dev)
            assert nrel(val[t][live], v[live]) <= 1e-5
    assert not alive[1] and float(val[3][1]) == float(val[1][1])


def test_under_autocast(gpu_lib):
    m = model(5)
    h = torch.randn(33, 64, device=dev)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        a = m._fused_head(m.continuation_head, h)
        b = m.continuation_head(h)
        ids, logp = m.sample_moves(h, torch.rand(33, device=dev), top_p=0.9)
    assert a.dtype == torch.bfloat16 and nrel(a.float(), b.float()) <= 3e-2
    assert bool((ids >= 0).all()) and bool(torch.isfinite(logp).all())


def test_stream_of_every_form_of_a_device(gpu_lib):
    from redpanda_amd import _lib
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for d in (torch.device("cuda", 0), torch.device("cuda"), "cuda", "cuda:0", 0, None):
            assert _lib.stream_of(d) == st.cuda_stream
