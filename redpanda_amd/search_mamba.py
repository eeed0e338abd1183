"""Search Mamba: the causal rollout model MARS advances with O(1) steps.

API- and state_dict-compatible with the reference's engine/search_mamba.py
(SearchMambaConfig :24-36, SearchMamba :39-384) over the HIP backbone in
redpanda_amd.mamba: prime_board (one causal scan returning the cache, on the
HIP scan kernel), _expand_cache, eval_step / backbone.step (the fused step
kernel), dynamics_rollout (trains through step via the scan kernel's analytic
backward), and the line-evaluation helpers.  The heads are plain torch
modules with the reference's names and init; the paths that the reference does
not have (dropout in dynamics_rollout, sample_moves, sample_rollout) run their
middle, GELU and layer norm, in one kernel, with dropout and sampling from
given random numbers on the device.
"""

import json
from dataclasses import asdict
from dataclasses import fields as dc_fields

import torch
import torch.nn as nn

from redpanda_amd.layernorm import hip_layernorm
from redpanda_amd.mamba import Mamba, MambaConfig
from redpanda_amd.sampling import hip_sample


class SearchMambaConfig(MambaConfig):
    """engine/search_mamba.py:24-36.  Deliberately NOT re-decorated as a
    dataclass, like the reference: the generated __init__ is MambaConfig's,
    so an instance built without arguments carries MambaConfig's defaults
    (d_model 512, 16 layers, d_state 64, mimo_p 4), and the class-level
    values below only show through attribute lookup on the class."""
    d_model: int = 384
    n_layer: int = 12
    d_state: int = 32
    expand: int = 2
    use_complex: bool = True
    mimo_p: int = 2
    use_bcnorm: bool = True


class SearchMamba(nn.Module):
    """Causal value-equivalent dynamics model (engine/search_mamba.py:39-384)."""

    def __init__(self, config: SearchMambaConfig = None, vocab_size: int = 8192,
                 eval_dim: int = 512):
        super().__init__()
        if config is None:
            config = SearchMambaConfig(vocab_size=vocab_size)
        config.bidirectional = False  # the rollout model must be causal
        self.config = config
        self.eval_dim = eval_dim
        self.backbone = Mamba(config)
        d = config.d_model
        self.line_value_head = nn.Sequential(
            nn.Linear(d, d), nn.GELU(), nn.LayerNorm(d),
            nn.Linear(d, d // 2), nn.GELU(), nn.Linear(d // 2, 1))
        self.value_head = nn.Sequential(
            nn.Linear(d, d), nn.GELU(), nn.LayerNorm(d), nn.Linear(d, 1))
        self.continuation_head = nn.Sequential(
            nn.Linear(d, d * 2), nn.GELU(), nn.LayerNorm(d * 2),
            nn.Linear(d * 2, config.vocab_size))
        self.consistency_proj = nn.Sequential(
            nn.Linear(d, d), nn.GELU(), nn.Linear(d, eval_dim))
        self.apply(self._init_weights)

    def _init_weights(self, m):
        if isinstance(m, nn.Linear):
            nn.init.orthogonal_(m.weight, gain=1.0)
            if m.bias is not None:
                nn.init.constant_(m.bias, 0)

    def _device(self):
        return next(self.parameters()).device

    # ── whole-sequence scoring (one causal scan per line) ──

    def forward(self, board_encoding, move_sequences):
        """(B, L_board) + (B, L_moves) token ids -> (B,) line scores."""
        hidden = self.backbone(torch.cat([board_encoding, move_sequences], dim=-1))
        return self.line_value_head(hidden[:, -1, :]).squeeze(-1)

    def evaluate_lines(self, board_encoding, move_sequences):
        if board_encoding.dim() == 1:
            board_encoding = board_encoding.unsqueeze(0)
        k = move_sequences.shape[0]
        return self.forward(board_encoding.expand(k, -1), move_sequences)

    def evaluate_with_continuation(self, board_encoding, move_sequences):
        if board_encoding.dim() == 1:
            board_encoding = board_encoding.unsqueeze(0)
        k = move_sequences.shape[0]
        full = torch.cat([board_encoding.expand(k, -1), move_sequences], dim=-1)
        final = self.backbone(full)[:, -1, :]
        return self.line_value_head(final).squeeze(-1), self.continuation_head(final)

    # ── O(1) cached evaluation ──

    def prime_board(self, board_encoding, compact=False):
        """Encode one board (ids (L,) or (1, L), list or tensor) and return
        (final_hidden, cache) for step() (engine/search_mamba.py:162-175).
        compact=True keeps each layer's beta in rank-1 rows [dt*u | B]
        (half the state bytes per step; same results)."""
        if not torch.is_tensor(board_encoding):
            board_encoding = torch.as_tensor(board_encoding, dtype=torch.long,
                                             device=self._device())
        if board_encoding.dim() == 1:
            board_encoding = board_encoding.unsqueeze(0)
        return self.backbone.prime_cache(board_encoding, compact=compact)

    @staticmethod
    def _expand_cache(cache, k):
        """Broadcast a batch-1 cache to k rows (engine/search_mamba.py:177-187).

        The reference materialises k copies (expand().contiguous()); here the
        rows are stride-0 views of the one state, which the step kernel reads
        in place, and every step returns fresh per-row states.  Callers that
        clone or concatenate the cache get contiguous tensors as before; an
        in-place write into the returned views is not supported (torch
        rejects it)."""
        return [(h.expand(k, *h.shape[1:]), b.expand(k, *b.shape[1:])) for h, b in cache]

    @torch.no_grad()
    def evaluate_lines_fast(self, board_encoding, move_sequences, lengths=None):
        """K lines from one board: prime once, then step every line in lockstep."""
        device = self._device()
        _, cache = self.prime_board(board_encoding.to(device))
        k, L = move_sequences.shape
        move_sequences = move_sequences.to(device)
        cache = self._expand_cache(cache, k)
        hiddens = []
        for t in range(L):
            hidden, cache = self.backbone.step(token_id=move_sequences[:, t], cache=cache)
            hiddens.append(hidden)
        hiddens = torch.stack(hiddens, dim=1)
        if lengths is not None:
            idx = (lengths.to(device).clamp(min=1) - 1).view(k, 1, 1).expand(-1, 1, hiddens.shape[-1])
            final = hiddens.gather(1, idx).squeeze(1)
        else:
            final = hiddens[:, -1, :]
        return self.line_value_head(final).squeeze(-1)

    @torch.no_grad()
    def score_branch(self, board_cache, move_sequence):
        device = self._device()
        cache = self._expand_cache(board_cache, 1)
        hidden = None
        for tok in move_sequence:
            hidden, cache = self.backbone.step(
                token_id=torch.tensor([int(tok)], device=device), cache=cache)
        quality = self.line_value_head(hidden).squeeze(-1)
        return quality.item(), self.continuation_head(hidden).squeeze(0)

    @staticmethod
    def _fused_head(head, h, dropout=0.0, seed=None, stream=0):
        """A head's Linear -> GELU -> LayerNorm [-> dropout] -> rest, GELU, norm
        and dropout in one pass; the norm's result in the first Linear's dtype
        (fp32, or the autocast dtype that the next Linear takes)."""
        x, norm = head[0](h), head[2]
        x = hip_layernorm(x, norm.weight, norm.bias, norm.eps, gelu=True, p=dropout, seed=seed,
                          stream=stream)
        for m in head[3:]:
            x = m(x)
        return x

    def dynamics_rollout(self, board_encoding, move_tokens, dropout=0.0, seed=None):
        """Differentiable: prime on (B, L_board), step through (B, T) moves;
        returns per-step values (B, T), continuation logits (B, T, vocab) and
        consistency features (B, T, eval_dim) (engine/search_mamba.py:252-273).

        dropout > 0 (training): the value and the continuation head drop out
        behind their norms, with masks of `seed` (an int, or an int64 tensor of
        one element on the device, which a captured step reads on each replay)
        that no pass stores; step t draws streams 2 t and 2 t + 1, so that a call
        takes a seed of its own beside the backbone's (whose layers draw streams
        from 0 on).  It drops wherever it is asked to: self.training is not looked
        at."""
        _, cache = self.backbone.prime_cache(board_encoding)
        vs, cs, fs = [], [], []
        for t in range(move_tokens.shape[1]):
            h, cache = self.backbone.step(token_id=move_tokens[:, t], cache=cache)
            if dropout:
                v = self._fused_head(self.value_head, h, dropout, seed, 2 * t)
                c = self._fused_head(self.continuation_head, h, dropout, seed, 2 * t + 1)
            else:
                v, c = self.value_head(h), self.continuation_head(h)
            vs.append(torch.tanh(v).squeeze(-1))
            cs.append(c)
            fs.append(self.consistency_proj(h))
        return torch.stack(vs, 1), torch.stack(cs, 1), torch.stack(fs, 1)

    @torch.no_grad()
    def sample_moves(self, hidden, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """The next move of every rollout, drawn from the continuation head:
        (token ids (R,) int64, their log-probabilities (R,)).  hidden (R,
        d_model); u (R,) uniform numbers; legal: None or (R, M) ids padded with
        -1, the moves to draw among (their logits alone are read); the settings
        as in hip_sample.  -1 for a rollout without a move.  The reference draws
        on the host from the top candidates (engine/mars_search.py:261-276)."""
        logits = self._fused_head(self.continuation_head, hidden)
        return hip_sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                          tokens=legal, logprob=True)

    @torch.no_grad()
    def sample_rollout(self, board_encoding, u, legal=None, compact=True, **settings):
        """K rollouts of T plies from one board, on the device from end to end:
        u (T, K) uniform numbers -> tokens (T, K) int64, log-probabilities
        (T, K), values (T, K) of the states the moves lead to.  legal: None, or a
        function of (ply, the tokens before it or None) that gives the ply's (K,
        M) legal ids padded with -1.  A rollout without a move ends: its tokens
        are -1 from there on, its value stays (the board's own before the first
        move).  settings: hip_sample's."""
        T, k = u.shape
        hidden, cache = self.prime_board(board_encoding.to(self._device()), compact=compact)
        value = torch.tanh(self._fused_head(self.value_head, hidden)).squeeze(-1).expand(k)
        hidden, cache = hidden.expand(k, -1).contiguous(), self._expand_cache(cache, k)
        tokens, logps, values, alive = [], [], [], None
        for t in range(T):
            moves = None if legal is None else legal(t, tokens[-1] if tokens else None)
            ids, logp = self.sample_moves(hidden, u[t], moves, **settings)
            alive = ids >= 0 if alive is None else alive & (ids >= 0)
            ids = torch.where(alive, ids, -1)
            # an ended rollout steps on with token 0, unseen
            hidden, cache = self.backbone.step(token_id=ids.clamp(min=0), cache=cache)
            v = torch.tanh(self._fused_head(self.value_head, hidden)).squeeze(-1)
            value = torch.where(alive, v, value)
            tokens.append(ids)
            logps.append(torch.where(alive, logp, float("-inf")))
            values.append(value)
        if T == 0:
            return (u.new_empty((0, k), dtype=torch.int64), u.new_empty((0, k), dtype=torch.float32),
                    value.new_empty((0, k)))
        return torch.stack(tokens), torch.stack(logps), torch.stack(values)

    @torch.no_grad()
    def eval_step(self, cache, move_token):
        """One O(1) node evaluation: (value, continuation logits, new cache)."""
        tok = torch.tensor([int(move_token)], device=self._device())
        h, cache = self.backbone.step(token_id=tok, cache=cache)
        value = torch.tanh(self.value_head(h)).squeeze(-1).item()
        return value, self.continuation_head(h).squeeze(0), cache

    # ── checkpoints: state_dict + JSON config, loaded with weights_only=True ──

    @staticmethod
    def _config_path(path):
        cp = path.replace(".pt", "_config.json").replace(".pth", "_config.json")
        return path + ".config.json" if cp == path else cp

    def save_pretrained(self, path):
        torch.save(self.state_dict(), path)
        cfg = asdict(self.config)
        cfg["eval_dim"] = self.eval_dim
        with open(self._config_path(path), "w") as fh:
            json.dump(cfg, fh, indent=2)

    @classmethod
    def from_pretrained(cls, path, device="cpu", config=None):
        eval_dim = 512
        if config is None:
            with open(cls._config_path(path)) as fh:
                cfg = json.load(fh)
            eval_dim = int(cfg.get("eval_dim", 512))
            valid = {f.name for f in dc_fields(SearchMambaConfig)}
            config = SearchMambaConfig(**{k: v for k, v in cfg.items() if k in valid})
        model = cls(config, eval_dim=eval_dim)
        model.load_state_dict(torch.load(path, map_location=device, weights_only=True))
        return model

