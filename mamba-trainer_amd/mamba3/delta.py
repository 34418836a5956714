"""A stack of gated delta rule blocks on the gfx950 kernels, bf16 activations
with the residual stream in f32:

    y = RMSNorm(r)                                   (block_norm of the block before)
    q, k, v, z, a, b, gate = in_proj(y)              (one product, read in place)
    g = -exp(a_log) softplus(a + dt_bias),  beta = sigmoid(b)
    o = delta_rule(q, k, v, g, beta)                 (a window) or delta_step_ (a token)
    x = out_proj(RMSNorm(o) * silu(z))
    r, y = block_norm(x, r, gate, ...)               (r += scale * silu(gate) * RMSNorm(x); the next norm)

Serving: `forward` over a padded batch of windows, `forward_cached` for windows
that continue and for single tokens, the states updated in place.  The same
operators train through torch's autograd (`ssm.delta_rule` and `nn.block_norm`
are differentiable).  No reference counterpart (its mixer is Mamba-3's); the
projections and norms are those of the Mamba-3 stack (models/hybrid.rs:446-456).
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import math
from typing import List, Optional

import torch

from . import _lib
from .error import ConfigError, ShapeError
from .nn import Linear, RmsNorm, _bf16_dev, _stream, block_norm, normal, residual_scaled
from .ssm.delta import DeltaInputs, delta_rule, delta_step_


@dataclasses.dataclass
class GatedDeltaConfig:
    d_model: int = 768
    n_layers: int = 12
    n_heads: int = 12
    n_groups: int = 12            # heads / groups consecutive heads share q and k
    head_dim: int = 64
    d_state: int = 128
    block_gate: bool = True       # a silu gate on each block's normed output
    norm_eps: float = 1e-5
    int8_weights: bool = False
    seed: int = 0

    def validate(self) -> None:
        if min(self.d_model, self.n_layers, self.n_heads, self.n_groups, self.head_dim, self.d_state) <= 0:
            raise ConfigError("invalid configuration: delta stack dimensions must all be positive")
        if self.n_heads % self.n_groups != 0:
            raise ConfigError(f"invalid configuration: n_heads ({self.n_heads}) must be a multiple of "
                              f"n_groups ({self.n_groups})")

    def d_inner(self) -> int:
        return self.n_heads * self.head_dim

    def columns(self):
        """Widths of in_proj's pieces, in order; the row is padded to a multiple of eight."""
        qk = self.n_groups * self.d_state
        cols = dict(q=qk, k=qk, v=self.d_inner(), z=self.d_inner(),
                    gate=self.d_model if self.block_gate else 0, a=self.n_heads, b=self.n_heads)
        cols["pad"] = -sum(cols.values()) % 8
        return cols


class GatedDeltaMixer:
    """in_proj, the delta rule, its normed gate, out_proj."""

    def __init__(self, cfg: GatedDeltaConfig, *, device, gen: torch.Generator):
        cfg.validate()
        self.cfg, self.cols = cfg, cfg.columns()
        self.in_proj = Linear(normal((cfg.d_model, sum(self.cols.values())), 0.02, device, gen),
                              int8_weights=cfg.int8_weights)
        self.out_proj = Linear(residual_scaled((cfg.d_inner(), cfg.d_model), 0.02, cfg.n_layers, device, gen),
                               int8_weights=cfg.int8_weights)
        self.norm = RmsNorm(cfg.d_inner(), device, eps=cfg.norm_eps)
        # softplus(dt_bias) log-uniform over 0.001 .. 0.1, decay rates over 1 .. 16, as the Mamba-3 mixer's
        u = torch.rand((2, cfg.n_heads), generator=gen, device=device)
        dt = torch.exp(math.log(1e-3) + u[0] * math.log(100.0))
        self.dt_bias = (dt + torch.log(-torch.expm1(-dt))).float()
        self.a_log = torch.log(1.0 + 15.0 * u[1]).float()

    def _pieces(self, x: torch.Tensor):
        rows = self.in_proj.apply(x)
        at, out = 0, {}
        for name, width in self.cols.items():
            out[name] = rows[..., at:at + width]
            at += width
        return out

    def _gates(self, p):
        shape = p["a"].shape
        g = torch.empty(shape, dtype=torch.float32, device=p["a"].device)
        beta = torch.empty_like(g)
        n = g.numel() // shape[-1]
        _lib.check(_lib.lib().m3_delta_gates(n, shape[-1], _lib.M3_BF16, p["a"].data_ptr(), p["b"].data_ptr(),
                                             sum(self.cols.values()), self.a_log.data_ptr(),
                                             self.dt_bias.data_ptr(), g.data_ptr(), beta.data_ptr(), _stream(g)))
        return g, beta

    def _finish(self, y: torch.Tensor, p) -> torch.Tensor:
        d = self.cfg.d_inner()
        out = torch.empty(tuple(y.shape[:-2]) + (d,), dtype=torch.bfloat16, device=y.device)
        _lib.check(_lib.lib().m3_mixer_gate(out.numel() // d, d, y.data_ptr(), p["z"].data_ptr(),
                                            sum(self.cols.values()), self.norm.weight.data_ptr(),
                                            C.c_float(self.norm.eps), out.data_ptr(), _stream(y)))
        return self.out_proj.apply(out)

    def apply(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
              lengths: Optional[torch.Tensor] = None):
        """x [B, T, d_model] -> (output, the block gate's columns or None, the state after)."""
        c = self.cfg
        x = _bf16_dev(x, "delta mixer input")
        if x.dim() != 3 or x.shape[2] != c.d_model:
            raise ShapeError(f"shape error: GatedDeltaMixer expects [batch, seq, {c.d_model}], got {tuple(x.shape)}")
        p = self._pieces(x)
        g, beta = self._gates(p)
        q, k = (p[n].unflatten(-1, (c.n_groups, c.d_state)) for n in ("q", "k"))
        v = p["v"].unflatten(-1, (c.n_heads, c.head_dim))
        gate = p["gate"] if c.block_gate else None
        if x.shape[1] == 1 and state is not None:
            y = delta_step_(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state, qk_norm=True, lengths=lengths)
            return self._finish(y.unsqueeze(1), p), gate, state
        inputs = DeltaInputs(q, k, v, g, beta).with_qk_norm(True)
        inputs.state, inputs.lengths = state, lengths
        out = delta_rule(inputs)
        return self._finish(out.y, p), gate, out.state


class GatedDeltaStack:
    """n_layers of [GatedDeltaMixer -> block_norm] over f32 residual rows."""

    def __init__(self, cfg: GatedDeltaConfig, device):
        cfg.validate()
        self.cfg = cfg
        gen = torch.Generator(device=device)
        gen.manual_seed(cfg.seed)
        self.mixers = [GatedDeltaMixer(cfg, device=device, gen=gen) for _ in range(cfg.n_layers)]
        ones = lambda: torch.ones(cfg.d_model, dtype=torch.float32, device=device)
        self.norms = [RmsNorm(cfg.d_model, device, eps=cfg.norm_eps) for _ in range(cfg.n_layers + 1)]
        self.post = [ones() for _ in range(cfg.n_layers)]
        self.scale = [ones() / math.sqrt(2.0 * cfg.n_layers) for _ in range(cfg.n_layers)]

    def empty_cache(self, batch: int, device) -> List[torch.Tensor]:
        c = self.cfg
        return [torch.zeros((batch, c.n_heads, c.head_dim, c.d_state), dtype=torch.float32, device=device)
                for _ in self.mixers]

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [B, T, d_model] bf16 -> the normed output; lengths [B]: tokens past them are padding."""
        return self._run(x, None, lengths)

    def forward_cached(self, x: torch.Tensor, cache: List[torch.Tensor],
                       lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """A window or one token, each layer's state updated in place in `cache` (a
        sequence of length 0 keeps its state)."""
        if len(cache) != len(self.mixers):
            raise ConfigError(f"invalid configuration: cache has {len(cache)} entries but the stack has "
                              f"{len(self.mixers)} layers")
        return self._run(x, cache, lengths)

    def _run(self, x, cache, lengths):
        y, r = self.norms[0].apply(x), x.float()
        for i, mixer in enumerate(self.mixers):
            out, gate, state = mixer.apply(y, None if cache is None else cache[i], lengths)
            if cache is not None and state is not cache[i]:
                cache[i].copy_(state)
            r, y = block_norm(out, r, post_weight=self.post[i], gate=gate, scale=self.scale[i],
                              pre_weight=self.norms[i + 1].weight, eps=self.cfg.norm_eps)
        return y
