"""The gated delta rule on the gfx950 kernels (include/mamba3_delta.h): a
recurrent mixer on the scan's state layout, S [B, H, P, N] in f32,

    S~ = exp(g_t) S_{t-1};  u_t = beta_t (v_t - S~ k_t)
    S_t = S~ + u_t k_t^T;   y_t = scale S_t q_t

over a window (`delta_rule`, differentiable) and one token at a time in place
(`delta_step_`).  As in `ssm.scan`, torch tensors are device buffers only; there
is no CPU path.  No reference counterpart: its mixers add outer products only.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _lib
from .._lib import stream_of as _stream
from ..error import ArgumentError, RankError, ShapeError
from .scan import _dtype_code, _expect_shape, _f32, _ptr


class DeltaInputs:
    """q, k [B, T, G, N] and v [B, T, H, P] in one type (H a multiple of G: a
    group's heads share its q and k), g (log decay, at most 0) and beta (write
    strength) [B, T, H] in f32.  q, k and v may be columns of wider rows, one
    row a token (a projection's output): they are read in place."""

    def __init__(self, q, k, v, g, beta):
        self.q, self.k, self.v, self.g, self.beta = q, k, v, g, beta
        self.state: Optional[torch.Tensor] = None
        self.lengths: Optional[torch.Tensor] = None
        self.scale: Optional[float] = None
        self.qk_norm = False
        self.want_state = True

    def with_state(self, state: torch.Tensor):
        """S before the window, f32 [B, H, P, N] (default: zeros)."""
        self.state = state
        return self

    def with_lengths(self, lengths: torch.Tensor):
        """Valid tokens of each sequence, int32 [B] on the device; tokens past
        them are padding: not used, y and gradients zero."""
        self.lengths = lengths
        return self

    def with_scale(self, scale: float):
        """Factor of y (default d_state ** -0.5)."""
        self.scale = scale
        return self

    def with_qk_norm(self, qk_norm: bool):
        """Bring each q and k to unit length first: x rsqrt(sum x^2 + 1e-6)."""
        self.qk_norm = qk_norm
        return self

    def with_state_output(self, want_state: bool):
        self.want_state = want_state
        return self


@dataclass
class DeltaOutput:
    y: torch.Tensor                   # [B, T, H, P]
    state: Optional[torch.Tensor]     # S after the window [B, H, P, N], f32


@dataclass
class DeltaGrads:
    """Gradients of delta_rule's inputs (h0: of the state before the window)."""
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    g: torch.Tensor
    beta: torch.Tensor
    h0: Optional[torch.Tensor]


def _rows(t: torch.Tensor, tokens: int, heads: int, width: int):
    """(tensor, elements between tokens) of a [B, T, heads, width] tensor, or of
    [B, heads, width] for one token a sequence: in place where its tokens' rows
    are contiguous and evenly spaced, else a contiguous copy."""
    row = heads * width
    if t.is_contiguous():
        return t, row
    st = t.stride()
    batch = t.shape[0]
    ok = (width == 1 or st[-1] == 1) and (heads == 1 or st[-2] == width)
    if tokens == 1:           # a token's spacing is the sequence's
        step = st[0] if batch > 1 else row
    else:
        step = st[1]
        ok = ok and (batch == 1 or st[0] == tokens * step)
    if not ok or step < row or t.numel() == 0:
        return t.contiguous(), row
    return t, step


def _args(inputs: DeltaInputs, step: bool = False):
    """The checked m3_delta_inputs, the tensors it points into, and (B, T, H, P, N, G).
    step: the tensors are of one token a sequence, without the T axis."""
    q, k, v, g, beta = inputs.q, inputs.k, inputs.v, inputs.g, inputs.beta
    rank = 3 if step else 4
    for t in (v, q, k):
        if t.dim() != rank:
            raise RankError(rank, t.dim(), t.shape)
    shape = v.shape
    B, H, P = shape[0], shape[-2], shape[-1]
    T = 1 if step else shape[1]
    G, N = k.shape[-2], k.shape[-1]
    code = _dtype_code(v)
    lead = (B,) if step else (B, T)
    dev = v.get_device()
    for t, what in ((q, "q"), (k, "k")):
        _expect_shape(t, lead + (G, N), what)
        if t.dtype != v.dtype or t.get_device() != dev:
            raise ShapeError(f"shape error: {what} is {t.dtype} on {t.device} but v is {v.dtype} on "
                             f"{v.device}")
    if dev < 0:
        raise ArgumentError(f"v must be a ROCm device tensor (got {v.device}); "
                            "the delta rule has no CPU path")
    v, vs = _rows(v, T, H, P)
    q, qs = _rows(q, T, G, N)
    k, ks = _rows(k, T, G, N)
    g, beta = _f32(g, "g"), _f32(beta, "beta")
    _expect_shape(g, lead + (H,), "g")
    _expect_shape(beta, lead + (H,), "beta")
    lengths, h0 = inputs.lengths, _f32(inputs.state, "state")
    if lengths is not None:
        _expect_shape(lengths, (B,), "lengths")
        if not lengths.is_cuda:
            raise ArgumentError("lengths must be a ROCm device tensor")
        lengths = lengths.to(torch.int32).contiguous()
    if h0 is not None:
        _expect_shape(h0, (B, H, P, N), "state")
    for t, what in ((g, "g"), (beta, "beta"), (lengths, "lengths"), (h0, "state")):
        if t is not None and t.get_device() != dev:
            raise ArgumentError(f"{what} is on {t.device}, v on {v.device}")
    scale = inputs.scale
    if scale is None:
        scale = N ** -0.5 if N > 0 else 0.0
    cin = _lib.DeltaInputsC(B, T, H, G, P, N, code, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks,
                            vs, g.data_ptr(), beta.data_ptr(),
                            None if lengths is None else lengths.data_ptr(),
                            None if h0 is None else h0.data_ptr(), scale, 1 if inputs.qk_norm else 0)
    return cin, (q, k, v, g, beta, lengths, h0), (B, T, H, P, N, G)


def _workspace(cin, need: int, device):
    """A workspace from torch's stream-ordered allocator, set in cin."""
    if need == 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    cin.workspace, cin.workspace_bytes = ws.data_ptr(), need
    return ws


def _forward(inputs: DeltaInputs) -> DeltaOutput:
    cin, keep, (B, T, H, P, N, _) = _args(inputs)
    v = keep[2]
    y = torch.empty((B, T, H, P), dtype=v.dtype, device=v.device)
    state = (torch.empty((B, H, P, N), dtype=torch.float32, device=v.device)
             if inputs.want_state else None)
    ws = _workspace(cin, int(_lib.lib().m3_delta_rule_workspace_bytes(C.byref(cin))), v.device)   # noqa: F841
    _lib.check(_lib.lib().m3_delta_rule(C.byref(cin), y.data_ptr(), _ptr(state), _stream(v)))
    return DeltaOutput(y, state)


def delta_rule(inputs: DeltaInputs) -> DeltaOutput:
    """The gated delta rule over a window; differentiable (the backward is
    m3_delta_rule_backward)."""
    tensors = (inputs.q, inputs.k, inputs.v, inputs.g, inputs.beta, inputs.state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        cfg = (inputs.lengths, inputs.scale, inputs.qk_norm, inputs.want_state)
        y, state = _DeltaFn.apply(cfg, *tensors)
        return DeltaOutput(y, state)
    return _forward(inputs)


def _inputs_of(cfg, q, k, v, g, beta, state) -> DeltaInputs:
    di = DeltaInputs(q, k, v, g, beta)
    di.state = state
    di.lengths, di.scale, di.qk_norm, di.want_state = cfg
    return di


class _DeltaFn(torch.autograd.Function):
    """delta_rule as one differentiable node."""

    @staticmethod
    def forward(ctx, cfg, *tensors):
        out = _forward(_inputs_of(cfg, *tensors))
        ctx.cfg = cfg
        ctx.save_for_backward(*tensors)
        ctx.set_materialize_grads(False)
        return out.y, out.state

    @staticmethod
    def backward(ctx, dy, dstate):
        tensors = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(tensors[2])
        d = delta_rule_backward(_inputs_of(ctx.cfg, *tensors), dy, dstate)
        grads = (d.q, d.k, d.v, d.g, d.beta, d.h0)
        return (None, *(None if t is None else g.to(t.dtype) for t, g in zip(tensors, grads)))


def delta_rule_backward(inputs: DeltaInputs, dy: torch.Tensor,
                        dstate: Optional[torch.Tensor] = None) -> DeltaGrads:
    """Gradients of delta_rule for dL/dy = dy (and dL/dstate of the state after
    the window)."""
    cin, keep, (B, T, H, P, N, G) = _args(inputs)
    v, h0 = keep[2], keep[6]
    if not dy.is_cuda or dy.device != v.device:
        raise ArgumentError(f"dy must be on {v.device} (got {dy.device})")
    _expect_shape(dy, (B, T, H, P), "dy")
    dy = dy.to(v.dtype).contiguous()
    dstate = _f32(dstate, "dstate")
    if dstate is not None:
        _expect_shape(dstate, (B, H, P, N), "dstate")
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=v.device)
    d = DeltaGrads(new(B, T, G, N, dtype=v.dtype), new(B, T, G, N, dtype=v.dtype),
                   new(B, T, H, P, dtype=v.dtype), new(B, T, H), new(B, T, H),
                   None if h0 is None else new(B, H, P, N))
    gc = _lib.DeltaGradsC(dy.data_ptr(), _ptr(dstate), d.q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(),
                          d.g.data_ptr(), d.beta.data_ptr(), _ptr(d.h0))
    ws = _workspace(cin, int(_lib.lib().m3_delta_rule_backward_workspace_bytes(C.byref(cin))),   # noqa: F841
                    v.device)
    _lib.check(_lib.lib().m3_delta_rule_backward(C.byref(cin), C.byref(gc), _stream(v)))
    return d


def delta_step_(q, k, v, g, beta, state: torch.Tensor, *, scale: Optional[float] = None,
                qk_norm: bool = False, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token a sequence: q, k [B, G, N], v [B, H, P], g, beta [B, H]; `state`
    [B, H, P, N] (f32) is updated IN PLACE; returns y [B, H, P].  A sequence
    whose lengths entry is 0 keeps its state (an empty slot of a batch)."""
    inputs = DeltaInputs(q, k, v, g, beta)
    inputs.scale, inputs.qk_norm, inputs.lengths = scale, qk_norm, lengths
    cin, keep, (B, _, H, P, N, _) = _args(inputs, step=True)
    v = keep[2]
    if (state.dtype != torch.float32 or not state.is_contiguous()
            or state.get_device() != v.get_device()):
        raise ArgumentError(f"state must be a contiguous float32 tensor on {v.device}")
    _expect_shape(state, (B, H, P, N), "state")
    y = v.new_empty((B, H, P))
    _lib.check(_lib.lib().m3_delta_step(C.byref(cin), state.data_ptr(), y.data_ptr(), _stream(v)))
    return y
