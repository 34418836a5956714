"""Layers around the scan, over the C ABI of mamba3_mixer.h (bf16 activations).

Mirrors the reference's `nn` items the Mamba-3 language model uses:
RmsNorm (src/nn/norm.rs:17-105), Linear with an optional int8 weight fake
quantizer (src/nn/linear.rs:40-185, src/nn/quant.rs:95-103, 231-330), Embedding
(src/nn/embedding.rs) and the initialisers (src/nn/init.rs:90-110).  Weights
are held on the device; every computation runs in libmamba3_hip.so.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import math
from typing import Optional

import torch

from . import _lib
from ._lib import stream_of as _stream
from .error import ArgumentError, ShapeError, UnsupportedError


def _bf16_dev(t: torch.Tensor, what: str) -> torch.Tensor:
    if not t.is_cuda:
        raise ArgumentError(f"{what} must be a ROCm device tensor (there is no CPU path)")
    if t.dtype != torch.bfloat16:
        raise ArgumentError(f"{what} must be bfloat16, got {t.dtype}")
    return t.contiguous()


def as_written(obj, cls, name: str) -> bool:
    """Whether obj.<name> is the method of cls itself, which a call past it may
    stand for: no subclass's, none set on the object, no other object's."""
    return getattr(type(obj), name, None) is getattr(cls, name) and name not in vars(obj)


def normal(shape, std: float, device, gen: torch.Generator) -> torch.Tensor:
    """Initializer::Normal {mean 0, std} (init.rs:98-100)."""
    return torch.randn(shape, device=device, generator=gen, dtype=torch.float32) * std


def residual_scaled(shape, std: float, n_layers: int, device, gen: torch.Generator) -> torch.Tensor:
    """Initializer::ResidualScaled: std / sqrt(2 * n_layers) (init.rs:105-108)."""
    return normal(shape, std / math.sqrt(2.0 * max(n_layers, 1)), device, gen)


def tensor_param(owner, attr: str):
    """A checkpoint Param over an f32 device tensor held as `owner.<attr>`."""
    from .checkpoint import Param
    t = getattr(owner, attr)
    return Param(tuple(t.shape), lambda: getattr(owner, attr),
                 lambda v: getattr(owner, attr).copy_(v.to(torch.float32)))


_WS = {}


def linear_workspace(device) -> torch.Tensor:
    """The scratch m3_linear may use (one per device; stream-ordered use)."""
    key = (device.type, device.index)
    ws = _WS.get(key)
    if ws is None:
        ws = torch.empty(int(_lib.lib().m3_linear_workspace_bytes()), dtype=torch.uint8,
                         device=device)
        _WS[key] = ws
    return ws


class RmsNorm:
    """norm.rs:70-105: y = x * rsqrt(mean(x^2) + eps) * w over the last axis."""

    def __init__(self, dim: int, device, eps: float = 1e-5, weight: bool = True):
        self.dim, self.eps = dim, eps
        self.weight = torch.ones(dim, dtype=torch.float32, device=device) if weight else None

    def apply(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        x = _bf16_dev(x, "RmsNorm input")
        if x.shape[-1] != self.dim:
            raise ShapeError(f"shape error: RmsNorm expects a trailing dimension of {self.dim}, "
                             f"got {tuple(x.shape)}")
        y = torch.empty_like(x) if out is None else out
        rows = x.numel() // self.dim
        _lib.check(_lib.lib().m3_rms_norm(rows, self.dim, x.data_ptr(), self.dim,
                                          None if self.weight is None else self.weight.data_ptr(),
                                          C.c_float(self.eps), y.data_ptr(), self.dim, _stream(x)))
        return y


class Linear:
    """linear.rs:40-185 for bf16 activations: y = x @ w, w stored
    [in_features, out_features] as in the reference (no bias term).

    With `int8_weights` (QuantConfig::int8_weights, quant.rs:95-103) the weight
    used is the fake-quantized w' = code * scale (per output channel); the
    codes go to the GEMM as exact bf16 and the scales are applied in its
    epilogue, so w' is never rounded to bf16.  Without it the weight is used
    as bf16.  The GEMM operand is held transposed, codes_t [out, in]
    (m3_linear_nt); `codes` is its [in, out] view.
    """

    def __init__(self, weight: torch.Tensor, int8_weights: bool = False,
                 bias: Optional[torch.Tensor] = None):
        if weight.dim() != 2:
            raise ShapeError(f"shape error: a Linear weight is [in, out], got {tuple(weight.shape)}")
        if bias is not None:
            # SsmConfig::bias is false for the projections of every model here
            raise UnsupportedError("unsupported: Linear bias is not on the gfx950 path")
        self.weight = weight.float().contiguous()          # master copy, f32
        self.int8_weights = int8_weights
        self.codes: Optional[torch.Tensor] = None
        self.codes_t: Optional[torch.Tensor] = None
        self.scales: Optional[torch.Tensor] = None
        self.prepare()

    @property
    def in_features(self) -> int:
        return self.weight.shape[0]

    @property
    def out_features(self) -> int:
        return self.weight.shape[1]

    def prepare(self) -> None:
        """Derive the GEMM operands from the master weight (after any update)."""
        k, n = self.weight.shape
        if self.int8_weights:
            codes = torch.empty((k, n), dtype=torch.bfloat16, device=self.weight.device)
            self.scales = torch.empty(n, dtype=torch.float32, device=self.weight.device)
            _lib.check(_lib.lib().m3_quantize_int8_columns(
                k, n, self.weight.data_ptr(), codes.data_ptr(), self.scales.data_ptr(),
                _stream(self.weight)))
        else:
            codes = self.weight.to(torch.bfloat16)
            self.scales = None
        self.codes_t = codes.t().contiguous()
        self.codes = self.codes_t.t()

    def param(self):
        """The master weight [in, out] as a checkpoint Param; setting it
        re-derives the GEMM operands (codes and scales)."""
        from .checkpoint import Param

        def put(v):
            self.weight.copy_(v.to(torch.float32))
            self.prepare()
        return Param(tuple(self.weight.shape), lambda: self.weight, put)

    def effective_weight(self) -> torch.Tensor:
        """The weight the product uses, in f32 (w' for the quantized form)."""
        if self.scales is None:
            return self.codes.float()
        return self.codes.float() * self.scales

    def apply(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [..., in] -> [..., out]; `residual` [..., out] is added (it may be `out`)."""
        x = _bf16_dev(x, "Linear input")
        if x.shape[-1] != self.in_features:
            raise ShapeError(f"shape error: Linear expects a trailing dimension of "
                             f"{self.in_features}, got {tuple(x.shape)}")
        m = x.numel() // self.in_features
        shape = tuple(x.shape[:-1]) + (self.out_features,)
        y = torch.empty(shape, dtype=torch.bfloat16, device=x.device) if out is None else out
        if residual is not None:
            residual = _bf16_dev(residual, "Linear residual")
        ws = linear_workspace(x.device)
        _lib.check(_lib.lib().m3_linear_nt(
            m, self.in_features, self.out_features, x.data_ptr(), self.codes_t.data_ptr(),
            None if self.scales is None else self.scales.data_ptr(),
            None if residual is None else residual.data_ptr(), y.data_ptr(), ws.data_ptr(),
            ws.numel(), _stream(x)))
        return y

    def apply_normed(self, x: torch.Tensor, norm: RmsNorm) -> torch.Tensor:
        """apply(norm.apply(x)): for the few rows of a decode step in one
        launch (m3_norm_linear_nt), whose operand is rounded to bf16 before the
        row's factor instead of after it; elsewhere as two calls."""
        x = _bf16_dev(x, "Linear input")
        m = x.numel() // max(x.shape[-1], 1)
        if (m <= 4 and as_written(self, Linear, "apply") and as_written(norm, RmsNorm, "apply")
                and x.shape[-1] == self.in_features == norm.dim):
            y = torch.empty(tuple(x.shape[:-1]) + (self.out_features,), dtype=torch.bfloat16,
                            device=x.device)
            st = _lib.lib().m3_norm_linear_nt(
                m, self.in_features, self.out_features, x.data_ptr(),
                None if norm.weight is None else norm.weight.data_ptr(), C.c_float(norm.eps),
                self.codes_t.data_ptr(), None if self.scales is None else self.scales.data_ptr(),
                None, y.data_ptr(), _stream(x))
            if st != _lib.M3_ERR_UNSUPPORTED:
                _lib.check(st)
                return y
        return self.apply(norm.apply(x))


def linear_normed(linear, x: torch.Tensor, norm) -> torch.Tensor:
    """linear.apply(norm.apply(x)), in one launch where `linear` is a Linear."""
    if isinstance(linear, Linear):
        return linear.apply_normed(x, norm)
    return linear.apply(norm.apply(x))


_TYPES = {torch.float32: _lib.M3_F32, torch.bfloat16: _lib.M3_BF16, torch.float16: _lib.M3_F16}
_ACTIVATIONS = {"none": 0, "silu": 1, "sigmoid": 2}


def _gate_rows(gate: torch.Tensor):
    """A gate read in place: (tensor, elements between its rows).  Rows that are
    evenly spaced and contiguous (columns of a projection) stay where they
    are; anything else is copied."""
    dim = gate.shape[-1]
    if gate.is_contiguous() or gate.dim() < 2:
        return gate.contiguous(), dim
    stride = want = gate.stride(-2)
    ok = gate.stride(-1) == 1 and stride >= dim
    for size, st in zip(reversed(gate.shape[:-1]), reversed(gate.stride()[:-1])):
        ok = ok and (size == 1 or st == want)
        want *= size
    return (gate, stride) if ok else (gate.contiguous(), dim)


def _block_norm_args(x, residual, post_weight, gate, scale, pre_weight, eps, activation, post_norm):
    """The checked arguments of m3_block_norm, and the tensors they point into."""
    dev = x.get_device()
    if dev < 0:
        raise ArgumentError(f"x must be a ROCm device tensor (got {x.device}); there is no CPU path")
    code = _TYPES.get(x.dtype)
    if code is None:
        raise UnsupportedError(f"unsupported: storage dtype {x.dtype}; use float32, bfloat16 or float16")
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ArgumentError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    shape = x.shape
    if len(shape) == 0:
        raise ShapeError("shape error: a block norm takes rows, got a scalar")
    dim = shape[-1]
    if residual.shape != shape:
        raise ShapeError(f"shape error: residual has shape {list(residual.shape)}, expected "
                         f"{list(shape)}")
    if residual.dtype != x.dtype and residual.dtype != torch.float32:
        raise UnsupportedError("unsupported: the residual stream is in x's type or in float32, got "
                               f"{residual.dtype}")
    if residual.get_device() != dev:
        raise ArgumentError(f"residual is on {residual.device}, x on {x.device}")
    x, residual = x.contiguous(), residual.contiguous()
    gate_stride, gate_ptr = dim, None
    if gate is not None:
        if gate.dtype != x.dtype or gate.shape != shape:
            raise ShapeError(f"shape error: gate is {gate.dtype} {list(gate.shape)}, expected {x.dtype} "
                             f"{list(shape)}")
        if gate.get_device() != dev:
            raise ArgumentError(f"gate is on {gate.device}, x on {x.device}")
        gate, gate_stride = _gate_rows(gate)
        gate_ptr = gate.data_ptr()
    weights, ptrs = [], []
    for t, what in ((post_weight, "post_weight"), (scale, "scale"), (pre_weight, "pre_weight")):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != dim:
                raise ShapeError(f"shape error: {what} has shape {list(t.shape)}, expected [{dim}]")
            if t.get_device() != dev:
                raise ArgumentError(f"{what} is on {t.device}, x on {x.device}")
            if t.dtype != torch.float32 or not t.is_contiguous():
                t = t.float().contiguous()
        weights.append(t)
        ptrs.append(None if t is None else t.data_ptr())
    args = _lib.BlockNormC(x.numel() // dim if dim else 0, dim, code, _TYPES[residual.dtype],
                           1 if post_norm else 0, act, eps, x.data_ptr(), residual.data_ptr(), gate_ptr,
                           gate_stride, *ptrs)
    return args, (x, residual, gate, *weights)


def block_norm(x: torch.Tensor, residual: torch.Tensor, *, post_weight=None, gate=None, scale=None,
               pre_weight=None, eps: float = 1e-5, activation: str = "silu", post_norm: bool = True,
               normed: bool = True):
    """What stands between two blocks, in one pass over the rows: with
    n = RMSNorm(x) * post_weight (n = x without post_norm),

        residual' = residual + scale * act(gate) * n
        y = RMSNorm(residual') * pre_weight

    Returns (residual', y); y is None without `normed`.  x, gate and y share a
    type; residual and residual' have x's or float32.  Weights are f32 [dim]
    and may be None (ones); gate None is no gate, activation "none" a plain
    factor.  A gate whose rows are columns of a wider row is read in place.
    Differentiable."""
    tensors = (x, residual, gate, post_weight, scale, pre_weight)
    if torch.is_grad_enabled() and (
            x.requires_grad or residual.requires_grad
            or (gate is not None and gate.requires_grad)
            or (post_weight is not None and post_weight.requires_grad)
            or (scale is not None and scale.requires_grad)
            or (pre_weight is not None and pre_weight.requires_grad)):
        r, y = _BlockNormFn.apply((eps, activation, post_norm, normed), *tensors)
        return r, y
    return _block_norm_forward(tensors, eps, activation, post_norm, normed)


def _block_norm_forward(tensors, eps, activation, post_norm, normed):
    x, residual, gate, post_weight, scale, pre_weight = tensors
    args, keep = _block_norm_args(x, residual, post_weight, gate, scale, pre_weight, eps, activation,
                                  post_norm)
    x, residual = keep[0], keep[1]
    r = torch.empty_like(residual)
    y = torch.empty_like(x) if normed else None
    _lib.check(_lib.lib().m3_block_norm(C.byref(args), r.data_ptr(), None if y is None else y.data_ptr(),
                                        _stream(x)))
    return r, y


@dataclasses.dataclass
class BlockNormGrads:
    """Gradients of block_norm's inputs (None where the input is absent)."""
    x: torch.Tensor
    residual: torch.Tensor
    gate: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    scale: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]


def block_norm_backward(x, residual, dresidual, dy, *, post_weight=None, gate=None, scale=None,
                        pre_weight=None, eps: float = 1e-5, activation: str = "silu",
                        post_norm: bool = True) -> BlockNormGrads:
    """Gradients of block_norm for dL/dresidual' = dresidual and dL/dy = dy
    (either may be None: zero)."""
    args, keep = _block_norm_args(x, residual, post_weight, gate, scale, pre_weight, eps, activation,
                                  post_norm)
    x, residual, gate = keep[:3]
    douts = []
    for t, like, what in ((dresidual, residual, "dresidual"), (dy, x, "dy")):
        if t is not None:
            if t.device != x.device:
                raise ArgumentError(f"{what} is on {t.device}, x on {x.device}")
            if tuple(t.shape) != tuple(like.shape):
                raise ShapeError(f"shape error: {what} has shape {list(t.shape)}, expected "
                                 f"{list(like.shape)}")
            t = t.to(like.dtype).contiguous()
        douts.append(t)
    new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=x.device)
    g = BlockNormGrads(new(x), new(residual), new(gate), *(new(t) for t in keep[3:]))
    need = int(_lib.lib().m3_block_norm_backward_workspace_bytes(C.byref(args)))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
    ptr = lambda t: None if t is None else t.data_ptr()
    gc = _lib.BlockNormGradsC(ptr(douts[0]), ptr(douts[1]), *(ptr(t) for t in (
        g.x, g.residual, g.gate, g.post_weight, g.scale, g.pre_weight)))
    _lib.check(_lib.lib().m3_block_norm_backward(C.byref(args), C.byref(gc), ws.data_ptr(), ws.numel(),
                                                 _stream(x)))
    return g


class _BlockNormFn(torch.autograd.Function):
    """block_norm as one differentiable node."""

    @staticmethod
    def forward(ctx, cfg, *tensors):
        ctx.cfg = cfg
        ctx.save_for_backward(*tensors)
        ctx.set_materialize_grads(False)
        return _block_norm_forward(tensors, *cfg)

    @staticmethod
    def backward(ctx, dres, dy):
        x, residual, gate, post_weight, scale, pre_weight = ctx.saved_tensors
        eps, activation, post_norm, _ = ctx.cfg
        g = block_norm_backward(x, residual, dres, dy, post_weight=post_weight, gate=gate, scale=scale,
                                pre_weight=pre_weight, eps=eps, activation=activation,
                                post_norm=post_norm)
        out = (g.x, g.residual, g.gate, g.post_weight, g.scale, g.pre_weight)
        return (None, *(None if t is None else d.to(t.dtype) for t, d in zip(ctx.saved_tensors, out)))


class Embedding:
    """embedding.rs: a [vocab, dim] table (Normal std 0.02), bf16 rows."""

    def __init__(self, table: torch.Tensor):
        self.table = table.to(torch.bfloat16).contiguous()

    @property
    def vocab(self) -> int:
        return self.table.shape[0]

    @property
    def dim(self) -> int:
        return self.table.shape[1]

    def param(self):
        """The table as a checkpoint Param: read as f32, stored back as bf16
        (round to nearest even, as the reference's from_f32 for bf16)."""
        from .checkpoint import Param
        return Param(tuple(self.table.shape), lambda: self.table.float(),
                     lambda v: self.table.copy_(v.to(torch.float32).to(torch.bfloat16)))

    def lookup(self, ids: torch.Tensor) -> torch.Tensor:
        if not ids.is_cuda:
            raise ArgumentError("ids must be a ROCm device tensor (there is no CPU path)")
        ids32 = ids.to(torch.int32).contiguous()
        out = torch.empty(tuple(ids.shape) + (self.dim,), dtype=torch.bfloat16, device=ids.device)
        _lib.check(_lib.lib().m3_embedding_lookup(ids32.numel(), self.dim, ids32.data_ptr(),
                                                  self.vocab, self.table.data_ptr(),
                                                  out.data_ptr(), _stream(ids32)))
        return out
