"""What the gated delta rule and the block norm refuse, before any device work (no GPU needed: the
pointers are stand-ins that are never dereferenced)."""
import ctypes as C

import pytest
import torch

FAKE = 1 << 20


def delta_args(**kw):
    from mamba3 import _lib
    base = dict(batch=2, seq=8, heads=4, groups=2, head_dim=16, d_state=32, dtype=_lib.M3_BF16, q=FAKE, k=FAKE,
                v=FAKE, q_stride=0, k_stride=0, v_stride=0, g=FAKE, beta=FAKE, lengths=None, state=None, scale=1.0,
                qk_norm=0, workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.DeltaInputsC(**base)


@pytest.mark.parametrize("kw,status,message", [
    (dict(groups=3), 1, "n_heads (4) must be a multiple of n_groups (3)"),
    (dict(heads=0), 1, "must all be positive"),
    (dict(d_state=0), 1, "must all be positive"),
    (dict(head_dim=1025), 4, "head_dim up to 1024"),
    (dict(d_state=257), 4, "d_state up to 256"),
    (dict(batch=1 << 20, seq=1 << 20), 4, "must stay below 2^31"),
    (dict(dtype=7), 6, "unknown dtype"),
    (dict(q_stride=63), 2, "shorter than the rows"),
    (dict(v_stride=63), 2, "shorter than the rows"),
    (dict(k=None), 6, "q, k, v, g and beta are required"),
])
def test_delta_rule_refusals(kw, status, message):
    from mamba3 import _lib
    L = _lib.lib()
    before = L.m3_launch_count()
    cin = delta_args(**kw)
    grads = _lib.DeltaGradsC(*([FAKE] * 7), None)
    for st in (L.m3_delta_rule(C.byref(cin), FAKE, None, None),
               L.m3_delta_rule_backward(C.byref(cin), C.byref(grads), None)):
        assert st == status, L.m3_last_error()
        assert message in L.m3_last_error().decode()
    assert L.m3_launch_count() == before


def test_delta_gates_refusals():
    from mamba3 import _lib
    L = _lib.lib()
    call = lambda rows, heads, dt, stride, a: L.m3_delta_gates(rows, heads, dt, a, FAKE, stride, FAKE, None, FAKE, FAKE, None)
    assert call(4, 0, 1, 8, FAKE) == _lib.M3_ERR_CONFIG
    assert call(4, 4, 5, 8, FAKE) == _lib.M3_ERR_ARGUMENT
    assert call(4, 9, 1, 8, FAKE) == _lib.M3_ERR_SHAPE
    assert call(1 << 31, 4, 1, 8, FAKE) == _lib.M3_ERR_UNSUPPORTED
    assert call(4, 4, 1, 8, None) == _lib.M3_ERR_ARGUMENT
    assert call(0, 4, 1, 8, None) == _lib.M3_OK


def test_delta_rule_buffers():
    from mamba3 import _lib
    L = _lib.lib()
    cin = delta_args()
    assert L.m3_delta_rule(C.byref(cin), None, None, None) == _lib.M3_ERR_ARGUMENT
    assert L.m3_delta_rule(None, FAKE, None, None) == _lib.M3_ERR_ARGUMENT
    assert L.m3_delta_step(C.byref(cin), FAKE, FAKE, None) == _lib.M3_ERR_SHAPE        # seq 8
    one = delta_args(seq=1)
    assert L.m3_delta_step(C.byref(one), None, FAKE, None) == _lib.M3_ERR_ARGUMENT
    grads = _lib.DeltaGradsC(*([FAKE] * 7), None)
    assert L.m3_delta_rule_backward(C.byref(cin), None, None) == _lib.M3_ERR_ARGUMENT
    assert L.m3_delta_rule_backward(C.byref(cin), C.byref(grads), None) == _lib.M3_ERR_ARGUMENT   # no workspace
    assert b"workspace holds 0 bytes" in L.m3_last_error()
    need = L.m3_delta_rule_backward_workspace_bytes(C.byref(cin))
    assert need > 0
    off = delta_args(workspace=FAKE + 16, workspace_bytes=need)
    assert L.m3_delta_rule_backward(C.byref(off), C.byref(grads), None) == _lib.M3_ERR_ARGUMENT
    assert b"256-byte aligned" in L.m3_last_error()
    grads.dstate0 = FAKE                                                               # without a state
    assert L.m3_delta_rule_backward(C.byref(cin), C.byref(grads), None) == _lib.M3_ERR_ARGUMENT
    # an empty batch asks for nothing
    assert L.m3_delta_rule(C.byref(delta_args(batch=0, q=None)), None, None, None) == _lib.M3_OK
    assert L.m3_delta_rule_workspace_bytes(C.byref(delta_args(groups=3))) == 0


def test_delta_python_refusals():
    from mamba3 import ArgumentError, RankError, ShapeError, UnsupportedError
    from mamba3.ssm import DeltaInputs, delta_rule, delta_step_
    q, v, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 6), torch.zeros(1, 4, 2)
    with pytest.raises(ArgumentError, match="no CPU path"):
        delta_rule(DeltaInputs(q, q, v, g, g))
    with pytest.raises(RankError):
        delta_rule(DeltaInputs(q[0], q, v, g, g))
    with pytest.raises(RankError):
        delta_rule(DeltaInputs(q, q, v[0], g, g))
    with pytest.raises(ShapeError):
        delta_rule(DeltaInputs(q[:, :3], q, v, g, g))
    with pytest.raises(UnsupportedError):
        delta_rule(DeltaInputs(q.double(), q.double(), v.double(), g, g))
    with pytest.raises(RankError):
        delta_step_(q, q, v, g, g, torch.zeros(1, 2, 6, 8))


def norm_args(**kw):
    from mamba3 import _lib
    base = dict(rows=4, dim=64, dtype=_lib.M3_BF16, residual_dtype=_lib.M3_F32, post_norm=1, activation=1, eps=1e-5,
                x=FAKE, residual=FAKE, gate=FAKE, gate_stride=64, post_weight=None, scale=None, pre_weight=None)
    base.update(kw)
    return _lib.BlockNormC(**base)


@pytest.mark.parametrize("kw,status,message", [
    (dict(dim=0), 2, "empty axis"),
    (dict(dim=32769), 4, "rows of up to 32768 values"),
    (dict(rows=1 << 31), 4, "below 2^31"),
    (dict(dtype=9), 6, "unknown dtype"),
    (dict(residual_dtype=2), 4, "in x's type or in f32"),
    (dict(activation=3), 6, "unknown gate activation"),
    (dict(eps=-1.0), 1, "eps must be non-negative"),
    (dict(eps=float("nan")), 1, "eps must be non-negative"),
    (dict(gate_stride=63), 2, "shorter than the row"),
    (dict(x=None), 6, "x and residual are required"),
])
def test_block_norm_refusals(kw, status, message):
    from mamba3 import _lib
    L = _lib.lib()
    before = L.m3_launch_count()
    a = norm_args(**kw)
    g = _lib.BlockNormGradsC(*([FAKE] * 8))
    for st in (L.m3_block_norm(C.byref(a), FAKE, FAKE, None),
               L.m3_block_norm_backward(C.byref(a), C.byref(g), FAKE, 1 << 40, None)):
        assert st == status, L.m3_last_error()
        assert message in L.m3_last_error().decode()
    assert L.m3_launch_count() == before


def test_block_norm_buffers():
    from mamba3 import _lib
    L = _lib.lib()
    a = norm_args()
    g = _lib.BlockNormGradsC(*([FAKE] * 8))
    assert L.m3_block_norm(C.byref(a), None, FAKE, None) == _lib.M3_ERR_ARGUMENT
    need = L.m3_block_norm_backward_workspace_bytes(C.byref(a))
    assert need >= 4 * 3 * 64
    assert L.m3_block_norm_backward(C.byref(a), C.byref(g), FAKE, need - 1, None) == _lib.M3_ERR_ARGUMENT
    assert L.m3_block_norm_backward(C.byref(a), None, FAKE, need, None) == _lib.M3_ERR_ARGUMENT
    g.dgate = None
    assert L.m3_block_norm_backward(C.byref(a), C.byref(g), FAKE, need, None) == _lib.M3_ERR_ARGUMENT
    assert L.m3_block_norm(C.byref(norm_args(rows=0, x=None)), None, None, None) == _lib.M3_OK


def test_block_norm_python_refusals():
    from mamba3 import ArgumentError
    from mamba3.nn import block_norm
    x = torch.zeros(2, 8)
    with pytest.raises(ArgumentError, match="no CPU path"):
        block_norm(x, x)
