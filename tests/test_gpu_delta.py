"""The gated delta rule (m3_delta_rule, m3_delta_step, m3_delta_rule_backward) on the GPU against its
64-bit restatement, where it can go wrong: lengths around the chunk, shapes that fill no tile, shared
key heads, carried states, padding that holds NaN, decays that end a state, strides, streams."""
import pytest
import torch

import delta_cases as dc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def run(c):
    from mamba3.ssm import delta_rule
    out = delta_rule(dc.inputs_of(c))
    torch.cuda.synchronize()
    return out.y, out.state


def check_forward(c):
    y, s = run(c)
    yo, so = dc.oracle(c)
    dc.check(y, yo, "y")
    dc.check(s, so, "state")


def check_backward(c):
    from mamba3.ssm import delta_rule_backward
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    torch.cuda.synchronize()
    _, _, want = dc.oracle_grads(c)
    size = dc.unit_sizes(c) if c["k"].shape[-1] == 1 else {}
    for n in dc.NAMES:
        if want[n] is None:
            assert getattr(d, n) is None
        else:
            dc.check(getattr(d, n), want[n], "d" + n, size.get(n, 0.0))


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("T", [1, 2, 17, 63, 64, 65, 128, 200])
def test_lengths_around_a_chunk(T, dtype):
    check_forward(dc.make(T, 2, T, 2, 2, 64, 128, dtype))
    check_backward(dc.make(T + 1000, 2, T, 2, 2, 64, 128, dtype))


@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("P,N", [(64, 64), (16, 16), (48, 96), (128, 32), (24, 40), (7, 5), (1, 1), (65, 127),
                                 (200, 128), (64, 100)])
def test_head_shapes(P, N, dtype):
    for T, carried in ((9, True), (130, False)):
        check_forward(dc.make(P * 1000 + N, 1, T, 2, 1, P, N, dtype, carried=carried))
        check_backward(dc.make(P * 1000 + N, 1, T, 2, 1, P, N, dtype, carried=carried))


@pytest.mark.parametrize("P,N", [(64, 256), (33, 130), (300, 64)])
def test_wide_heads_forward(P, N):
    check_forward(dc.make(5, 1, 70, 2, 1, P, N, BF))


@pytest.mark.parametrize("H,G", [(4, 1), (6, 3), (5, 5), (8, 2)])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_shared_key_heads(H, G, qk_norm):
    for dtype in (BF, FL):
        c = dc.make(H, 2, 100, H, G, 32, 64, dtype, qk_norm=qk_norm)
        check_forward(c)
        check_backward(c)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_padding_is_not_read(dtype):
    """Sequences of 150, 64, 1 and 0 valid tokens whose padding holds NaN and infinities: results and
    gradients as without the padding, zeros there, the empty sequence's state untouched."""
    c = dc.make(3, 4, 150, 4, 2, 48, 64, dtype, lengths=[150, 64, 1, 0])
    clean = dict(c)
    for n in ("q", "k", "v", "g", "beta", "dy"):
        t = c[n].clone()
        bad = torch.tensor([float("nan"), float("inf"), float("-inf")], device=DEV)
        for b, m in enumerate([150, 64, 1, 0]):
            pad = t[b, m:]
            pad.copy_(bad.to(t.dtype).repeat(pad.numel() // 3 + 1)[:pad.numel()].view(pad.shape))
        clean[n], c[n] = c[n], t
    y, s = run(c)
    yo, so = dc.oracle(clean)
    dc.check(y, yo, "y")
    dc.check(s, so, "state")
    assert torch.equal(s[3], c["h0"][3])
    from mamba3.ssm import delta_rule_backward
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    _, _, want = dc.oracle_grads({**clean, "dy": torch.where(
        (torch.arange(150, device=DEV)[None] < c["lengths"][:, None])[..., None, None], clean["dy"], 0)})
    for n in dc.NAMES:
        dc.check(getattr(d, n), want[n], "d" + n)
        if n != "h0":
            for b, m in enumerate([150, 64, 1, 0]):
                assert (getattr(d, n)[b, m:] == 0).all(), n
    assert torch.equal(d.h0[3], c["dh"][3])


def test_lengths_are_clamped():
    c = dc.make(4, 3, 70, 2, 2, 16, 32, BF, lengths=[1000, -5, 70])
    check_forward(c)
    check_backward(c)


@pytest.mark.parametrize("dtype", [BF, FL])
def test_decays_that_end_a_state(dtype):
    """-inf (a new document), the type's lowest value, and zero among ordinary log decays."""
    c = dc.make(5, 2, 140, 2, 2, 32, 64, dtype)
    c["g"][0, 10] = c["g"][1, 64] = c["g"][0, 0] = float("-inf")
    c["g"][0, 70:73] = torch.finfo(torch.float32).min
    c["g"][1, 20:30] = 0.0
    c["g"][1, 100] = -95.0
    check_forward(c)
    from mamba3.ssm import delta_rule_backward
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    # the oracle differentiates exp there: finite stand-ins with the same (zero) decay
    _, _, want = dc.oracle_grads({**c, "g": c["g"].clamp(min=-800.0)})
    for n in dc.NAMES:
        dc.check(getattr(d, n), want[n], "d" + n)


@pytest.mark.parametrize("dtype", [BF, FL])
def test_hard_keys(dtype):
    """The same key for all tokens of a chunk with full write strength (the inverse's largest
    entries), zero keys, and write strengths of 0 and up to 2."""
    c = dc.make(6, 2, 128, 2, 2, 32, 64, dtype, decay=(1e-4, 1e-2))
    c["k"][0] = c["k"][0, :1]
    c["beta"][0] = 1.0
    c["k"][1, 30:40] = 0.0
    c["beta"][1, :20] = 0.0
    c["beta"][1, 60:] = 2 * c["beta"][1, 60:]
    check_forward(c)
    check_backward(c)


def test_empty_windows():
    from mamba3.ssm import delta_rule, delta_rule_backward
    c = dc.make(7, 2, 0, 2, 2, 16, 32, BF)
    out = delta_rule(dc.inputs_of(c))
    assert out.y.shape == (2, 0, 2, 16) and torch.equal(out.state, c["h0"])
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    assert torch.equal(d.h0, c["dh"]) and d.q.shape == (2, 0, 2, 32)
    c = dc.make(8, 0, 5, 2, 2, 16, 32, BF)
    assert delta_rule(dc.inputs_of(c)).y.shape == (0, 5, 2, 16)
    c = dc.make(8, 2, 0, 2, 2, 16, 32, BF, carried=False)
    assert (delta_rule(dc.inputs_of(c)).state == 0).all()


def packed(c, extra=0):
    """The case's q, k, v as columns of one row per token, `extra` elements more between rows."""
    B, T, H, P = c["v"].shape
    G, N = c["k"].shape[2:]
    w = 2 * G * N + H * P
    rows = torch.empty((B, T, w + extra), dtype=c["v"].dtype, device=DEV)
    rows[..., :w] = torch.cat([c[n].flatten(2) for n in ("q", "k", "v")], -1)
    q, k, v = rows[..., :w].split([G * N, G * N, H * P], -1)
    return {**c, "q": q.unflatten(-1, (G, N)), "k": k.unflatten(-1, (G, N)), "v": v.unflatten(-1, (H, P))}


@pytest.mark.parametrize("extra", [0, 8, 3])
@pytest.mark.parametrize("T", [1, 6, 90])
def test_columns_of_a_projection(T, extra):
    """Read in place at the row's stride (3 more elements: no row 16-byte aligned), bit for bit as
    contiguous copies; so are the gradients."""
    from mamba3.ssm import delta_rule_backward
    c = dc.make(9, 3, T, 4, 2, 32, 64, BF, lengths=None)
    p = packed(c, extra)
    for a, b in zip(run(c), run(p)):
        assert torch.equal(a, b)
    x, y = (delta_rule_backward(dc.inputs_of(z), z["dy"], z["dh"]) for z in (c, p))
    for n in dc.NAMES:
        assert torch.equal(getattr(x, n), getattr(y, n)), n


def test_other_orders_are_copied():
    """Transposed, expanded and sliced inputs."""
    c = dc.make(10, 2, 40, 3, 3, 32, 32, FL)
    want = run(c)
    t = dict(c)
    t["q"] = c["q"].transpose(1, 2).contiguous().transpose(1, 2)
    t["k"] = c["k"].transpose(2, 3).contiguous().transpose(2, 3)
    t["v"] = torch.stack([c["v"], c["v"]], -1)[..., 0]
    t["g"] = c["g"].transpose(0, 1).contiguous().transpose(0, 1)
    for a, b in zip(want, run(t)):
        assert torch.equal(a, b)
    e = dict(c, beta=torch.full((1,), 0.5, device=DEV).expand(2, 40, 3))
    for a, b in zip(run(dict(c, beta=torch.full((2, 40, 3), 0.5, device=DEV))), run(e)):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows so far apart that element and byte offsets pass 32 bits."""
    B, T, G, N = 1, 70, 2, 64
    stride = (5 << 30) // (2 * T) // 8 * 8 * 2     # 5 Gi elements over the window
    c = dc.make(11, B, T, G, G, 16, N, BF)
    big = torch.empty(T * stride, dtype=BF, device=DEV)
    k = big.as_strided((B, T, G, N), (T * stride, stride, N, 1))
    k.copy_(c["k"])
    a, b = run(c), run(dict(c, k=k))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("B,H,G,P,N", [(1, 24, 24, 64, 128), (3, 4, 2, 64, 64), (70, 8, 8, 64, 128), (2, 2, 1, 7, 5),
                                       (2, 3, 3, 130, 256), (5, 2, 2, 24, 40)])
def test_step(B, H, G, P, N, dtype):
    from mamba3.ssm import delta_step_
    c = dc.make(B, B, 3, H, G, P, N, dtype)
    yo, so = dc.oracle(c)
    s = c["h0"].clone()
    where = s.data_ptr()
    ys = [delta_step_(*(c[n][:, t] for n in ("q", "k", "v", "g", "beta")), s, qk_norm=True) for t in range(3)]
    dc.check(torch.stack(ys, 1), yo, "y")
    dc.check(s, so, "state")
    assert s.data_ptr() == where


def test_step_leaves_empty_slots():
    from mamba3.ssm import delta_step_
    c = dc.make(12, 4, 1, 2, 2, 64, 128, BF)
    n = torch.tensor([1, 0, 1, 0], dtype=torch.int32, device=DEV)
    s = c["h0"].clone()
    a = [c[x][:, 0].clone() for x in ("q", "k", "v", "g", "beta")]
    for t in a:
        t[1::2] = float("nan")
    y = delta_step_(*a, s, qk_norm=True, lengths=n)
    assert torch.equal(s[1::2], c["h0"][1::2]) and (y[1::2] == 0).all()
    yo, so = dc.oracle(c)
    dc.check(y[::2], yo[::2, 0], "y")
    dc.check(s[::2], so[::2], "state")


def test_window_equals_steps():
    """A window and its tokens one by one agree to rounding, and two windows chained through the
    state are one."""
    from mamba3.ssm import DeltaInputs, delta_rule, delta_step_
    c = dc.make(13, 2, 150, 4, 4, 64, 128, FL)
    y, s = run(c)
    st = c["h0"].clone()
    ys = torch.stack([delta_step_(*(c[n][:, t] for n in ("q", "k", "v", "g", "beta")), st, qk_norm=True)
                      for t in range(150)], 1)
    dc.check(ys, y.double().cpu(), "y")
    dc.check(st, s.double().cpu(), "state")
    cut = lambda a, b: [c[n][:, a:b] for n in ("q", "k", "v", "g", "beta")]
    one = delta_rule(DeltaInputs(*cut(0, 67)).with_qk_norm(True).with_state(c["h0"]))
    two = delta_rule(DeltaInputs(*cut(67, 150)).with_qk_norm(True).with_state(one.state))
    dc.check(torch.cat([one.y, two.y], 1), y.double().cpu(), "y")
    dc.check(two.state, s.double().cpu(), "state")


def test_autograd_and_options():
    """The differentiable call: gradients of every input, without a state output, a given scale, and
    two windows chained through the state."""
    from mamba3.ssm import DeltaInputs, delta_rule
    c = dc.make(14, 2, 90, 4, 2, 32, 64, FL)
    leaves = {n: c[n].clone().requires_grad_() for n in dc.NAMES}
    a = [leaves[n] for n in ("q", "k", "v", "g", "beta")]
    one = delta_rule(DeltaInputs(*(t[:, :40] for t in a)).with_qk_norm(True).with_state(leaves["h0"]))
    two = delta_rule(DeltaInputs(*(t[:, 40:] for t in a)).with_qk_norm(True).with_state(one.state))
    y = torch.cat([one.y, two.y], 1)
    ((y * c["dy"]).sum() + (two.state * c["dh"]).sum()).backward()
    _, _, want = dc.oracle_grads(c)
    for n in dc.NAMES:
        dc.check(leaves[n].grad, want[n], "d" + n)
    out = delta_rule(dc.inputs_of(c).with_state_output(False).with_scale(2.0))
    assert out.state is None
    yo, _ = dc.delta_f64(*(c[n] for n in dc.NAMES), None, 2.0, True)
    dc.check(out.y, yo, "y")


def test_gradients_against_differences():
    """Directional central differences of the 64-bit forward: the gradient along random directions."""
    from mamba3.ssm import delta_rule_backward
    c = dc.make(15, 1, 75, 2, 1, 16, 32, FL)
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    host = {n: c[n].double().cpu() for n in dc.NAMES}
    gen = torch.Generator().manual_seed(1)

    def loss(**over):
        y, s = dc.delta_f64(*({**host, **over}[n] for n in dc.NAMES), None, None, True)
        return float((y * c["dy"].double().cpu()).sum() + (s * c["dh"].double().cpu()).sum())

    for n in dc.NAMES:
        u = torch.randn(host[n].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        diff = (loss(**{n: host[n] + h * u}) - loss(**{n: host[n] - h * u})) / (2 * h)
        g = getattr(d, n).double().cpu()
        # along a random direction the value is about |g|, its error 1e-5 of that; the
        # differences' own is h^2 times third derivatives and 1e-16 / h of the loss
        assert abs(float((g * u).sum()) - diff) <= 1e-4 * float(g.norm()), n


@pytest.mark.parametrize("dtype", [BF, FL])
def test_same_bits_every_time(dtype):
    from mamba3.ssm import delta_rule_backward
    c = dc.make(16, 3, 333, 6, 2, 48, 64, dtype)
    first = run(c)
    gfirst = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    for _ in range(3):
        for a, b in zip(first, run(c)):
            assert torch.equal(a, b)
        d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
        for n in dc.NAMES:
            assert torch.equal(getattr(gfirst, n), getattr(d, n)), n


def test_another_stream():
    c = dc.make(17, 2, 300, 4, 4, 64, 128, BF)
    want = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_graph_replays_on_changed_inputs():
    """Window, gradient and step captured together: replays on changed inputs equal eager calls."""
    from mamba3.ssm import delta_rule, delta_rule_backward, delta_step_
    c = dc.make(18, 2, 200, 4, 2, 64, 128, BF)
    state = c["h0"].clone()

    def all_of(st):
        out = delta_rule(dc.inputs_of(c))
        d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
        y = delta_step_(*(c[n][:, 0] for n in ("q", "k", "v", "g", "beta")), st, qk_norm=True)
        return [out.y, out.state, y, st] + [getattr(d, n) for n in dc.NAMES]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of(state.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of(state)
    for rep in range(4):
        c["v"].copy_(torch.randn_like(c["v"]))
        c["h0"].normal_()
        c["dy"].mul_(0.5)
        before = state.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(all_of(before), got)):
            assert torch.equal(a, b), (rep, i)


@pytest.mark.parametrize("B,H,G,P,N,T,lengths,dtype", [
    (1, 2, 2, 64, 128, 1500, None, BF), (2, 2, 1, 48, 96, 900, [900, 130], BF), (1, 1, 1, 16, 32, 2100, None, FL),
    (1, 3, 3, 130, 64, 700, None, HF), (2, 1, 1, 7, 5, 600, [0, 600], FL)])
def test_long_windows_of_few_heads(B, H, G, P, N, T, lengths, dtype):
    """Windows that are cut into segments run side by side, sequences that end before the last of
    them (or at once) among them; in place on the carried state as well."""
    c = dc.make(T, B, T, H, G, P, N, dtype, lengths=lengths, decay=(1e-4, 1e-1))
    check_forward(c)
    check_backward(c)
    c = dc.make(T, B, T, H, G, P, N, dtype, lengths=lengths, carried=False)
    check_forward(c)


def test_state_updated_in_place_by_a_window():
    import ctypes as C
    from mamba3 import _lib
    L = _lib.lib()
    for T in (5, 130, 800):
        c = dc.make(T, 2, T, 2, 2, 64, 128, BF)
        want_y, want_s = run(c)
        s, y = c["h0"].clone(), torch.empty_like(c["v"])
        cin = _lib.DeltaInputsC(2, T, 2, 2, 64, 128, _lib.M3_BF16, c["q"].data_ptr(), c["k"].data_ptr(),
                                c["v"].data_ptr(), 0, 0, 0, c["g"].data_ptr(), c["beta"].data_ptr(), None,
                                s.data_ptr(), 128 ** -0.5, 1, None, 0)
        need = int(L.m3_delta_rule_workspace_bytes(C.byref(cin)))
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=DEV)
        cin.workspace, cin.workspace_bytes = ws.data_ptr(), need
        _lib.check(L.m3_delta_rule(C.byref(cin), y.data_ptr(), s.data_ptr(), _lib.stream_of(s)))
        assert torch.equal(y, want_y) and torch.equal(s, want_s), T
