"""The gated delta stack: prefill, padded batches, decoding and a training step, each through the
operators together, against a 64-bit restatement of the same stack."""
import pytest
import torch

import delta_cases as dc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(**kw):
    from mamba3 import GatedDeltaConfig, GatedDeltaStack
    base = dict(d_model=128, n_layers=2, n_heads=4, n_groups=2, head_dim=32, d_state=64, seed=3)
    base.update(kw)
    return GatedDeltaStack(GatedDeltaConfig(**base), DEV)


def rms(x, w, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def restated(stack, x, lengths=None, states=None):
    """The stack in f64 on the CPU with the weights that the products use; activations are not
    rounded in between."""
    c = stack.cfg
    f = lambda t: t.double().cpu()
    r, out_states = f(x), []
    y = rms(r, f(stack.norms[0].weight), c.norm_eps)
    for i, m in enumerate(stack.mixers):
        rows = y @ f(m.in_proj.effective_weight())
        p = dict(zip(m.cols, rows.split(list(m.cols.values()), -1)))
        g = -torch.exp(f(m.a_log)) * torch.nn.functional.softplus(p["a"] + f(m.dt_bias))
        q, k = (p[n].unflatten(-1, (c.n_groups, c.d_state)) for n in ("q", "k"))
        o, s = dc.delta_f64(q, k, p["v"].unflatten(-1, (c.n_heads, c.head_dim)), g, torch.sigmoid(p["b"]),
                            None if states is None else states[i], lengths, None, True)
        out_states.append(s)
        o = rms(o.flatten(-2), f(m.norm.weight), c.norm_eps) * torch.nn.functional.silu(p["z"])
        n = rms(o @ f(m.out_proj.effective_weight()), f(stack.post[i]), c.norm_eps) * f(stack.scale[i])
        r = r + (n * torch.nn.functional.silu(p["gate"]) if c.block_gate else n)
        y = rms(r, f(stack.norms[i + 1].weight), c.norm_eps)
    return y, out_states


def off(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert torch.isfinite(a).all()
    return float((a - b).norm() / b.norm())


# bf16 activations between the operators: some ten roundings of 2^-9 (rms) a layer, two layers
TOL = 3e-2


@pytest.mark.parametrize("kw", [{}, dict(block_gate=False, n_groups=4), dict(int8_weights=True, head_dim=64, d_state=128)])
@pytest.mark.parametrize("T", [5, 150])
def test_prefill(T, kw):
    stack = make(**kw)
    x = torch.randn((2, T, 128), device=DEV).to(torch.bfloat16)
    want, _ = restated(stack, x)
    assert off(stack.forward(x), want) < TOL


def test_padded_batch_then_tokens():
    """Prompts of 90, 33 and 0 tokens in one padded prefill, then three tokens each, step by step:
    outputs and states as the prompts' own."""
    stack = make()
    lens = [90, 33, 0]
    x = torch.randn((3, 90, 128), device=DEV).to(torch.bfloat16)
    more = torch.randn((3, 3, 128), device=DEV).to(torch.bfloat16)
    cache = stack.empty_cache(3, DEV)
    y = stack.forward_cached(x, cache, torch.tensor(lens, dtype=torch.int32, device=DEV))
    ys = torch.cat([stack.forward_cached(more[:, t:t + 1], cache) for t in range(3)], 1)
    for b, n in enumerate(lens):
        whole = torch.cat([x[b:b + 1, :n], more[b:b + 1]], 1)
        want, states = restated(stack, whole)
        if n:
            assert off(y[b:b + 1, :n], want[:, :n]) < TOL
        assert off(ys[b:b + 1], want[:, n:]) < TOL
        for s, w in zip(cache, states):
            assert off(s[b:b + 1], w) < TOL


def test_gates():
    from mamba3 import _lib
    rows = torch.randn((7, 24), device=DEV) * 8
    rows[0, 0], rows[1, 1], rows[2, 8] = 200.0, -200.0, -200.0
    for code, dt in ((_lib.M3_F32, torch.float32), (_lib.M3_BF16, torch.bfloat16), (_lib.M3_F16, torch.float16)):
        r = rows.to(dt)
        a_log, bias = torch.randn(5, device=DEV), torch.randn(5, device=DEV)
        g, beta = torch.empty((7, 5), device=DEV), torch.empty((7, 5), device=DEV)
        _lib.check(_lib.lib().m3_delta_gates(7, 5, code, r.data_ptr(), r[:, 8:].data_ptr(), 24, a_log.data_ptr(),
                                             bias.data_ptr(), g.data_ptr(), beta.data_ptr(), _lib.stream_of(g)))
        a, b = r[:, :5].double(), r[:, 8:13].double()
        want = -torch.exp(a_log.double()) * torch.nn.functional.softplus(a + bias.double(), threshold=1e9)
        assert off(g, want) < 1e-6 and off(beta, torch.sigmoid(b)) < 1e-6


def test_training_step():
    """The operators under autograd with torch's products: one block's loss and every gradient against
    the same block in f64."""
    from mamba3.nn import block_norm
    from mamba3.ssm import DeltaInputs, delta_rule
    B, T, D, H, P, N = 2, 70, 48, 2, 16, 32
    gen = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(s, generator=gen)
    host = dict(x=rn(B, T, D), wi=rn(D, 2 * H * N + H * P + 2 * H) * D ** -0.5, wo=rn(H * P, D) * (H * P) ** -0.5,
                post=1 + 0.1 * rn(D), scale=0.5 + 0.1 * rn(D), pre=1 + 0.1 * rn(D))
    seed = rn(B, T, D)

    def block(p, delta, norm):
        q, k, v, a, b = (p["x"] @ p["wi"]).split([H * N, H * N, H * P, H, H], -1)
        o = delta(q.unflatten(-1, (H, N)), k.unflatten(-1, (H, N)), v.unflatten(-1, (H, P)),
                  -torch.nn.functional.softplus(a), torch.sigmoid(b))
        return norm(o.flatten(-2) @ p["wo"], p["x"], p)

    def norm64(x, r, p):
        r = r + p["scale"] * rms(x, p["post"], 1e-5)
        return r + rms(r, p["pre"], 1e-5)

    def own(q, k, v, g, b):
        return delta_rule(DeltaInputs(q, k, v, g, b).with_qk_norm(True)).y

    def own_norm(x, r, p):
        r, y = block_norm(x, r, post_weight=p["post"], scale=p["scale"], pre_weight=p["pre"])
        return r + y

    grads = []
    for dev, dt, fns in (("cpu", torch.float64, (lambda *a: dc.delta_f64(*a, None, None, None, True)[0], norm64)),
                         (DEV, torch.float32, (own, own_norm))):
        p = {n: t.to(dev, dt).requires_grad_() for n, t in host.items()}
        (block(p, *fns) * seed.to(dev, dt)).sum().backward()
        grads.append({n: t.grad for n, t in p.items()})
    for n in host:
        assert off(grads[1][n], grads[0][n]) < 2e-5, n
