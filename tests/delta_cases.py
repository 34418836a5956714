"""The gated delta rule restated in 64 bits, token by token from its definition,
on the CPU: outputs, and gradients by torch's differentiation of exactly that."""
import torch

UNIT_EPS = 1e-6


def unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + UNIT_EPS)


def delta_f64(q, k, v, g, beta, h0=None, lengths=None, scale=None, qk_norm=False):
    """q, k [B,T,G,N], v [B,T,H,P], g, beta [B,T,H], h0 [B,H,P,N] -> y, state (f64, CPU).  Padding
    tokens are left out sequence by sequence, so what they hold cannot matter."""
    q, k, v, g, beta = (t.double().cpu() for t in (q, k, v, g, beta))
    B, T, H, P = v.shape
    G, N = k.shape[2], k.shape[3]
    scale = N ** -0.5 if scale is None else scale
    lens = [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]
    ys, states = [], []
    for b in range(B):
        S = torch.zeros(H, P, N, dtype=torch.float64) if h0 is None else h0[b].double().cpu()
        rows = []
        for t in range(lens[b]):
            kt, qt = k[b, t], q[b, t]
            if qk_norm:
                kt, qt = unit(kt), unit(qt)
            kt, qt = (x.repeat_interleave(H // G, 0)[:, None, :] for x in (kt, qt))
            S = torch.exp(g[b, t])[:, None, None] * S
            u = beta[b, t][:, None] * (v[b, t] - (S * kt).sum(-1))
            S = S + u[..., None] * kt
            rows.append(scale * (S * qt).sum(-1))
        rows += [torch.zeros(H, P, dtype=torch.float64)] * (T - lens[b])
        ys.append(torch.stack(rows) if rows else torch.zeros(0, H, P, dtype=torch.float64))
        states.append(S)
    return torch.stack(ys), torch.stack(states)


def make(seed, B, T, H, G, P, N, dtype, qk_norm=True, carried=True, lengths=None, device="cuda:0",
         decay=(0.001, 1.6)):
    """Inputs as a layer meets them: log decays over `decay`, write strengths in (0, 1), keys about
    one long where they are not brought to unit length."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=gen)
    k = rn(B, T, G, N) * (1.0 if qk_norm else N ** -0.5)
    lo, hi = decay
    g = -(lo * (hi / lo) ** torch.rand((B, T, H), generator=gen))
    out = dict(q=rn(B, T, G, N).to(dtype), k=k.to(dtype), v=rn(B, T, H, P).to(dtype), g=g,
               beta=torch.sigmoid(rn(B, T, H)), h0=0.3 * rn(B, H, P, N) if carried else None,
               dy=rn(B, T, H, P).to(dtype), dh=0.3 * rn(B, H, P, N))
    out = {n: None if t is None else t.to(device) for n, t in out.items()}
    out["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    out["qk_norm"] = qk_norm
    return out


def inputs_of(c):
    from mamba3.ssm import DeltaInputs
    di = DeltaInputs(c["q"], c["k"], c["v"], c["g"], c["beta"]).with_qk_norm(c["qk_norm"])
    if c["h0"] is not None:
        di = di.with_state(c["h0"])
    if c["lengths"] is not None:
        di = di.with_lengths(c["lengths"])
    return di


def oracle(c):
    return delta_f64(c["q"], c["k"], c["v"], c["g"], c["beta"], c["h0"],
                     None if c["lengths"] is None else c["lengths"].tolist(), None, c["qk_norm"])


NAMES = ("q", "k", "v", "g", "beta", "h0")


def oracle_grads(c):
    """y, state and the gradients of <y, dy> + <state, dh> (f64; None where there is no input)."""
    lens = None if c["lengths"] is None else c["lengths"].tolist()
    leaves = {n: None if c[n] is None else c[n].detach().double().cpu().requires_grad_() for n in NAMES}
    y, s = delta_f64(*(leaves[n] for n in NAMES), lens, None, c["qk_norm"])
    (y * c["dy"].double().cpu()).sum().add((s * c["dh"].double().cpu()).sum()).backward()
    zero = lambda t: torch.zeros_like(t) if t.grad is None else t.grad
    return y.detach(), s.detach(), {n: None if t is None else zero(t) for n, t in leaves.items()}


def unit_sizes(c):
    """{"q", "k": norm of the gradient on the way into the unit-length norm}: the norm's own gradient
    r (d - x^ (x^ . d)) takes d's part along x out, all of it for a vector of one element."""
    if not c["qk_norm"]:
        return {}
    lens = None if c["lengths"] is None else c["lengths"].tolist()
    q, k = (unit(c[n].double().cpu()).requires_grad_() for n in ("q", "k"))
    y, s = delta_f64(q, k, c["v"], c["g"], c["beta"], c["h0"], lens)
    ((y * c["dy"].double().cpu()).sum() + (s * c["dh"].double().cpu()).sum()).backward()
    out = {}
    for n, u in (("q", q), ("k", k)):
        x = c[n].double().cpu()
        out[n] = float((u.grad / torch.sqrt((x * x).sum(-1, keepdim=True) + UNIT_EPS)).norm())
    return out


# Error of an output against 64 bits, 2-norm over 2-norm.  f32 outputs: products of operands held in
# at least 16 bits (2^-17 each), summed in f32; the errors of many terms add as a random walk and a
# sum's cancellation may raise them a few times: 1e-5.  f16: half a unit in the last place of each
# value on top.  bf16: half a unit (2^-9) for the result and one for each of two operands rounded to
# the storage type.
TOL = {torch.float32: 1e-5, torch.float16: 2.0 ** -11 + 1e-5, torch.bfloat16: 3 * 2.0 ** -9}


def rel(got, want, size=0.0):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all(), "not finite"
    n = max(float(want.norm()), size)
    d = float((got - want).norm())
    return d / n if n > 0 else d


def check(got, want, what, size=0.0):
    """The error over the norm of the result or, where that is more, over `size`: that of the terms
    whose difference it is."""
    e = rel(got, want, size)
    assert e <= TOL[got.dtype], (what, e, TOL[got.dtype])
