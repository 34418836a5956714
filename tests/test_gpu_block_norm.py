"""block_norm (m3_block_norm and its gradient) against its formula in 64 bits, differentiated by torch,
and against differences."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
# one rounding to the storage type (half a unit in the last place: 2^-11 of a value for f16's 11
# significant bits, 2^-8 for bf16's 8); f32: sums of a row and of a column of rounded terms, a random
# walk of 2^-24 each
TOL = {FL: 2e-6, HF: 2.0 ** -11 + 2e-6, BF: 2.0 ** -8 + 2e-6}
ACT = {"none": lambda z: z, "silu": lambda z: z * torch.sigmoid(z), "sigmoid": torch.sigmoid}


def formula(x, residual, gate, post_weight, scale, pre_weight, eps, activation, post_norm):
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if post_norm else x
    n = n if post_weight is None else n * post_weight
    n = n if gate is None else n * ACT[activation](gate)
    n = n if scale is None else n * scale
    r = residual + n
    y = r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
    return r, y if pre_weight is None else y * pre_weight


NAMES = ("x", "residual", "gate", "post_weight", "scale", "pre_weight")


def make(seed, shape, dtype, rdtype, without=()):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=gen)
    d = shape[-1]
    c = dict(x=rn(*shape).to(dtype), residual=(2 * rn(*shape)).to(rdtype), gate=rn(*shape).to(dtype),
             post_weight=1 + 0.2 * rn(d), scale=0.5 + 0.2 * rn(d), pre_weight=1 + 0.2 * rn(d))
    c = {n: None if n in without else t.to(DEV) for n, t in c.items()}
    return c, rn(*shape).to(rdtype).to(DEV), rn(*shape).to(dtype).to(DEV)


def rel(got, want, size=0.0):
    """The error over the norm of the result or, where that is more, over `size`: that of the terms
    whose difference it is."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    n = max(float(want.norm()), size)
    return float((got - want).norm()) / (n if n > 0 else 1.0)


def check(c, dr, dy, activation="silu", post_norm=True, eps=1e-5):
    from mamba3.nn import block_norm, block_norm_backward
    kw = {n: c[n] for n in NAMES[2:]}
    r, y = block_norm(c["x"], c["residual"], **kw, eps=eps, activation=activation, post_norm=post_norm)
    d = block_norm_backward(c["x"], c["residual"], dr, dy, **kw, eps=eps, activation=activation,
                            post_norm=post_norm)
    leaves = {n: None if c[n] is None else c[n].double().cpu().requires_grad_() for n in NAMES}
    ro, yo = formula(*(leaves[n] for n in NAMES), eps, activation, post_norm)
    (ro * dr.double().cpu()).sum().add((yo * dy.double().cpu()).sum()).backward()
    assert r.dtype == c["residual"].dtype and y.dtype == c["x"].dtype
    # dx = rx (t - x mean(t x) rx^2), t the gradient of the normed x: for a row of one value the two
    # terms are equal up to eps
    dr_all = leaves["residual"].grad
    t = dr_all * (1 if c["gate"] is None else ACT[activation](leaves["gate"].detach()))
    for n in ("scale", "post_weight"):
        t = t if c[n] is None else t * leaves[n].detach()
    rx = 1 / torch.sqrt((leaves["x"].detach() ** 2).mean(-1, keepdim=True) + eps)
    size = {"x": float((t * rx).norm())} if post_norm else {}
    for what, a, b in [("residual", r, ro), ("y", y, yo)]:
        assert rel(a, b) <= TOL[a.dtype], (what, rel(a, b))
    for n in NAMES:
        g = getattr(d, n)
        if c[n] is None:
            assert g is None
        else:
            e = rel(g, leaves[n].grad, size.get(n, 0.0))
            assert e <= TOL[g.dtype], ("d" + n, e)
    return r, y, d


@pytest.mark.parametrize("dtype,rdtype", [(BF, BF), (BF, FL), (HF, HF), (HF, FL), (FL, FL)])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (1, 1536), (130, 768), (17, 1001), (9, 2048), (6, 2056),
                                   (4, 2049), (3, 8192), (2, 9000), (2, 32768)])
def test_shapes_and_types(shape, dtype, rdtype):
    c, dr, dy = make(shape[0] * 7 + shape[1], shape, dtype, rdtype)
    check(c, dr, dy)


@pytest.mark.parametrize("without", [w for k in range(4) for w in itertools.combinations(NAMES[2:], k)])
def test_what_may_be_absent(without):
    c, dr, dy = make(len(without), (33, 520), BF, FL, without)
    check(c, dr, dy)
    check(c, dr, dy, post_norm=False)


@pytest.mark.parametrize("activation", sorted(ACT))
def test_activations(activation):
    c, dr, dy = make(1, (40, 264), FL, FL)
    c["gate"][0, :4] = torch.tensor([100.0, -100.0, 1e4, -1e4], device=DEV) if activation != "none" else 3.0
    check(c, dr, dy, activation=activation)


def test_many_rows():
    """More rows than the gradient has workgroups: each sums over several."""
    c, dr, dy = make(2, (2500, 264), BF, FL)
    check(c, dr, dy)


def test_zero_rows_and_no_rows():
    c, dr, dy = make(3, (4, 64), FL, FL)
    c["x"][1] = 0
    c["x"][2] = c["residual"][2] = 0
    check(c, dr, dy)
    c, dr, dy = make(3, (0, 64), FL, FL)
    check(c, dr, dy)


def test_missing_gradients_and_outputs():
    """One of the two outgoing gradients absent is a zero one; no norm after the add."""
    from mamba3.nn import block_norm, block_norm_backward
    c, dr, dy = make(4, (50, 264), BF, FL)
    kw = {n: c[n] for n in NAMES[2:]}
    for a, b in [((None, dy), (torch.zeros_like(dr), dy)), ((dr, None), (dr, torch.zeros_like(dy)))]:
        x, z = (block_norm_backward(c["x"], c["residual"], *p, **kw) for p in (a, b))
        for n in NAMES:
            assert torch.equal(getattr(x, n), getattr(z, n)), n
    r, y = block_norm(c["x"], c["residual"], **kw, normed=False)
    assert y is None and torch.equal(r, block_norm(c["x"], c["residual"], **kw)[0])


@pytest.mark.parametrize("extra", [0, 8, 5])
def test_gate_in_place(extra):
    """A gate that is columns of a wider row, aligned and not, as its contiguous copy."""
    from mamba3.nn import block_norm
    c, _, _ = make(5, (3, 11, 264), BF, BF)
    wide = torch.randn((3, 11, 264 + 8 + extra), device=DEV).to(BF)
    kw = {n: c[n] for n in NAMES[3:]}
    for lo in (0, 8 if extra != 5 else 3):
        gate = wide[..., lo:lo + 264]
        for a, b in zip(block_norm(c["x"], c["residual"], gate=gate, **kw),
                        block_norm(c["x"], c["residual"], gate=gate.contiguous(), **kw)):
            assert rel(a, b) <= TOL[BF]


def test_unaligned_rows():
    c, dr, dy = make(6, (20, 264), BF, BF)
    for n in ("x", "residual"):
        flat = torch.empty(20 * 264 + 1, dtype=BF, device=DEV)
        flat[1:] = c[n].flatten()
        c[n] = flat[1:].view(20, 264)
    check(c, dr, dy)


def test_autograd():
    from mamba3.nn import block_norm
    c, dr, dy = make(7, (2, 9, 96), FL, FL)
    leaves = {n: c[n].clone().requires_grad_() for n in NAMES}
    r, y = block_norm(leaves["x"], leaves["residual"], **{n: leaves[n] for n in NAMES[2:]})
    ((r * dr).sum() + (y * dy).sum()).backward()
    _, _, d = check(c, dr, dy)
    for n in NAMES:
        assert torch.equal(leaves[n].grad, getattr(d, n)), n


def test_gradients_against_differences():
    from mamba3.nn import block_norm_backward
    c, dr, dy = make(8, (7, 40), FL, FL)
    d = block_norm_backward(c["x"], c["residual"], dr, dy, **{n: c[n] for n in NAMES[2:]})
    host = {n: c[n].double().cpu() for n in NAMES}
    gen = torch.Generator().manual_seed(2)

    def loss(over):
        r, y = formula(*({**host, **over}[n] for n in NAMES), 1e-5, "silu", True)
        return float((r * dr.double().cpu()).sum() + (y * dy.double().cpu()).sum())

    for n in NAMES:
        u = torch.randn(host[n].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        diff = (loss({n: host[n] + h * u}) - loss({n: host[n] - h * u})) / (2 * h)
        g = getattr(d, n).double().cpu()
        assert abs(float((g * u).sum()) - diff) <= 1e-5 * float(g.norm()), n


def test_same_bits_every_time_and_in_a_graph():
    from mamba3.nn import block_norm, block_norm_backward
    c, dr, dy = make(9, (1500, 520), BF, FL)
    kw = {n: c[n] for n in NAMES[2:]}

    def all_of():
        r, y = block_norm(c["x"], c["residual"], **kw)
        d = block_norm_backward(c["x"], c["residual"], dr, dy, **kw)
        return [r, y] + [getattr(d, n) for n in NAMES]

    first = all_of()
    for a, b in zip(first, all_of()):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of()
    for _ in range(3):
        c["x"].copy_(torch.randn_like(c["x"]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(all_of(), got):
            assert torch.equal(a, b)
