"""The gated delta rule's workspaces: a call writes nothing before or after the bytes it asked for,
and nothing that they held before the call reaches a result."""
import pytest
import torch

import delta_cases as dc

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
GUARD = 1 << 16


def calls(c):
    from mamba3.ssm import delta_rule, delta_rule_backward
    out = delta_rule(dc.inputs_of(c))
    d = delta_rule_backward(dc.inputs_of(c), c["dy"], c["dh"])
    torch.cuda.synchronize()
    return [out.y, out.state] + [getattr(d, n) for n in dc.NAMES if getattr(d, n) is not None]


@pytest.mark.parametrize("B,H,G,P,N,T,lengths,dtype", [
    (1, 2, 2, 64, 128, 1500, None, BF),          # segments, fetched straight to LDS
    (2, 2, 1, 48, 96, 900, [900, 130], BF), (1, 1, 1, 16, 32, 1100, None, FL), (1, 3, 3, 130, 64, 700, None, HF),
    (3, 4, 2, 64, 128, 130, [130, 0, 65], BF),   # whole windows
    (2, 2, 2, 7, 5, 100, [0, 100], FL), (1, 1, 1, 64, 64, 17, None, BF)])
def test_workspace_bounds_and_contents(monkeypatch, B, H, G, P, N, T, lengths, dtype):
    import mamba3.ssm.delta as module
    c = dc.make(T + 3, B, T, H, G, P, N, dtype, lengths=lengths)
    want = calls(c)
    asked = []

    def guarded(cin, need, device):
        if need == 0:
            return None
        buf = torch.full((GUARD + need + GUARD,), 0xFF, dtype=torch.uint8, device=device)   # NaN in every type
        cin.workspace, cin.workspace_bytes = buf.data_ptr() + GUARD, need
        asked.append((buf, need))
        return buf

    monkeypatch.setattr(module, "_workspace", guarded)
    got = calls(c)
    assert len(asked) == 2
    for buf, need in asked:
        assert bool((buf[:GUARD] == 0xFF).all()) and bool((buf[GUARD + need:] == 0xFF).all())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
