"""Paged calls whose tensors lie in one buffer, between each other's rows."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF, _case, _run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [(16, 2, 256), (4, 2, 64), (1, 1, 128)])
@pytest.mark.parametrize("form", ["token", "head", "pitch", "tokens apart", "heads apart"])
def test_attention_into_the_buffer_of_its_inputs(device, layout, form):
    H, _, D = layout
    c, *_ = _case(device, *layout, 16, [(70, 1), (200, 30), (40, 4)], BF, seed=41, gate=True)
    want = _run_attention(c)
    N = c["q"].shape[0]
    if form == "token":      # [token][q heads, gate heads, out heads]
        buf = torch.zeros(N, 3 * H, D, dtype=BF, device=device)
        q, gate, out = buf[:, :H], buf[:, H:2 * H], buf[:, 2 * H:]
    elif form == "head":     # [token][head][q, gate, out]
        buf = torch.zeros(N, H, 3 * D, dtype=BF, device=device)
        q, gate, out = buf[:, :, :D], buf[:, :, D:2 * D], buf[:, :, 2 * D:]
    elif form == "pitch":    # [token][q and gate by head | out heads]
        buf = torch.zeros(N, 3 * H * D, dtype=BF, device=device)
        both = buf[:, :2 * H * D].view(N, H, 2 * D)
        q, gate, out = both[:, :, :D], both[:, :, D:], buf[:, 2 * H * D:].view(N, H, D)
    elif form == "tokens apart":   # head-major: [head][q, gate, out][token]
        buf = torch.zeros(H, 3, N, D, dtype=BF, device=device)
        q, gate, out = (buf[:, i].transpose(0, 1) for i in range(3))
    else:                    # one tensor behind the other
        buf = torch.zeros(3, N, H, D, dtype=BF, device=device)
        q, gate, out = buf[0], buf[1], buf[2]
    q.copy_(c["q"])
    gate.copy_(c["gate"])
    c["q"], c["gate"] = q, gate
    held = q.clone(), gate.clone()
    got = _run_attention(c, out=out)
    assert got is out and torch.equal(out, want) and torch.equal(q, held[0]) and torch.equal(gate, held[1])


def test_overlapping_buffers_are_refused(device):
    from lightreason_amd.paged import paged_append

    c, *_ = _case(device, 8, 2, 64, 8, [(20, 2), (24, 3)], BF, seed=42, gate=True)
    buf = torch.zeros(6, 8, 64, dtype=BF, device=device)
    buf[:5] = c["q"]
    c["q"] = buf[:5]
    for out in (buf[1:], buf[:5], torch.zeros(5, 1, 64, dtype=BF, device=device).expand(5, 8, 64),
                torch.zeros(1, 8, 64, dtype=BF, device=device).expand(5, 8, 64)):
        with pytest.raises(ValueError):
            _run_attention(c, out=out)
    c["q"] = torch.zeros(5, 1, 64, dtype=BF, device=device).expand(5, 8, 64)   # read only: as good as any
    _run_attention(c)
    c["q"], c["gate"] = buf[:5].clone(), buf[:5]
    with pytest.raises(ValueError):
        _run_attention(c, out=buf[1:])
    k, slots = torch.zeros(5, 2, 64, dtype=BF, device=device), torch.arange(5, device=device)
    for q, q_out in ((buf[:5], buf[1:]), (buf[1:], buf[:5])):
        with pytest.raises(ValueError):
            paged_append(k, k, c["k_cache"], c["v_cache"], slots, q=q, q_out=q_out)
    flat = torch.zeros(8 * 5 * 64 + 64, dtype=BF, device=device)
    q_out = flat[:8 * 5 * 64].view(5, 8, 64)
    with pytest.raises(ValueError):
        paged_append(flat[-10 * 64:].view(5, 2, 64), k, c["k_cache"], c["v_cache"], slots, q=buf[:5], q_out=q_out)
    assert paged_append(k, k, c["k_cache"], c["v_cache"], slots, q=buf[:5], q_out=buf[:5]) is not None
