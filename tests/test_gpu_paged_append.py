"""The paged append of long steps, where a group of lanes takes four head rows.
Bounds: half a step of the type of the 64-bit value, plus 2^-20 of the row's
largest for the fp32 sums (fp16: half a step below its normal range)."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF, HF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [
    (1300, 16, 2, 256, 64), (3200, 3, 1, 256, 256), (6200, 5, 1, 128, 128), (6200, 4, 1, 128, 0),
    (12500, 1, 3, 64, 32), (24600, 0, 1, 64, 64)])
def test_append_of_long_steps(device, dtype, tokens, heads, kv_heads, dim, rotary):
    from lightreason_amd.paged import paged_append

    g = torch.Generator(device=device).manual_seed(tokens)
    N, page, pages = tokens, 16, tokens // 16 + 3

    def normal(*shape):
        return torch.empty(shape, device=device).normal_(generator=g).to(dtype)
    kc, vc = normal(pages, kv_heads, page, dim), normal(pages, kv_heads, page, dim)
    slots = torch.randperm(pages * page, generator=g, device=device)[:N]
    slots[7], slots[N - 1] = -1, pages * page
    q = normal(N, heads, 2 * dim)[:, :, :dim] if heads else None
    kv = normal(N, kv_heads, 2, dim)
    k, v = kv[:, :, 0], kv[:, :, 1]
    qn, kn = (0.1 * normal(dim).float()).to(dtype), (0.1 * normal(dim).float()).to(dtype)
    cos = sin = positions = c = s = None
    if rotary:
        angle = torch.rand(500, rotary // 2, device=device, generator=g) * 6.28
        angle = torch.cat([angle, angle], 1)
        cos, sin = angle.cos(), angle.sin()
        positions = torch.randint(0, 500, (N,), generator=g, device=device, dtype=torch.int32)
        c, s = cos[positions.long()], sin[positions.long()]
    kc0, vc0 = kc.clone(), vc.clone()
    out = torch.full((N, heads, dim), 7.0, dtype=dtype, device=device) if heads else None
    paged_append(k, v, kc, vc, slots, q=q, q_norm=qn if heads else None, k_norm=kn, cos=cos, sin=sin,
                 positions=positions, q_out=out)
    live = (slots >= 0) & (slots < pages * page)
    block, row = slots[live] // page, slots[live] % page

    def close(have, want):
        bound = ref.half_step(dtype) * want.abs() + 2.0 ** -20 * want.abs().amax(dim=-1, keepdim=True)
        if dtype == HF:
            bound = bound + 2.0 ** -25
        assert bool(((have.double() - want).abs() <= bound).all())
    close(kc[block, :, row], ref.norm_rope(k, kn, c, s, 1e-6)[live])
    assert torch.equal(vc[block, :, row], v[live])
    still = torch.ones(pages, page, dtype=torch.bool, device=device)
    still[block, row] = False
    still = still[:, None, :, None].expand_as(kc)
    assert torch.equal(kc[still], kc0[still]) and torch.equal(vc[still], vc0[still])
    if heads:
        close(out[live], ref.norm_rope(q, qn, c, s, 1e-6)[live])
        assert bool((out[~live] == 7.0).all())


def test_append_of_a_long_step_in_place_of_the_queries(device):
    from lightreason_amd.paged import paged_append

    x = torch.randn(3200, 3, 256, dtype=BF, device=device)
    k = torch.randn(3200, 1, 256, dtype=BF, device=device)
    kc, vc = (torch.zeros(200, 1, 16, 256, dtype=BF, device=device) for _ in range(2))
    cos, slots = torch.rand(3200, 32, device=device), torch.arange(3200, device=device)
    want = paged_append(k, k, kc, vc, slots, q=x, cos=cos, sin=cos)
    assert torch.equal(paged_append(k, k, kc, vc, slots, q=x, cos=cos, sin=cos, q_out=x), want)
