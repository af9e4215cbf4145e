"""Sums that cancel, in scan.delta_scan's chunks and their gradient on an MI355X:
two terms of 24 bits whose difference is all that is left, so that a factor held
in fewer bits than fp32 shows in the result however coarsely that is rounded."""

from __future__ import annotations

import pytest
import torch

import scan_ref as R
from lightreason_amd.scan import delta_scan

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [BF, FP])
NEAR = 1 - 2.0 ** -7   # (a bf16 number)


def _zeros(n, key_heads, heads, dim, value_dim, dtype, device):
    zeros = lambda *shape: torch.zeros(shape, dtype=dtype, device=device)
    return dict(query=zeros(n, key_heads, dim), key=zeros(n, key_heads, dim), value=zeros(n, heads, value_dim),
                g=torch.zeros(n, heads, device=device), beta=torch.zeros(n, heads, device=device),
                starts=torch.tensor([0, n], dtype=torch.int32, device=device))


def _bits(shape, device, seed):
    """Numbers in [1, 2) of 24 bits, and differences of 7 bits from 2^-13 up."""
    gen = torch.Generator().manual_seed(seed)
    full = 1 + torch.randint(2**22, 2**23, shape, generator=gen) * 2.0 ** -23
    step = torch.randint(1, 128, shape, generator=gen) * 2.0 ** -13
    return full.float().to(device), step.float().to(device)


@TYPES
@pytest.mark.parametrize("dim", [64, 128])
def test_outputs_of_a_state_whose_rows_cancel(device, dtype, dim):
    """q = e0 - e1 and steps without weight: an output is S0 - S1.  Every partial
    sum is a multiple of 2^-23 below 2, which fp32 holds, and the difference has 7
    bits: the output is exact."""
    x = _zeros(130, 2, 4, dim, 64, dtype, device)
    x["query"][..., 0], x["query"][..., 1] = 1.0, -1.0
    initial = torch.zeros(1, 4, dim, 64, device=device)
    full, step = _bits((4, 64), device, 1)
    initial[0, :, 0], initial[0, :, 1] = full, full - step
    out, final = delta_scan(**x, initial=initial, scale=1.0)
    assert torch.equal(out.float(), step.expand(130, 4, 64))
    assert torch.equal(final, initial)


@TYPES
def test_outputs_of_steps_that_cancel(device, dtype):
    """u0 - u1 with keys e0 and e1, values of 1 and weights of 24 bits: exact, as
    above."""
    H = 32
    x = _zeros(60, H, H, 64, 64, dtype, device)
    x["key"][0, :, 0] = x["key"][1, :, 1] = 1.0
    x["query"][2:, :, 0], x["query"][2:, :, 1] = 1.0, -1.0
    x["value"][:2] = 1.0
    full, step = _bits((H,), device, 2)
    x["beta"][0], x["beta"][1] = full / 2, (full - step) / 2
    out, _ = delta_scan(**x, scale=2.0)
    assert torch.equal(out[2:].float(), step[None, :, None].expand(58, H, 64))


@TYPES
def test_outputs_of_weights_that_cancel(device, dtype):
    """P_i0 u0 + P_i1 u1 = e^(G_i) (u0 - NEAR u1) = 0 for decays of 24 bits.  The two
    weights have one decay (the second token's is 0), are rounded once more (2^-24 of
    it each at most), and a handful of sums round by as much: 8 of 2^-24."""
    x = _zeros(60, 8, 8, 64, 64, dtype, device)
    x["key"][0, :, 0] = x["key"][1, :, 1] = 1.0
    x["beta"].fill_(1.0)
    x["query"][2:, :, 0], x["query"][2:, :, 1] = 1.0, -NEAR
    x["value"][0], x["value"][1] = NEAR, 1.0
    x["g"][2:] = -torch.rand(58, 8, generator=torch.Generator().manual_seed(3)).to(device) * 0.02
    out, _ = delta_scan(**x, scale=1.0)
    print(f"[scan] largest {float(out[2:].abs().max()):.3e}", flush=True)
    assert out[2:].abs().max() <= 8 * 2.0 ** -24


def _gradient(x, d_out, names, **kw):
    x = {n: t.detach().requires_grad_(n in names) for n, t in x.items()}
    out, _ = delta_scan(**x, **kw)
    return torch.autograd.grad(out, [x[n] for n in names], d_out)


@TYPES
def test_query_gradients_of_steps_that_cancel(device, dtype):
    """dq_i = e^(G_i) do_i (u0 k0 + u1 k1) with k0 = e0, k1 = -NEAR e0, u0 = NEAR and u1
    = 1 (v1 = 1 - NEAR^2, 255 2^-14): 0, within 8 roundings as above."""
    x = _zeros(60, 8, 8, 64, 64, dtype, device)
    x["key"][0, :, 0], x["key"][1, :, 0] = 1.0, -NEAR
    x["beta"].fill_(1.0)
    x["value"][0, :, 0], x["value"][1, :, 0] = NEAR, 1 - NEAR * NEAR
    x["g"][2:] = -torch.rand(58, 8, generator=torch.Generator().manual_seed(4)).to(device) * 0.02
    d_out = torch.zeros_like(x["value"])
    d_out[2:, :, 0] = 1.0
    dq, = _gradient(x, d_out, ["query"], scale=1.0)
    # (Token 0 has u0 k0 alone.)
    d_first = torch.zeros_like(d_out)
    d_first[0, :, 0] = 1.0
    first, = _gradient(x, d_first, ["query"], scale=1.0)
    assert (first[0, :, 0].float() == NEAR).all()
    print(f"[scan] largest {float(dq[2:].abs().max()):.3e}", flush=True)
    assert dq[2:].abs().max() <= 8 * 2.0 ** -24


@TYPES
def test_key_gradients_of_outputs_that_cancel(device, dtype):
    """dk_0 = e^(G_1) u0 (do_1 q_1 + do_2 q_2) with q_1 = e1, q_2 = -NEAR e1, do_1 = NEAR
    and do_2 = 1: 0, within 8 roundings."""
    H = 64
    x = _zeros(3, H, H, 64, 64, dtype, device)
    x["key"][0, :, 0] = 1.0
    x["beta"].fill_(1.0)
    x["value"][0, :, 0] = 1.0
    x["query"][1, :, 1], x["query"][2, :, 1] = 1.0, -NEAR
    x["g"][1] = -torch.rand(H, generator=torch.Generator().manual_seed(5)).to(device) * 0.5
    d_out = torch.zeros_like(x["value"])
    d_out[1, :, 0], d_out[2, :, 0] = NEAR, 1.0
    dk, = _gradient(x, d_out, ["key"], scale=1.0)
    print(f"[scan] largest {float(dk[0].abs().max()):.3e}", flush=True)
    assert dk[0].abs().max() <= 8 * 2.0 ** -24
    d_out[2] = 0.0
    dk, = _gradient(x, d_out, ["key"], scale=1.0)
    want = NEAR * x["g"][1].double().exp()
    R.check("one alone", dk[0, :, 1], want, (R.half(dtype) + 4 * 2.0 ** -24) * want)
