"""The gated delta rule over packed sequences in float64, and inputs and error
bounds for its tests."""

from __future__ import annotations

import math

import torch

EPS = 1e-6


def half(dtype) -> float:
    """Half a step of a rounding to dtype, relative to the value."""
    return torch.finfo(dtype).eps / 2


def inputs(lengths, key_heads, heads, dim, value_dim, dtype, seed, *, unit=True, lead=0, tail=0, device="cuda",
           beta_dtype=None, decay=(0.001, 1.6)):
    """Packed rows as the convolution leaves them (strided views of one row per
    token), ``lead`` and ``tail`` rows of no sequence around them."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    N = lead + sum(lengths) + tail
    normal = lambda *shape: torch.randn(shape, generator=gen, dtype=torch.float64)
    q, k = normal(N, key_heads, dim), normal(N, key_heads, dim)
    if unit:
        q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    v = normal(N, heads, value_dim)
    row = torch.cat([x.reshape(N, -1) for x in (q, k, v)], dim=1).to(dtype).to(device)
    a, b = key_heads * dim, 2 * key_heads * dim
    lo, hi = (math.log(x) for x in decay)
    g = -torch.exp(torch.rand(N, heads, generator=gen) * (hi - lo) + lo)
    starts = [lead]
    for n in lengths:
        starts.append(starts[-1] + n)
    return dict(query=row[:, :a].view(N, key_heads, dim), key=row[:, a:b].view(N, key_heads, dim),
                value=row[:, b:].view(N, heads, value_dim), g=g.float().to(device),
                beta=torch.sigmoid(normal(N, heads)).to(beta_dtype or dtype).to(device),
                starts=torch.tensor(starts, dtype=torch.int32, device=device))


def states(rows, heads, dim, value_dim, seed, device="cuda"):
    gen = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(rows, heads, dim, value_dim, generator=gen) * 0.3).to(device)


def rule(x, initial, *, normalize=False, scale=None):
    """(out, final, size): outputs and last states in float64, and per sequence,
    head and column the largest norm that the state's column, or a value of it,
    has had."""
    q, k, v, g, beta = (x[n].double() for n in ("query", "key", "value", "g", "beta"))
    H, K, D = v.shape[1], q.shape[1], q.shape[2]
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS) for t in (q, k))
    q, k = q.repeat_interleave(H // K, 1), k.repeat_interleave(H // K, 1)
    scale = D ** -0.5 if scale is None else scale
    out, finals, sizes = torch.zeros_like(v), [], []
    starts = x["starts"].tolist()
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        S = initial[s].double()
        size = S.norm(dim=1)
        for t in range(a, b):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None, :]
            out[t] = scale * (S * q[t][:, :, None]).sum(1)
            size = torch.maximum(size, torch.maximum(S.norm(dim=1), v[t].abs()))
        finals.append(S)
        sizes.append(size)
    if not finals:
        return out, torch.zeros(0, H, D, v.shape[2], dtype=torch.float64, device=v.device), None
    return out, torch.stack(finals), torch.stack(sizes)


def bounds(x, out, size, *, normalize=False, scale=None):
    """What out and final may be off by.  With |k| <= 1, 0 <= beta <= 1 and g <= 0
    a step of the rule does not lengthen an error in the state, so the errors of
    n steps add up.  A step makes, per column, the roundings of a sum of dim
    products and of a few operations (in the chunked form: sums of dim, 64 and 64
    products), each of at most 2^-24 of the column's norm or value: dim + 136
    roundings.  Rounding errors of either sign add up as a random walk; 8 standard
    deviations are allowed."""
    q = x["query"].double()
    D, H, K = q.shape[2], x["value"].shape[1], q.shape[1]
    if normalize:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS)
    scale = D ** -0.5 if scale is None else scale
    starts = x["starts"].tolist()
    norms = q.norm(dim=-1).repeat_interleave(H // K, 1)
    b_out, b_final = half(x["value"].dtype) * out.abs(), []
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        n = b - a
        state = 8 * math.sqrt((n + 1) * (D + 136)) * 2.0 ** -24 * size[s]
        b_final.append(state[:, None, :])
        if n:
            b_out[a:b] += scale * norms[a:b, :, None] * state[None] + 2.0 ** -24   # fp16 below its normal range
    return b_out, torch.stack(b_final)


def check(name, got, want, bound):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    worst = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    ratio = ((got - want).abs() / (bound + 1e-300)).max() if got.numel() else 0.0
    print(f"[scan] {name}: error / bound {float(ratio):.3f}", flush=True)
    assert torch.isfinite(got).all() and float(worst) <= 0.0, (name, float(ratio))
