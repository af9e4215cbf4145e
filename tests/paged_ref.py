"""Plain 64-bit forms of the paged-cache operators and of the draft
verification, for the tests: loops over sequences, heads and rows, written
from the definitions."""

from __future__ import annotations

import math
import random

import torch


def half_step(dtype) -> float:
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def block_table(lengths, page, pages, seed, width=None):
    """Shuffled pages: table rows [seqs][width] (-1 past a row's pages)."""
    counts = [-(-n // page) for n in lengths]
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = width or max(1, max(counts, default=0)) + 1
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    assert at <= pages
    return rows


def gathered(cache, blocks, n):
    """[kv_heads, n, dim] float64 of a row's first n positions."""
    x = cache[torch.tensor(blocks, dtype=torch.int64, device=cache.device)]
    return x.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n].double()


def attention(q, k_cache, v_cache, table, starts, kv_lengths, scale, gate=None):
    """(out, spread, score) in float64: the attention, the attention of |v|
    (both times the gate), and the largest sum |q||k| scale, for bounds.
    Rows of no sequence are 0; a row sums over the positions that it sees."""
    N, H, D = q.shape
    K, page = k_cache.shape[1], k_cache.shape[2]
    out = torch.zeros(N, H, D, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    score = 0.0
    for s, kv in enumerate(kv_lengths):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n == 0 or kv == 0:
            continue
        kv = min(kv, len(table[s]) * page)
        blocks = table[s][:-(-kv // page)]
        k, v = gathered(k_cache, blocks, kv), gathered(v_cache, blocks, kv)
        for h in range(H):
            kh, vh = k[h // (H // K)], v[h // (H // K)]
            for i in range(0, n, 512):
                j = min(n, i + 512)
                qh = q[a + i:a + j, h].double()
                x = (qh @ kh.t()) * scale
                seen = torch.arange(kv, device=q.device)[None] <= kv - n + torch.arange(i, j, device=q.device)[:, None]
                x = torch.where(seen, x, -math.inf)
                top = x.amax(dim=1, keepdim=True)
                w = torch.where(seen, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
                w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
                # values that nobody in this chunk sees with weight may be NaN:
                # take them out before the product
                used = seen.any(dim=0)
                clean = torch.isfinite(vh).all(dim=1)
                vz = torch.where((used & clean)[:, None], vh, 0.0)
                out[a + i:a + j, h] = w @ vz
                spread[a + i:a + j, h] = w @ vz.abs()
                dirty = torch.nonzero(used & ~clean).flatten().tolist()
                for p in dirty:
                    rows = torch.nonzero(seen[:, p]).flatten()
                    out[a + i + rows, h] += w[rows, p][:, None] * vh[p][None]
                kz = torch.where(torch.isfinite(kh), kh, 0.0)
                score = max(score, float((qh.abs() @ kz.abs().t()).max()) * abs(scale))
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, spread = out * g, spread * g
    return out, spread, score


def attention_bound(out, spread, score, dtype, dim, longest, vmax):
    """How far the kernel may be off, element by element: the rounding of the
    output (half a step of it); the rounding of each probability (half a step
    of its share, so half a step of the attention of |v|); scores in fp32 (a
    dot product of dim terms and its scaling, (dim + 4) 2^-24 sum|q||k| scale
    off in the exponent; twice, since the normaliser is off as well); exponent,
    running sums and products of `longest` positions in fp32 (2^-24 each, and
    2^-20 for the exponential); fp16 probabilities below 2^-14 keep steps of
    2^-24, half of one for every position."""
    h = half_step(dtype)
    soft = 2 * (dim + 4) * 2.0 ** -24 * score + 2 * longest * 2.0 ** -24 + 2.0 ** -20
    bound = h * out.abs() * (1 + 2.0 ** -6) + (h + soft) * spread
    if dtype == torch.float16:
        bound = bound + longest * 2.0 ** -25 * vmax + 2.0 ** -25
    return bound + 1e-30


def norm_rope(x, weight, cos, sin, eps):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps) * (1.0 + weight.double())
    if cos is not None:
        half = cos.shape[-1] // 2
        a, b = x[..., :half].clone(), x[..., half:2 * half].clone()
        c, s = cos.double()[:, None], sin.double()[:, None]
        x = x.clone()
        x[..., :half] = a * c[..., :half] - b * s[..., :half]
        x[..., half:2 * half] = b * c[..., half:] + a * s[..., half:]
    return x


def plan(new, lengths, held, table, free, page):
    """Lists: (starts, kv, held, positions, slots, table, free)."""
    held, table, free = list(held), [list(r) for r in table], list(free)
    starts, positions, slots = [0], [], []
    for r, (n, c) in enumerate(zip(new, lengths)):
        while held[r] * page < c + n:
            table[r][held[r]] = free.pop()
            held[r] += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r][p // page] * page + p % page)
        starts.append(starts[-1] + n)
    return starts, [c + n for c, n in zip(lengths, new)], held, positions, slots, table, free


def verify(tokens, target, starts, uniforms, samples, draft=None):
    """Lists (accepted, next), block by block in Python floats (64 bits)."""
    accepted, chosen = [], []
    target = target.double().cpu()
    draft = None if draft is None else draft.double().cpu()
    tokens = tokens.tolist()
    vocab = target.shape[1]

    def mass(x):
        return torch.where((x > 0) & torch.isfinite(x), x, 0.0)
    for b in range(len(starts) - 1):
        s, n = starts[b], starts[b + 1] - starts[b]
        if n <= 0:
            accepted.append(0)
            chosen.append(-1)
            continue
        j = 0
        while j + 1 < n:
            x = tokens[s + j + 1]
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else float(draft[s + j, x])
            if not float(uniforms[s + j]) * q < float(target[s + j, x]):
                break
            j += 1
        m = mass(target[s + j])
        if j + 1 < n:
            if draft is not None:
                rest = mass(target[s + j] - draft[s + j])
            else:
                rest = m.clone()
                if 0 <= tokens[s + j + 1] < vocab:
                    rest[tokens[s + j + 1]] = 0.0
            if float(rest.sum()) > 0:
                m = rest
        accepted.append(j)
        if not float(m.sum()) > 0:
            chosen.append(-1)
            continue
        run = torch.cumsum(m, 0)
        border = max(float(samples[b]), 0.0) * float(run[-1])
        at = int(torch.searchsorted(run, border, right=True))
        chosen.append(min(at, int(torch.nonzero(m)[-1])))
    return accepted, chosen
