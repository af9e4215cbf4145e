"""Paged attention: what a row does not see, and what is not finite.  Bounds as
in paged_ref.py."""

from __future__ import annotations

import math

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF, HF, _case, _run_attention

pytestmark = pytest.mark.gpu


# ---- attention: what a row does not see -------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout,kv,n", [((16, 2, 256), 230, 100), ((8, 2, 64), 230, 100), ((8, 1, 128), 40, 4),
                                         ((16, 2, 256), 2000, 1500)])
def test_attention_hidden_positions_leave_every_bit(device, layout, dtype, kv, n):
    # Other finite keys and values from a position on: rows before it keep
    # their bits, however far the scores of the rows behind it move.
    c, *_ = _case(device, *layout, 16, [(kv, n), (64, 2)], dtype, seed=25, gate=True)
    first = kv - n // 2
    clean = _run_attention(c, max_new=n)
    g = torch.Generator(device=device).manual_seed(26)
    for factor in (1.0, 40.0, 3000.0):
        for cache in (c["k_cache"], c["v_cache"]):
            for p in range(first, kv):
                row = cache[int(c["table"][0, p // 16]), :, p % 16]
                row.copy_(torch.empty(row.shape, device=device).normal_(0, factor, generator=g))
        out = _run_attention(c, max_new=n)
        seen = n - (kv - first)   # tokens before the position
        assert torch.equal(out[:seen], clean[:seen]) and torch.equal(out[n:], clean[n:])
        assert not torch.equal(out[seen:n], clean[seen:n])


@pytest.mark.parametrize("layout", [(16, 2, 256), (8, 2, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_rows_that_see_a_value_that_is_not_finite(device, bad, layout):
    # Position 150 of a chunk from 130 on: every row, those that see it
    # included, is finite where the 64-bit form is, and within the bound there.
    c, table, starts, kvs = _case(device, *layout, 16, [(230, 100), (64, 4), (400, 1)], BF, seed=10, gate=True)
    page = table[0][150 // 16]
    for where in ("v", "k", "both"):
        if where != "k":
            c["v_cache"][page, :, 150 % 16, 5] = bad
        if where != "v":
            c["k_cache"][page, :, 150 % 16, 7] = bad
        out = _run_attention(c)
        want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs, layout[2] ** -0.5,
                                            c["gate"])
        assert torch.equal(torch.isfinite(out), torch.isfinite(want))
        bound = ref.attention_bound(want, spread, score, BF, layout[2], 400, 6.0)
        ok = torch.isfinite(want)
        assert bool(((out.double() - want).abs() <= bound)[ok].all())
        if where == "v":
            c["v_cache"][page, :, 150 % 16, 5] = 1.0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout,seqs", [((16, 2, 256), [(230, 1), (64, 1), (5000, 2)]), ((8, 2, 64), [(90, 4), (3, 3)]),
                                         ((32, 8, 128), [(700, 1), (300, 8)]), ((16, 2, 256), [(230, 20), (700, 1)])])
def test_attention_infinite_values_that_a_row_sees(device, dtype, layout, seqs):
    # A visible infinite value times a weight is infinite, as in the formula.
    c, table, starts, kvs = _case(device, *layout, 16, seqs, dtype, seed=29, gate=True)
    for s, (kv, n) in enumerate(seqs):
        for p in {0, (kv - n) // 2, kv - n}:
            row = c["v_cache"][table[s][p // 16], :, p % 16]
            row[:, 5], row[:, 9], row[:, 11] = math.inf, -math.inf, math.nan
    out = _run_attention(c, max_new=max(n for _, n in seqs))
    want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs, layout[2] ** -0.5,
                                        c["gate"])
    top = float(c["v_cache"][torch.isfinite(c["v_cache"])].abs().max())
    bound = ref.attention_bound(want, spread, score, dtype, layout[2], max(kvs), top)
    ok = torch.isfinite(want)
    assert bool((~ok).any()) and torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.double()[torch.isinf(want)], want[torch.isinf(want)])
    assert bool(((out.double() - want).abs() <= bound)[ok].all())
