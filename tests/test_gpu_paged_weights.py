"""Paged attention at the ends of its types' ranges, against the definition.
Bounds as in paged_ref.py."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF, HF, _case, _one_element, _run_attention

pytestmark = pytest.mark.gpu


# ---- attention: weights stay within their type ------------------------------------

@pytest.mark.parametrize("layout", [(16, 2, 256), (6, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("kv,n", [(300, 1), (300, 100)])
def test_attention_weights_where_fp32_is_coarse(device, layout, kv, n):
    # Scores near 1.5e8 in powers of two, where neighbouring fp32 numbers are 16
    # apart: from position 128 on they are one step higher.  2^16 is no fp16
    # number.  All values are 1, so the result is the sum of the rounded weights
    # over that of the weights: a half step for the weights, one for the
    # result, and fp32 sums of kv terms.
    c, table, *_ = _case(device, *layout, 16, [(kv, n)], HF, seed=28)
    _one_element(c, 49152.0, [49152.0] * kv)
    c["q"][..., 1] = 16.0
    for p in range(kv):
        c["k_cache"][table[0][p // 16], :, p % 16, 1] = 16.0 if p >= 128 else 0.0
    c["v_cache"].masked_fill_(torch.isfinite(c["v_cache"]), 1.0)
    got = _run_attention(c, max_new=n, scale=0.0433)
    assert bool(((got.double() - 1.0).abs() <= 2 * ref.half_step(HF) + kv * 2.0 ** -23).all())


# ---- attention: many small weights ------------------------------------------------

@pytest.mark.parametrize("layout,kv,n", [((2, 1, 64), 60001, 1), ((16, 2, 256), 30001, 2), ((8, 1, 128), 30001, 40),
                                         ((16, 2, 256), 9001, 700)])
def test_attention_fp16_small_weights_count(device, layout, kv, n):
    # Every 32nd position has value 0 and the highest score, all others are 18
    # below it: weights of 2^-26 of its, 31 for each, are the whole result.
    # Relative to a point 2^7 or more below the highest, fp16 weights keep
    # steps of 2^-24: half of one for each weight is 2^-32 of the highest, for
    # 32 positions to each highest, with values of 30000; then the roundings
    # of attention_bound for the result, the weights' sizes and the scores.
    c, table, starts, kvs = _case(device, *layout, 64, [(kv, n)], HF, seed=27)
    _one_element(c, 1.0, [18.0 if p % 32 == 0 else 0.0 for p in range(kv)])
    c["v_cache"].masked_fill_(torch.isfinite(c["v_cache"]), 30000.0)
    for p in range(0, kv, 32):
        c["v_cache"][table[0][p // 64], :, p % 64] = 0.0
    got = _run_attention(c, max_new=n, scale=1.0)
    want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs, 1.0)
    h, D = ref.half_step(HF), layout[2]
    soft = 2 * (D + 4) * 2.0 ** -24 * score + 2 * kv * 2.0 ** -24 + 2.0 ** -20
    bound = h * want.abs() * (1 + 2.0 ** -6) + (h + soft) * spread + 32 * 2.0 ** -32 * 30000.0 + 2.0 ** -25
    assert float(want.min()) > 0.01   # what was lost when they vanished
    assert bool(((got.double() - want).abs() <= bound).all())


# ---- attention: weights in two parts ----------------------------------------------

@pytest.mark.parametrize("layout,seqs", [
    ((16, 2, 256), [(1, 1), (2, 1), (33, 1), (200, 1), (777, 1), (3000, 1)]),
    ((16, 2, 256), [(2, 2), (5, 3), (100, 4), (129, 4), (1000, 4), (64, 3)]),
    ((32, 8, 128), [(40, 8), (700, 7), (1500, 1)]), ((6, 2, 128), [(3, 3), (900, 10)]),
    ((8, 8, 64), [(32, 32), (600, 27)]), ((8, 1, 64), [(90, 4), (5000, 1)])])
def test_attention_of_few_rows_is_as_good_as_its_rounding(device, layout, seqs):
    # A bf16 weight is the upper half of its bits and the rounded rest: 2^-7 of
    # the weight at most, so 2^-7 h of it off.  Else as attention_bound: the
    # result's own rounding, scores, exponentials and sums in fp32.
    c, table, starts, kvs = _case(device, *layout, 16, seqs, BF, seed=51, gate=True)
    rows = max(n for _, n in seqs)
    assert rows * (layout[0] // layout[1]) <= 32
    got = _run_attention(c, max_new=rows)
    D, h = layout[2], ref.half_step(BF)
    want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs, D ** -0.5, c["gate"])
    soft = 2 * (D + 4) * 2.0 ** -24 * score + 2 * max(kvs) * 2.0 ** -24 + 2.0 ** -20
    bound = h * want.abs() * (1 + 2.0 ** -6) + (2.0 ** -7 * h + soft) * spread + 1e-30
    assert bool(((got.double() - want).abs() <= bound).all())
