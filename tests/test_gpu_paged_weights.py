"""Paged attention at the ends of its types' ranges, against the definition.
Bounds as in paged_ref.py."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import HF, _case, _one_element, _run_attention

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
