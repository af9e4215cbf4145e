"""Calls of the paged-cache operators that are settled on the host (no GPU)."""

from __future__ import annotations

import pytest
import torch

from lightreason_amd import paged


def test_plans_belong_to_their_pool():
    a, b = (paged.PageTable(2, 10, 16, device="cpu") for _ in range(2))
    plan = b.new_plan(4)
    with pytest.raises(ValueError, match="pool"):
        a.commit(plan)
    with pytest.raises(ValueError, match="pool"):
        a.plan(torch.ones(2, dtype=torch.int32), 4, out=plan)
    cache = torch.zeros(10, 2, 16, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="pool"):
        paged.paged_layer(None, torch.zeros(4, 2048, dtype=torch.bfloat16), None, None, cache, cache, a, plan)
