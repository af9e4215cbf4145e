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


def test_commit_of_blocks_refuses_before_any_launch():
    from lightreason_amd import _native

    lib, p = _native.library(), 256
    assert lib.lrmoe_page_commit_drafts(-1, *([p] * 9), None) == -1
    assert lib.lrmoe_page_commit_drafts(4097, *([p] * 9), None) == -1
    for i in range(9):
        assert lib.lrmoe_page_commit_drafts(1, *([p] * i + [None] + [p] * (8 - i)), None) == -1
    assert lib.lrmoe_page_commit_drafts(0, *([None] * 9), None) == 0
    pt = paged.PageTable(2, 10, 16, device="cpu")
    with pytest.raises(ValueError, match="accepted"):
        pt.commit(pt.new_plan(4), starts=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("first,others", [(1, (1.0, True)), (0, (False, 0.0)), (2.0, (2,)), (None, (0, False))])
def test_checked_forms_tell_types_apart(first, others):
    from lightreason_amd import _native

    forms, t = {}, torch.zeros(2, 3)
    key, form = _native.checked(forms, (t, None), first)
    assert form is None
    _native.remember(forms, key, "checked")
    assert _native.checked(forms, (t, None), first)[1] == "checked"
    for other in others:
        assert _native.checked(forms, (t, None), other)[1] is None
