"""The page pool under calls that its documentation allows: plans that replace
each other, plans of other pools, and rows whose lengths do not fit their pages."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x, device, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=device)


def _whole(pt):
    """Every page belongs to exactly one row or to the free stack."""
    held, table, count = pt.held.tolist(), pt.table.tolist(), pt.state[0].item()
    owned = [p for r, h in enumerate(held) for p in table[r][:h]]
    return sorted(owned + pt.free_pages[:count].tolist()) == list(range(pt.pages))


@pytest.mark.parametrize("first,second", [([1, 1], [0, 1]), ([0, 17], [1, 1]), ([1, 0], [0, 0]), ([3, 3], [3, 3])])
def test_a_plan_that_a_later_one_replaced_is_refused(device, first, second):
    from lightreason_amd.paged import PageTable

    pt = PageTable(2, 6, 16, device=device)
    a = pt.plan(_ints(first, device), 20)
    b = pt.plan(_ints(second, device), 20)
    pt.commit(a)   # its table entries are the second plan's now
    assert pt.state.tolist()[:3] == [6, 0, 8] and pt.lengths.tolist() == [0, 0] and pt.held.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="older"):
        pt.check()
    pt.state[2] = 0
    pt.commit(b)
    pt.check()
    assert pt.lengths.tolist() == second and _whole(pt)
    table = pt.table.tolist()
    assert b.slots.tolist()[:sum(second)] == [table[r][i // 16] * 16 + i % 16
                                              for r, n in enumerate(second) for i in range(n)]


def test_a_refused_plan_replaces_none(device):
    from lightreason_amd.paged import PageTable

    pt = PageTable(2, 6, 16, device=device)
    a = pt.plan(_ints([20, 3], device), 23)
    refused = pt.plan(_ints([20, 300], device), 400)
    assert refused.info[0].item() != 0
    pt.commit(a)
    pt.check()
    assert pt.lengths.tolist() == [20, 3] and _whole(pt)


def test_outputs_that_no_plan_was_made_into_are_refused(device):
    from lightreason_amd.paged import PageTable

    pt = PageTable(2, 6, 16, device=device)
    pt.commit(pt.plan(_ints([5, 1], device), 6))
    pt.commit(pt.new_plan(4))
    assert pt.state[2].item() == 8 and pt.lengths.tolist() == [5, 1]
    fresh = PageTable(2, 6, 16, device=device)
    fresh.commit(fresh.new_plan(4))
    assert fresh.state.tolist()[:3] == [6, 0, 8]


def test_plans_of_other_pools_are_refused(device):
    from lightreason_amd.paged import PageTable, paged_layer

    a, b = (PageTable(2, 6, 16, device=device) for _ in range(2))
    pa, pb = a.plan(_ints([3, 1], device), 4), b.plan(_ints([1, 1], device), 4)
    with pytest.raises(ValueError, match="pool"):
        b.commit(pa)
    with pytest.raises(ValueError, match="pool"):
        a.plan(_ints([1, 1], device), 4, out=pb)
    kc, vc = a.new_cache(1)
    with pytest.raises(ValueError, match="pool"):
        paged_layer(None, torch.zeros(4, 2048, dtype=torch.bfloat16, device=device), None, None, kc[0], vc[0], a, pb)
    a.commit(pa)
    b.commit(pb)
    assert a.lengths.tolist() == [3, 1] and b.lengths.tolist() == [1, 1]


def test_captured_plans_number_themselves(device):
    from lightreason_amd.paged import PageTable

    pt = PageTable(3, 40, 8, device=device)
    new, plan = torch.zeros(3, dtype=torch.int32, device=device), pt.new_plan(30)
    pt.plan(new, 30, out=plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pt.plan(new, 30, out=plan)
        pt.commit(plan)
    lengths = [0, 0, 0]
    for step in ([1, 9, 0], [8, 1, 1], [0, 0, 17]):
        new.copy_(_ints(step, device))
        between = pt.plan(new, 30)   # the program's own plan of the same step
        graph.replay()
        pt.commit(between)
        lengths = [a + b for a, b in zip(lengths, step)]
        assert pt.lengths.tolist() == lengths and pt.state[2].item() == 8 and _whole(pt)
        pt.state[2] = 0


def test_rows_longer_than_their_pages_are_refused(device):
    from lightreason_amd.paged import PageTable

    pt = PageTable(3, 30, 16, device=device)
    pt.commit(pt.plan(_ints([40, 16, 0], device), 56))
    for lengths, ok in (([48, 16, 0], True), ([49, 16, 0], False), ([40, 17, 0], False), ([40, 16, 1], False)):
        pt.lengths.copy_(_ints(lengths, device))
        plan = pt.plan(_ints([0, 0, 1], device), 4)
        assert plan.info.tolist()[:3] == ([0, 1, 1] if ok else [2, 0, 0])


def test_long_rows_without_pages_do_not_wrap_the_count(device):
    # 16 rows of 2^30 positions on pages of 8: their missing pages, 2^31, pass 31 bits.
    from lightreason_amd.paged import PageTable

    pt = PageTable(17, 30, 8, max_pages=4, device=device)
    pt.max_pages = 1 << 27   # what the rows may hold; nothing is read past the pages that a row has
    pt.lengths[:16] = 1 << 30
    plan = pt.plan(_ints([0] * 16 + [1], device), 4)
    assert plan.info.tolist()[:3] == [2, 0, 0] and set(plan.slots.tolist()) == {-1}
