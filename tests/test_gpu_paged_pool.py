"""The page pool under calls that its documentation allows: plans that replace
each other, plans of other pools, rows whose lengths do not fit their pages, and
commits of steps that mix prompts with verify blocks."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref

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


def test_accepted_counts_of_any_size(device):
    from lightreason_amd.paged import PageTable

    pt = PageTable(4, 10, 16, device=device)
    plan = pt.plan(_ints([5, 7, 0, 3], device), 15)
    pt.commit(plan, _ints([2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 1, -2 ** 31], device))
    assert pt.lengths.tolist() == [5, 7, 0, 1]


def test_a_step_of_prompts_and_verify_blocks(device):
    """Prompts, a chunk of a prompt that goes on, verify blocks, a decode
    position and rows that rest: probabilities only where something is drawn."""
    from lightreason_amd.paged import PageTable
    from lightreason_amd.verify import verify_drafts

    g = torch.Generator(device=device).manual_seed(1)
    pt = PageTable(7, 100, 16, device=device)
    pt.commit(pt.plan(_ints([0, 10, 30, 16, 50, 0, 5], device), 111))
    #        prompt, chunk, verify, verify, decode, rests, prompt of one
    new = [40, 25, 5, 4, 1, 0, 1]
    drawn = [1, 0, 5, 4, 1, 0, 1]   # rows of probabilities
    plan = pt.plan(_ints(new, device), 80)
    starts = [0]
    for n in drawn:
        starts.append(starts[-1] + n)
    N, vocab = starts[-1], 300
    target = torch.softmax(torch.empty(N, vocab, device=device).normal_(0, 2, generator=g), 1)
    draft = target.clone()   # drafts stand ...
    tokens = torch.multinomial(draft, 1, generator=g)[:, 0]
    tokens[1:] = tokens[:-1].clone()
    target[starts[2] + 2, tokens[starts[2] + 3]] = 0.0   # ... but for the third of the first block
    uniforms, samples = torch.rand(N, generator=g, device=device), torch.rand(7, generator=g, device=device)
    blocks = _ints(starts, device)
    accepted, token = verify_drafts(tokens, target, blocks, uniforms, samples, draft=draft)
    want = ref.verify(tokens, target, starts, uniforms.tolist(), samples.tolist(), draft)
    assert accepted.tolist() == want[0] == [0, 0, 2, 3, 0, 0, 0] and token.tolist() == want[1]
    pt.commit(plan, accepted, starts=blocks)
    pt.check()
    assert pt.lengths.tolist() == [40, 35, 33, 20, 51, 0, 6] and _whole(pt)
    # blocks that are the step's own: as without starts
    plan = pt.plan(_ints([3, 0, 2, 1, 1, 4, 1], device), 12)
    accepted = _ints([1, 0, 1, 0, 0, 0, 0], device)
    pt.commit(plan, accepted, starts=plan.starts)
    assert pt.lengths.tolist() == [42, 35, 35, 21, 52, 1, 7]
    # starts that fit no step: growth stays within 1 .. n
    plan = pt.plan(_ints([3, 2, 1, 0, 0, 0, 0], device), 6)
    pt.commit(plan, _ints([0, 9, -5, 0, 0, 0, 0], device), starts=_ints([0, 100, 50, 2 ** 31 - 1, -9, 0, 0, 0], device))
    assert pt.lengths.tolist() == [43, 37, 36, 21, 52, 1, 7]
    for bad in (blocks[:-1], blocks.long(), blocks.cpu()):
        with pytest.raises(ValueError):
            pt.commit(plan, accepted, starts=bad)
    with pytest.raises(ValueError, match="accepted"):
        pt.commit(plan, starts=blocks)
