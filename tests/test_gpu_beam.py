"""Beam selection and forks of rows and pages on an MI355X against plain forms
in Python and float64."""

from __future__ import annotations

import math
import random

import pytest
import torch

from lightreason_amd import _native
from lightreason_amd.beam import beam_select, fork_rows
from lightreason_amd.paged import PageTable

pytestmark = pytest.mark.gpu

INF = math.inf


def _select(logits, scores, finished=None):
    """The choice in float64, group by group."""
    G, W = scores.shape
    V = logits.shape[1]
    rows = logits.double().cpu()
    tokens, parents, best = [], [], []
    for g in range(G):
        found = []
        for w in range(W):
            s = float(scores[g, w])
            if not math.isfinite(s):
                continue
            if finished is not None and finished[g, w]:
                found.append((-s, w * V, w, -1))
                continue
            x = rows[g * W + w]
            finite = torch.isfinite(x).nonzero()[:, 0]
            if len(finite) == 0:
                continue
            # (Relative to the largest: next to -3e38 the sum's logarithm would be lost.)
            above = x[finite] - x[finite].max()
            logp = above - torch.log(torch.exp(above).sum()) + s
            value, order = torch.sort(logp, descending=True, stable=True)
            found += [(-v, w * V + t, w, t) for v, t in zip(value[:W].tolist(), finite[order[:W]].tolist())]
        found = sorted(found)[:W]
        place = [None] * W
        for e in found:
            if place[e[2]] is None:
                place[e[2]] = e
        spare = [w for w in range(W) if place[w] is None]
        for e in found:
            if place[e[2]] is not e:
                place[spare.pop(0)] = e
        tokens.append([-1 if e is None else e[3] for e in place])
        parents.append([g * W + (w if e is None else e[2]) for w, e in enumerate(place)])
        best.append([-INF if e is None else -e[0] for e in place])
    return torch.tensor(tokens), torch.tensor(parents), torch.tensor(best, dtype=torch.float64)


def _check(logits, scores, finished=None):
    tokens, parents, best = beam_select(logits, scores, finished=finished)
    t, p, b = _select(logits, scores, finished)
    assert tokens.dtype == torch.int64 and parents.dtype == torch.int32 and best.dtype == torch.float32
    assert torch.equal(tokens.cpu(), t) and torch.equal(parents.cpu().long(), p)
    got = best.double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(b))
    ok = torch.isfinite(b)
    # One rounding to fp32 of the score; the sum of exponentials: each within
    # 2^-22 (a product of up to 2^7 rounded, and the exponential's own step) and
    # 38 additions, so 2^-18 relative at most and as much of the logarithm.
    assert ((got[ok] - b[ok]).abs() <= b[ok].abs() * 2.0 ** -24 + 2.0 ** -18).all()


def _logits(rows, vocab, dtype, seed, device):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * 2.5).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 4, 3), (2, 3, 65), (3, 8, 2047), (2, 5, 2049), (1, 16, 8193),
                                               (2, 32, 5000), (4, 2, 50001), (1, 4, 151936)])
def test_best_continuations(device, dtype, groups, beams, vocab):
    logits = _logits(groups * beams, vocab, dtype, vocab + beams, device)
    scores = (-torch.rand(groups, beams, generator=torch.Generator().manual_seed(beams)) * 6).to(device)
    _check(logits, scores)
    scores[:, 1:] = -INF    # a first step
    _check(logits, scores)


def test_ties_go_to_the_lowest_beam_and_token(device):
    """Coarse logits, equal beams, rows that are the same everywhere."""
    logits = torch.randint(-2, 3, (12, 6000), generator=torch.Generator().manual_seed(1)).float().to(device)
    logits[4:8] = logits[4:5]
    logits[8:] = 0.0
    for dtype in (torch.float32, torch.bfloat16):
        _check(logits.to(dtype), torch.zeros(3, 4, device=device))
    zeros = torch.zeros(2, 4097, device=device)
    zeros[:, ::2] = -0.0
    tokens, parents, _ = beam_select(zeros, torch.zeros(1, 2, device=device))
    assert tokens.tolist() == [[0, 1]] and parents.tolist() == [[0, 0]]


def test_logits_and_scores_that_are_not_finite(device):
    logits = _logits(8, 3000, torch.float32, 3, device)
    logits[0, 5:] = -INF          # five tokens left
    logits[1] = -INF              # none
    logits[2, 7] = INF
    logits[2, 8] = float("nan")
    logits[3] = float("nan")
    logits[4, 1:] = torch.finfo(torch.float32).min
    logits[5] = torch.finfo(torch.float32).min
    logits[6, :2900] = -INF
    scores = torch.tensor([[-1.0, 0.0, -2.0, 0.0], [-3.0, -1.0, -0.5, -INF]], device=device)
    _check(logits, scores)
    for bad in (float("nan"), INF, -INF):
        _check(logits, torch.full((2, 4), bad, device=device))
        mixed = scores.clone()
        mixed[0, 0] = bad
        _check(logits, mixed)


def test_finished_beams(device):
    logits = _logits(12, 700, torch.bfloat16, 4, device)
    scores = (-torch.rand(3, 4, generator=torch.Generator().manual_seed(4)) * 3).to(device)
    finished = torch.zeros(3, 4, dtype=torch.bool, device=device)
    finished[0, 1] = finished[1, :] = finished[2, 0] = finished[2, 3] = True
    scores[2, 3] = -INF
    _check(logits, scores, finished)
    _check(logits, scores, finished.to(torch.uint8))
    logits[0] = float("nan")      # a finished beam's logits are not looked at
    finished[0, 0] = True
    _check(logits, scores, finished)


def test_strided_rows_and_unaligned_ones(device):
    wide = _logits(6, 4100, torch.bfloat16, 5, device)
    scores = -torch.arange(6.0, device=device).view(2, 3) / 7
    for view in (wide[:, 1:4000], wide[:, 3:3003], wide[:, 8:4096]):
        _check(view, scores)
    _check(wide.float()[:, 1:3000], scores)


def test_scores_in_place_of_graph_replays(device):
    """A captured search step whose scores, logits and flags change."""
    logits = _logits(8, 9000, torch.float32, 6, device)
    scores = torch.zeros(2, 4, device=device)
    finished = torch.zeros(2, 4, dtype=torch.bool, device=device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        beam_select(logits, scores, finished=finished)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = beam_select(logits, scores, finished=finished)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(4):
        logits.copy_(_logits(8, 9000, torch.float32, 60 + i, device))
        finished[i % 2, i] = True
        want = beam_select(logits, scores, finished=finished)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        scores.copy_(got[2])


# ---- rows -------------------------------------------------------------------------

def _parents(rng, rows, moved=0.5):
    keeps = [rng.random() >= moved for _ in range(rows)]
    keeps[rng.randrange(rows)] = True
    stay = [r for r in range(rows) if keeps[r]]
    return [r if keeps[r] else rng.choice(stay) for r in range(rows)]


@pytest.mark.parametrize("rows", [1, 2, 7, 40])
def test_rows_follow_their_parents(device, rows):
    rng = random.Random(rows)
    parents = _parents(rng, rows)
    index = torch.tensor(parents, dtype=torch.int32, device=device)
    gen = torch.Generator().manual_seed(rows)
    tensors = [torch.randn(rows, 4, 64, 64, generator=gen).to(device),
               torch.randn(rows, 1001, 4, generator=gen).bfloat16().to(device),
               torch.randint(100, (rows,), generator=gen).to(device),
               torch.rand(rows, 3, generator=gen).lt(0.5).to(device),
               torch.randn(rows, 33, generator=gen).half().to(device)[:, 1:],    # strided rows
               torch.randn(rows, 0, generator=gen).to(device),
               torch.randn(rows, 70001, generator=gen).to(device)]
    tensors += [torch.randn(rows, 5, generator=gen).to(device) for _ in range(70)]
    want = [t[index.long()].clone() for t in tensors]
    fork_rows(index, tensors)
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)
    fork_rows(index, tensors[0])      # again: nothing changes
    assert torch.equal(tensors[0], want[0])


def test_parents_that_move_themselves_are_left_out(device):
    t = torch.arange(6.0, device=device)[:, None].repeat(1, 9)
    parents = torch.tensor([1, 0, 2, 2, 9, -1], dtype=torch.int32, device=device)
    fork_rows(parents, [t])
    assert t[:, 0].tolist() == [0.0, 1.0, 2.0, 2.0, 4.0, 5.0]


# ---- pages ------------------------------------------------------------------------

def _pool(device, rows=6, pages=40, page=16, lengths=(20, 20, 33, 0, 16, 1), heads=2, dim=64, layers=2):
    pool = PageTable(rows, pages, page, max_pages=6, device=device)
    caches = pool.new_cache(layers, heads, dim)
    for c in caches:
        c.copy_(torch.randn(c.shape, generator=torch.Generator().manual_seed(1)))
    new = torch.tensor(lengths, dtype=torch.int32, device=device)
    pool.commit(pool.plan(new, sum(lengths)))
    return pool, caches


def _content(pool, caches, row):
    n = int(pool.lengths[row])
    pages = pool.table[row, :-(-n // pool.page)].long()
    return [c[:, pages].transpose(1, 2).reshape(c.shape[0], c.shape[2], -1, c.shape[4])[:, :, :n].clone() for c in caches]


@pytest.mark.parametrize("parents", [[0, 0, 2, 2, 0, 5], [2, 2, 2, 2, 2, 2], [0, 1, 2, 3, 4, 5], [0, 1, 3, 3, 3, 3]])
def test_rows_take_over_pages(device, parents):
    pool, caches = _pool(device)
    before = [_content(pool, caches, r) for r in range(6)]
    held, free = pool.held.tolist(), int(pool.state[0])
    lengths = pool.lengths.tolist()
    pool.fork(torch.tensor(parents, dtype=torch.int32, device=device), *caches)
    pool.check()
    used = []
    for r, p in enumerate(parents):
        assert int(pool.lengths[r]) == lengths[p]
        need = -(-lengths[p] // 16) if p != r else 0
        assert int(pool.held[r]) == max(held[r], need)
        used += pool.table[r, :int(pool.held[r])].tolist()
        for got, want in zip(_content(pool, caches, r), before[p]):
            assert torch.equal(got, want)
    assert len(set(used)) == len(used)
    assert int(pool.state[0]) == free - (sum(pool.held.tolist()) - sum(held))
    assert sorted(used + pool.free_pages[:int(pool.state[0])].tolist()) == list(range(40))
    # The search goes on: a position per row, committed.
    plan = pool.plan(torch.ones(6, dtype=torch.int32, device=device), 6)
    pool.commit(plan)
    pool.check()
    assert pool.lengths.tolist() == [lengths[p] + 1 for p in parents]
    slots = plan.slots.tolist()
    assert len(set(slots)) == 6
    pool.release(torch.ones(6, dtype=torch.bool, device=device))
    pool.check()
    assert int(pool.state[0]) == 40


def test_forks_that_are_refused_change_only_the_status(device):
    for parents, pages, bit in (([1, 0, 2, 3, 4, 5], 40, _native.PAGE_STATUS_ROW),
                                ([0, 0, 2, 3, 4, 6], 40, _native.PAGE_STATUS_ROW),
                                ([0, -1, 2, 3, 4, 5], 40, _native.PAGE_STATUS_ROW),
                                ([2, 2, 2, 2, 2, 2], 10, _native.PAGE_STATUS_POOL)):
        pool, caches = _pool(device, pages=pages)
        kept = [t.clone() for t in (pool.table, pool.held, pool.lengths, pool.state, *caches)]
        pool.fork(torch.tensor(parents, dtype=torch.int32, device=device), *caches)
        for a, b in zip((pool.table, pool.held, pool.lengths, *caches), kept[:3] + kept[4:]):
            assert torch.equal(a, b)
        assert pool.state.tolist() == [kept[3][0], kept[3][1], bit, kept[3][3]]
        with pytest.raises(RuntimeError):
            pool.check()


def test_a_plan_from_before_a_fork_is_stale(device):
    pool, caches = _pool(device)
    plan = pool.plan(torch.ones(6, dtype=torch.int32, device=device), 6)
    pool.fork(torch.tensor([0, 0, 2, 3, 4, 5], dtype=torch.int32, device=device), *caches)
    pool.commit(plan)
    assert pool.status() == _native.PAGE_STATUS_STALE


def test_speculative_pages_and_one_layer_caches(device):
    """A row that holds more pages than its length needs keeps them; caches of
    one layer, strided, of another width."""
    pool, caches = _pool(device)
    pool.lengths[2] = 17
    pool.lengths[0] = 16
    parents = torch.tensor([0, 1, 2, 3, 0, 2], dtype=torch.int32, device=device)
    wide = torch.randn(40, 3, 16, 72, device=device).half()
    one = wide[..., 8:]
    want = [_content(pool, caches + (one[None],), r) for r in range(6)]
    edge = wide[..., :8].clone()
    pool.fork(parents, caches[0], one, caches[1])
    pool.check()
    assert pool.held.tolist() == [2, 2, 3, 0, 1, 2]
    for r, p in enumerate(parents.tolist()):
        for a, b in zip(_content(pool, caches + (one[None],), r), want[p]):
            assert torch.equal(a, b)
    assert torch.equal(wide[..., :8], edge)
    pool.fork(parents)     # lengths and pages alone
    pool.check()


def test_many_rows(device):
    rng = random.Random(3)
    R = 1500
    lengths = [rng.randrange(0, 40) for _ in range(R)]
    pool = PageTable(R, 6000, 16, max_pages=3, device=device)
    caches = pool.new_cache(1, 1, 64)
    for c in caches:
        c.copy_(torch.randn(c.shape, generator=torch.Generator().manual_seed(2)))
    pool.commit(pool.plan(torch.tensor(lengths, dtype=torch.int32, device=device), sum(lengths)))
    before = [_content(pool, caches, r) for r in range(R)]
    parents = _parents(rng, R)
    pool.fork(torch.tensor(parents, dtype=torch.int32, device=device), *caches)
    pool.check()
    assert pool.lengths.tolist() == [lengths[p] for p in parents]
    for r, p in enumerate(parents):
        for a, b in zip(_content(pool, caches, r), before[p]):
            assert torch.equal(a, b), r


def test_forks_of_more_rows_than_a_call_counts(device):
    """Tensors that need several calls by their pieces, and one that fits none: it
    is refused, and nothing has moved."""
    rows = 1 << 22
    parents = torch.arange(rows, dtype=torch.int32, device=device)
    parents[1::2] -= 1
    tensors = [torch.randint(0, 2**15, (rows,), device=device, dtype=torch.int16) for _ in range(5)]
    before = [t.clone() for t in tensors]
    fork_rows(parents, tensors)
    for t, b in zip(tensors, before):
        assert torch.equal(t, b[parents.long()])
    more = torch.zeros(1 << 24, 1, dtype=torch.uint8, device=device)
    parents = torch.arange(1 << 24, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="tensor 0 has"):
        fork_rows(parents, [more])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 16, 151936), (2, 32, 50001), (1, 32, 151936), (1, 9, 151936),
                                               (1, 8, 163840), (1, 8, 163841), (1, 1, 1400000)])
def test_more_candidates_than_a_wave_keeps_in_registers(device, dtype, groups, beams, vocab):
    """Slices times beams around and above what the join holds."""
    logits = _logits(groups * beams, vocab, dtype, vocab + beams, device)
    scores = (-torch.rand(groups, beams, generator=torch.Generator().manual_seed(beams)) * 6).to(device)
    _check(logits, scores)
    scores[:, 1:] = -INF    # a first step
    _check(logits, scores)


def test_ties_over_many_slices(device):
    """Equal values in every slice, and a few that are larger far apart."""
    logits = torch.randint(-2, 2, (32, 50001), generator=torch.Generator().manual_seed(2)).float().to(device)
    logits[:, 40000] = logits[:, 7] = 3.0
    logits[5:9] = 0.0
    logits[9, :] = -INF
    logits[9, ::4000] = 1.0
    for dtype in (torch.float32, torch.bfloat16):
        _check(logits.to(dtype), torch.zeros(1, 32, device=device))
        scores = torch.full((1, 32), -INF, device=device)
        scores[0, 9] = 0.0   # 13 continuations for 32 beams
        _check(logits.to(dtype), scores)
