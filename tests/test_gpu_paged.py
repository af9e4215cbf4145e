"""The paged-cache operators and the draft verification on the GPU against
their plain 64-bit forms (paged_ref.py): page plans, commits and releases,
the append, the attention over the whole range of step shapes, drafts, and a
speculative loop of all of them, eager and captured.

Integers are equal.  The append's values are within half a step of their
type of the 64-bit value, plus 2^-20 of the row's largest for the fp32 sums;
the attention's bound is derived in paged_ref.attention_bound."""

from __future__ import annotations

import math
import random

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _ints(x, device, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=device)


# ---- plan, commit, release --------------------------------------------------------

def _pool(device, rows, pages, page, max_pages, lengths, seed=0):
    from lightreason_amd.paged import PageTable

    pt = PageTable(rows, pages, page, max_pages=max_pages, device=device)
    held = [-(-n // page) for n in lengths]
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (max_pages - h))
        at += h
    free = order[at:]
    pt.table.copy_(_ints(table, device))
    pt.held.copy_(_ints(held, device))
    pt.lengths.copy_(_ints(lengths, device))
    pt.free_pages[:len(free)] = _ints(free, device)
    pt.state[0] = len(free)
    return pt, held, table, free


@pytest.mark.parametrize("rows,page,spread,room", [(1, 8, 1, 0), (3, 16, 40, 7), (70, 64, 300, 1), (257, 16, 33, 0),
                                                   (1000, 32, 20, 100), (4096, 16, 9, 3)])
def test_plan_matches_the_list_form(device, rows, page, spread, room):
    rng = random.Random(rows)
    lengths = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 6 * page)]) for _ in range(rows)]
    new = [rng.choice([0, 1, 1, rng.randint(0, spread)]) for _ in range(rows)]
    width = max(-(-(c + n) // page) for c, n in zip(lengths, new)) + 1
    pages = sum(-(-(c + n) // page) for c, n in zip(lengths, new)) + 2
    pt, held, table, free = _pool(device, rows, pages, page, width, lengths, seed=rows)
    starts, kv, held2, positions, slots, table2, free2 = ref.plan(new, lengths, held, table, free, page)
    tokens = sum(new) + room
    for _ in range(2):   # a plan made twice is the same plan
        plan = pt.plan(_ints(new, device), tokens)
        assert plan.info.tolist()[:3] == [0, sum(new), len(free) - len(free2)]
        assert plan.starts.tolist() == starts and plan.kv_lengths.tolist() == kv and plan.held.tolist() == held2
        assert plan.positions.tolist() == positions + [0] * room
        assert plan.slots.tolist() == slots + [-1] * room
        assert pt.table.tolist() == table2
        assert pt.held.tolist() == held and pt.lengths.tolist() == lengths
    pt.commit(plan)
    assert pt.lengths.tolist() == kv and pt.held.tolist() == held2
    assert pt.state.tolist() == [len(free2), 1, 0, 0]
    pt.check()
    pt.commit(plan)   # a second commit of it is stale
    assert pt.lengths.tolist() == kv and pt.state.tolist()[:3] == [len(free2), 1, 8]
    with pytest.raises(RuntimeError, match="older"):
        pt.check()


@pytest.mark.parametrize("what,bit", [("tokens", 1), ("negative", 1), ("row", 2), ("length", 2), ("pool", 4)])
def test_plan_that_does_not_fit_changes_nothing(device, what, bit):
    page, lengths = 16, [5, 0, 33]
    pt, held, table, free = _pool(device, 3, 7, page, 4, lengths)
    new = {"tokens": [4, 4, 4], "negative": [1, -1, 1], "row": [0, 0, 32], "length": [1, 1, 1],
           "pool": [20, 50, 0]}[what]
    if what == "pool":
        pt.state[0] = 2
    if what == "length":
        pt.lengths[1] = -3
        lengths = [5, -3, 33]
    plan = pt.plan(_ints(new, device), 11 if what == "tokens" else 100)
    assert plan.info.tolist()[:3] == [bit, 0, 0]
    assert plan.starts.tolist() == [0] * 4 and plan.kv_lengths.tolist() == lengths and plan.held.tolist() == held
    assert set(plan.slots.tolist()) == {-1} and set(plan.positions.tolist()) == {0}
    assert pt.table.tolist() == table
    before = pt.state.tolist()
    pt.commit(plan)
    assert pt.lengths.tolist() == lengths and pt.state.tolist() == [before[0], 0, bit, 0]
    with pytest.raises(RuntimeError):
        pt.check()


def test_release_returns_pages_and_the_pool_stays_whole(device):
    rng = random.Random(3)
    rows, pages, page = 37, 150, 8
    from lightreason_amd.paged import PageTable

    pt = PageTable(rows, pages, page, max_pages=20, device=device)
    lengths = [0] * rows
    for step in range(30):
        new = [rng.randint(0, 6) if n + 6 < 20 * page else 0 for n in lengths]
        plan = pt.plan(_ints(new, device), 6 * rows)
        fits = plan.info[0].item() == 0
        pt.commit(plan)
        if fits:
            lengths = [a + b for a, b in zip(lengths, new)]
        else:
            pt.state[2] = 0
        mask = [rng.random() < (0.2 if fits else 0.6) for _ in range(rows)]
        stale = pt.plan(_ints([1] + [0] * (rows - 1), device), 4)
        pt.release(_ints(mask, device, torch.bool if step % 2 else torch.uint8))
        lengths = [0 if m else n for n, m in zip(lengths, mask)]
        assert pt.lengths.tolist() == lengths
        held, table, count = pt.held.tolist(), pt.table.tolist(), pt.state[0].item()
        owned = [p for r in range(rows) for p in table[r][:held[r]]]
        assert sorted(owned + pt.free_pages[:count].tolist()) == list(range(pages))   # no page lost or twice
        if stale.info[0].item() == 0:
            pt.commit(stale)
            assert pt.state[2].item() == 8 and pt.lengths.tolist() == lengths
            pt.state[2] = 0


def test_commit_with_accepted_counts(device):
    pt, *_ = _pool(device, 4, 40, 16, 8, [3, 0, 40, 7])
    plan = pt.plan(_ints([5, 0, 1, 9], device), 20)
    pt.commit(plan, _ints([2, 6, 0, 100], device))
    assert pt.lengths.tolist() == [3 + 3, 0, 40 + 1, 7 + 9]
    assert pt.held.tolist() == plan.held.tolist()


# ---- append -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,norm,rope32,nhd", [
    (16, 2, 256, 64, True, True, False), (16, 2, 256, 64, True, False, True), (8, 8, 64, 64, False, True, False),
    (5, 1, 128, 128, True, True, True), (0, 3, 128, 16, True, False, False), (4, 2, 64, 0, True, True, False),
    (2, 1, 256, 256, False, False, False)])
def test_append(device, dtype, heads, kv_heads, dim, rotary, norm, rope32, nhd):
    from lightreason_amd.paged import paged_append

    g = torch.Generator(device=device).manual_seed(dim + heads)
    N, page, pages = 77, 16, 9

    def normal(*shape):
        return torch.empty(shape, device=device).normal_(generator=g).to(dtype)
    shape = (pages, page, kv_heads, dim) if nhd else (pages, kv_heads, page, dim)
    kc, vc = normal(*shape), normal(*shape)
    if nhd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    rng = random.Random(dim)
    slots = rng.sample(range(pages * page), N)
    for i, s in ((5, -1), (6, pages * page), (76, -1)):   # padding and a slot outside the pool: left out
        slots[i] = s
    qg = normal(N, max(heads, 1), 2 * dim)
    qg[3] *= 30.0
    q = qg[:, :, :dim] if heads else None
    kv = normal(N, kv_heads, 2, dim)
    k, v = kv[:, :, 0], kv[:, :, 1]
    qn, kn = (0.1 * normal(dim).float()).to(dtype), (0.1 * normal(dim).float()).to(dtype)
    cos = sin = positions = None
    if rotary:
        angle = torch.rand(500, rotary // 2, device=device, generator=g) * 6.28
        angle = torch.cat([angle, angle], 1)
        cos, sin = angle.cos(), angle.sin()
        if not rope32:
            cos, sin = cos.to(dtype), sin.to(dtype)
        positions = _ints([rng.randint(0, 499) for _ in range(N)], device)
    kc0, vc0 = kc.clone(), vc.clone()
    out = torch.full((N, heads, dim), 7.0, dtype=dtype, device=device) if heads else None
    got = paged_append(k, v, kc, vc, _ints(slots, device, torch.int64), q=q, q_norm=qn if norm and heads else None,
                       k_norm=kn if norm else None, eps=1e-6, cos=cos, sin=sin, positions=positions, q_out=out)
    assert (got is None) == (heads == 0)
    live = [i for i, s in enumerate(slots) if 0 <= s < pages * page]
    c, s = (cos[positions.long()], sin[positions.long()]) if rotary else (None, None)

    def close(have, want):
        bound = ref.half_step(dtype) * want.abs() + 2.0 ** -20 * want.abs().amax(dim=-1, keepdim=True)
        if dtype == HF:
            bound = bound + 2.0 ** -25
        assert bool(((have.double() - want).abs() <= bound).all())
    wk, wv = kc0.double(), vc0.clone()
    rk = ref.norm_rope(k, kn if norm else None, c, s, 1e-6)
    for i in live:
        wk[slots[i] // page, :, slots[i] % page] = rk[i]
        wv[slots[i] // page, :, slots[i] % page] = v[i]
    assert torch.equal(vc, wv)
    close(kc, wk)
    written = torch.zeros(pages, page, dtype=torch.bool, device=device)
    for i in live:
        written[slots[i] // page, slots[i] % page] = True
    still = ~written[:, None, :, None].expand_as(kc)
    assert torch.equal(kc[still], kc0[still])
    if heads:
        rq = ref.norm_rope(q, qn if norm else None, c, s, 1e-6)
        close(out[live], rq[live])
        for i in set(range(N)) - set(live):
            assert bool((out[i] == 7.0).all())


def test_append_position_outside_the_rotary_table_is_nan(device):
    from lightreason_amd.paged import paged_append

    k = torch.ones(3, 1, 64, dtype=BF, device=device)
    kc, vc = torch.zeros(1, 1, 8, 64, dtype=BF, device=device), torch.zeros(1, 1, 8, 64, dtype=BF, device=device)
    cos = torch.ones(4, 16, device=device)
    paged_append(k, k, kc, vc, _ints([0, 1, 2], device, torch.int64), cos=cos, sin=cos,
                 positions=_ints([-1, 3, 4], device))
    nan = torch.isnan(kc[0, 0])
    assert nan[0, :16].all() and nan[2, :16].all() and not nan[1].any() and not nan[:, 16:].any()


def test_append_in_place_of_the_queries(device):
    from lightreason_amd.paged import paged_append

    x = torch.randn(9, 4, 128, dtype=BF, device=device)
    k = torch.randn(9, 2, 128, dtype=BF, device=device)
    kc, vc = torch.zeros(2, 2, 8, 128, dtype=BF, device=device), torch.zeros(2, 2, 8, 128, dtype=BF, device=device)
    cos = torch.rand(9, 32, device=device)
    slots = torch.arange(9, device=device)
    want = paged_append(k, k, kc, vc, slots, q=x, cos=cos, sin=cos)
    got = paged_append(k, k, kc, vc, slots, q=x, cos=cos, sin=cos, q_out=x)
    assert got is x and torch.equal(got, want)


# ---- attention --------------------------------------------------------------------

def _case(device, heads, kv_heads, dim, page, seqs, dtype, seed=0, gate=False, nhd=False, pad=0, extra=3):
    """seqs: (kv_length, new) pairs.  Positions past a row's length, and pages
    of nobody, hold NaN."""
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.empty(shape, device=device).normal_(generator=g).to(dtype)
    kvs, new = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // page) for n in kvs) + extra
    table = ref.block_table(kvs, page, pages, seed)
    shape = (pages, page, kv_heads, dim) if nhd else (pages, kv_heads, page, dim)
    kc, vc = normal(*shape), normal(*shape)
    if nhd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    dead = torch.ones(pages, page, dtype=torch.bool, device=device)
    for row, n in zip(table, kvs):
        for i in range(-(-n // page)):
            dead[row[i], :max(0, min(page, n - i * page))] = False
    for c in (kc, vc):
        c.masked_fill_(dead[:, None, :, None], math.nan)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    N = starts[-1] + pad
    both = normal(N, heads, 2 * dim)   # queries and gates interleaved, as one projection writes them
    q, gt = both[:, :, :dim], both[:, :, dim:]
    return dict(q=q, k_cache=kc, v_cache=vc, table=_ints(table, device), starts=_ints(starts, device),
                kv_lengths=_ints(kvs, device), gate=gt if gate else None), table, starts, kvs


def _run_attention(c, **kw):
    from lightreason_amd.paged import paged_attention

    return paged_attention(c["q"], c["k_cache"], c["v_cache"], c["table"], c["starts"], c["kv_lengths"],
                           gate=c["gate"], **kw)


def _check(c, table, starts, kvs, out, scale=None):
    dim = c["q"].shape[2]
    want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs,
                                        dim ** -0.5 if scale is None else scale, c["gate"])
    finite = c["v_cache"][torch.isfinite(c["v_cache"])]
    bound = ref.attention_bound(want, spread, score, out.dtype, dim, max(kvs + [1]), float(finite.abs().max()))
    live = slice(starts[0], starts[-1])
    off = (out.double() - want).abs()[live]
    same_nan = torch.isnan(out[live]) == torch.isnan(want[live])
    assert bool(same_nan.all())
    excess = torch.nan_to_num(off / bound[live], nan=0.0)
    worst = float(excess.max()) if excess.numel() else 0.0
    print(f"worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


LAYOUTS = [(16, 2, 256), (32, 8, 128), (8, 8, 64), (5, 1, 128), (6, 2, 256)]
STEPS = {
    "one": [(1, 1)],
    "decode": [(1, 1), (2, 1), (31, 1), (32, 1), (33, 1), (64, 1), (65, 1), (200, 1), (777, 1)],
    "idle": [(0, 0), (50, 1), (9, 0), (0, 0), (70, 2), (128, 0)],
    "verify": [(5, 5), (100, 4), (129, 9), (1000, 16), (64, 3)],
    "prompts": [(130, 130), (1, 1), (257, 257), (63, 63)],
    "chunks": [(700, 90), (513, 128), (300, 299), (1025, 1)],
    "nothing": [(3, 5), (0, 4), (40, 2)],   # more new positions than cached: rows that see nothing
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention(device, layout, step, dtype):
    seqs = STEPS[step]
    page = {256: 16, 128: 64, 64: 8}[layout[2]]
    c, table, starts, kvs = _case(device, *layout, page, seqs, dtype, seed=len(seqs), gate=step != "prompts",
                                  nhd=layout[0] == 32, pad=3)
    out = torch.full(c["q"].shape, 9.0, dtype=dtype, device=device)
    for max_new in (None, max(n for _, n in seqs)):
        got = _run_attention(c, out=out, max_new=max_new)
        assert got is out
        assert bool((out[starts[-1]:] == 9.0).all())   # tokens behind the last sequence
        _check(c, table, starts, kvs, out)
        assert torch.equal(out, _run_attention(c, out=out.clone(), max_new=max_new))   # the same bits again


@pytest.mark.parametrize("page", [8, 32, 128, 1024])
def test_attention_page_sizes(device, page):
    c, *rest = _case(device, 16, 2, 256, page, [(1500, 1), (page, 1), (page + 1, 40), (2 * page - 1, 7)], BF, seed=page)
    _check(c, *rest, _run_attention(c))


@pytest.mark.parametrize("seqs,layout", [([(40001, 1)], (16, 2, 256)), ([(30000, 7), (9, 1)], (16, 2, 256)),
                                         ([(20011, 600)], (16, 2, 256)), ([(33000, 1)], (32, 8, 128)),
                                         ([(12000, 12000 - 9000)], (4, 1, 64)), ([(9000, 1)] * 3, (64, 1, 128))])
def test_attention_long(device, seqs, layout):
    c, *rest = _case(device, *layout, 64, seqs, BF, seed=7, gate=True)
    _check(c, *rest, _run_attention(c, max_new=max(n for _, n in seqs)))


@pytest.mark.parametrize("seqs,layout,dtype", [([(2500, 2500), (1, 1), (700, 690)], (16, 2, 256), BF),
                                               ([(1900, 1900)], (7, 1, 128), HF), ([(5, 5), (4100, 1500)], (96, 2, 64), BF)])
def test_attention_prompts_of_many_split_counts(device, seqs, layout, dtype):
    # Tiles of one sequence with one split and with several.
    c, *rest = _case(device, *layout, 32, seqs, dtype, seed=23, gate=True, pad=1)
    _check(c, *rest, _run_attention(c, max_new=max(n for _, n in seqs)))


def test_attention_many_rows(device):
    rng = random.Random(5)
    seqs = [(rng.randint(1, 60), 1) if rng.random() < 0.8 else (rng.randint(0, 9), 0) for _ in range(1500)]
    c, *rest = _case(device, 8, 2, 64, 8, seqs, BF, seed=8)
    _check(c, *rest, _run_attention(c, max_new=1))


def test_attention_scale_and_large_scores(device):
    # Scores far apart: the running maximum moves by hundreds between tiles.
    c, *rest = _case(device, 16, 2, 256, 16, [(900, 1), (500, 70)], BF, seed=9)
    c["k_cache"][::3] *= 20.0
    _check(c, *rest, _run_attention(c, scale=0.25), scale=0.25)
    zero = _run_attention(c, scale=0.0)   # every position alike
    _check(c, *rest, zero, scale=0.0)


@pytest.mark.parametrize("layout", [(16, 2, 256), (8, 2, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_what_a_row_does_not_see(device, bad, layout):
    # Position 150 of one sequence (token 20 of a chunk that starts at 130) has
    # values and keys that are not finite: earlier tokens keep their results.
    c, table, starts, kvs = _case(device, *layout, 16, [(230, 100), (64, 4), (400, 1)], BF, seed=10, gate=True)
    clean = _run_attention(c)
    page = table[0][150 // 16]
    c["v_cache"][page, :, 150 % 16, 5] = bad
    c["k_cache"][page, :, 150 % 16, 7] = bad
    out = _run_attention(c)
    assert torch.equal(out[100:], clean[100:])
    want, spread, score = ref.attention(c["q"][:20], c["k_cache"], c["v_cache"], table, [0, 20], [150],
                                        layout[2] ** -0.5, c["gate"][:20])
    bound = ref.attention_bound(want, spread, score, BF, layout[2], 150, 6.0)
    assert bool(((out[:20].double() - want).abs() <= bound).all())
    # rows that see it: NaN where the 64-bit form has no finite value
    assert not bool(torch.isfinite(out[20:100, :, 5]).all())


def test_attention_bad_table_entries_make_their_rows_nan(device):
    c, table, starts, kvs = _case(device, 16, 2, 256, 16, [(100, 1), (90, 3), (80, 1), (300, 40)], BF, seed=11)
    clean = _run_attention(c)
    for row, entry in ((1, -1), (3, 10 ** 6)):
        c["table"][row, 2] = entry
    for max_new in (None, 40):
        out = _run_attention(c, max_new=max_new)
        assert bool(torch.isnan(out[1:4]).all()) and bool(torch.isnan(out[5:]).all())
        for keep in (0, 4):
            assert torch.equal(out[keep], clean[keep])
    c["table"][:, -1] = 10 ** 6   # entries past the rows' pages are not used
    c["table"][1, 2], c["table"][3, 2] = table[1][2], table[3][2]
    assert torch.equal(_run_attention(c), clean)


def test_attention_lengths_past_the_table_are_cut(device):
    c, table, starts, kvs = _case(device, 8, 2, 64, 8, [(16, 2), (24, 1)], BF, seed=12)
    c["table"] = c["table"][:, :3].contiguous()
    c["kv_lengths"][1] = 10 ** 9
    table = [r[:3] for r in table]
    _check(c, table, starts, [16, 24], _run_attention(c))


def test_attention_offsets_past_32_bits(device):
    # A cache of more than 2^31 elements, its last pages in use.
    pages, page, K, D = 70000, 64, 2, 256
    kc = torch.empty(pages, K, page, D, dtype=BF, device=device)
    vc = torch.empty_like(kc)
    seqs = [(150, 1), (200, 90)]
    table = [[69999, 69990, 69995, -1], [69998, 12, 69997, 69996]]
    for c in (kc, vc):
        for row in table:
            for p in row:
                c[p].normal_()
    q = torch.randn(91, 16, D, device=device).to(BF)
    c = dict(q=q, k_cache=kc, v_cache=vc, table=_ints(table, device), starts=_ints([0, 1, 91], device),
             kv_lengths=_ints([150, 200], device), gate=None)
    from lightreason_amd.paged import paged_append

    slots = _ints([69999 * 64 + 5, 69996 * 64 + 7], device, torch.int64)
    k = torch.randn(2, K, D, device=device).to(BF)
    paged_append(k, k, kc, vc, slots)
    assert torch.equal(kc[69999, :, 5], k[0]) and torch.equal(vc[69996, :, 7], k[1])
    out = _run_attention(c)
    want, spread, score = ref.attention(q, kc, vc, table, [0, 1, 91], [150, 200], D ** -0.5)
    bound = ref.attention_bound(want, spread, score, BF, D, 200, 8.0)
    assert bool(((out.double() - want).abs() <= bound).all())


def test_attention_over_as_many_positions_as_a_row_can_hold(device):
    # 2^30 positions, all in two pages: the attention over those 2048.  The
    # longest chain of fp32 sums is a wave's share of a split, 2^18 at most.
    c, table, starts, _ = _case(device, 2, 1, 64, 1024, [(2048, 2)], BF, seed=22)
    c["table"] = c["table"][:, :2].repeat(1, 1 << 19).contiguous()
    c["kv_lengths"] = _ints([1 << 30], device)
    got = _run_attention(c, max_new=2)
    want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, [2048], 64 ** -0.5)
    bound = ref.attention_bound(want, spread, score, BF, 64, 1 << 18, 0.0)
    assert bool(((got.double() - want).abs() <= bound)[1:].all())


@pytest.mark.parametrize("layout", [(16, 2, 256), (12, 3, 128), (1, 1, 64)])
def test_attention_strided_caches_and_output(device, layout):
    # Keys and values side by side in one pool of pages, rows of all heads
    # together; the output one half of a wider buffer.
    heads, K, D = layout
    c, table, starts, kvs = _case(device, *layout, 16, [(77, 1), (333, 50), (1000, 3)], BF, seed=13, gate=True)
    pages, page = c["k_cache"].shape[0], 16
    pool = torch.empty(pages, page, 2, K, D, dtype=BF, device=device)
    pool[:, :, 0], pool[:, :, 1] = c["k_cache"].transpose(1, 2), c["v_cache"].transpose(1, 2)
    want = _run_attention(c)
    wide = torch.full((c["q"].shape[0], heads, 2 * D), 5.0, dtype=BF, device=device)
    c["k_cache"], c["v_cache"] = pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2)
    out = _run_attention(c, out=wide[:, :, D:])
    assert torch.equal(out, want) and bool((wide[:, :, :D] == 5.0).all())


def test_attention_with_a_bound_that_is_too_small(device):
    c, table, starts, kvs = _case(device, 16, 2, 256, 16, [(900, 300), (700, 700), (4000, 2)], BF, seed=14, gate=True)
    _check(c, table, starts, kvs, _run_attention(c, max_new=1))
    _check(c, table, starts, kvs, _run_attention(c, max_new=0))


def _one_element(c, q0, keys):
    """Queries of q0 in element 0 and 0 elsewhere; keys[p] in element 0 of
    every position p of sequence 0."""
    c["q"].zero_()
    c["q"][..., 0] = q0
    page = c["k_cache"].shape[2]
    for p, x in enumerate(keys):
        c["k_cache"][int(c["table"][0, p // page]), :, p % page, 0] = x


@pytest.mark.parametrize("layout", [(16, 2, 256), (6, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("dtype,q0,k0,scale", [(BF, 2.0 ** 64, -(2.0 ** 63), 1.0), (BF, 2.0 ** 20, 1.5 * 2.0 ** 20, 0.3),
                                               (HF, 60000.0, 60000.0, 0.7), (HF, -60000.0, 60000.0, 0.7)])
@pytest.mark.parametrize("kv,n", [(300, 1), (300, 200)])
def test_attention_scores_at_the_ends_of_the_range(device, layout, dtype, q0, k0, scale, kv, n):
    # Every third position has the row's highest score, the others one that is
    # lower by far more than a softmax tells apart: their weights are exactly
    # 1 and 0 and the result is a mean of values.  Error: fp32 sums of kv
    # terms, a division (kv + 2 roundings of 2^-24 at most), one rounding.
    c, table, starts, kvs = _case(device, *layout, 16, [(kv, n)], dtype, seed=20)
    lower = k0 * (0.5 if q0 * k0 > 0 else 1.5)
    _one_element(c, q0, [k0 if p % 3 == 1 else lower for p in range(kv)])
    got = _run_attention(c, max_new=n, scale=scale)
    v = ref.gathered(c["v_cache"], table[0][:-(-kv // 16)], kv)
    used = (torch.arange(kv, device=device) % 3 == 1).double()
    sums, sizes = (v * used[:, None]).cumsum(1), (v.abs() * used[:, None]).cumsum(1)
    at = kv - n + torch.arange(n, device=device)
    count = used.cumsum(0)[at][:, None, None]
    group = layout[0] // layout[1]

    def rows(x):
        return x[:, at].transpose(0, 1).repeat_interleave(group, dim=1) / count
    want, size = rows(sums), rows(sizes)
    bound = want.abs() * ref.half_step(dtype) + size * (kv + 2) * 2.0 ** -24 * 1.01 + torch.finfo(dtype).tiny
    live = count[:, 0, 0] > 0
    assert bool(((got.double() - want).abs() <= bound)[live].all())


@pytest.mark.parametrize("layout", [(16, 2, 256), (8, 2, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_rows_whose_scores_are_all_minus_infinity_are_nan(device, layout, dtype):
    # As the softmax of such a row is; a row that sees one finite score ignores them.
    for kv, n in ((40, 40), (9, 1), (40, 1), (300, 300)):
        c, table, starts, kvs = _case(device, *layout, 16, [(kv, n), (0, 2)], dtype, seed=21)
        c["q"][..., 0] = 1.0
        page = 16
        for p in range(min(kv, 10)):
            c["k_cache"][table[0][p // page], :, p % page, 0] = -math.inf
        got = _run_attention(c, max_new=n)
        lost = max(0, min(n, 10 - (kv - n)))   # rows that see such positions only
        assert bool(torch.isnan(got[:lost]).all()) and bool((got[n:] == 0).all())
        want, spread, score = ref.attention(c["q"], c["k_cache"], c["v_cache"], table, starts, kvs, layout[2] ** -0.5)
        top = float(c["v_cache"][torch.isfinite(c["v_cache"])].abs().max())
        bound = ref.attention_bound(want, spread, score, dtype, layout[2], kv, top)
        assert bool(((got.double() - want).abs() <= bound)[lost:n].all())


def test_attention_starts_out_of_order_are_an_empty_step(device):
    c, *_ = _case(device, 8, 2, 64, 8, [(20, 2), (24, 3)], BF, seed=15)
    out = torch.full(c["q"].shape, 3.0, dtype=BF, device=device)
    for bad in ([0, 4, 2], [-1, 2, 5], [0, 2, 6]):
        c["starts"] = _ints(bad, device)
        assert bool((_run_attention(c, out=out) == 3.0).all())


def test_calls_check_what_a_checked_form_cannot_tell(device):
    from lightreason_amd.paged import paged_append, paged_attention

    c, *_ = _case(device, 8, 2, 64, 8, [(20, 2), (24, 3)], BF, seed=16)
    q = c["q"].contiguous()
    args = (c["k_cache"], c["v_cache"], c["table"], c["starts"], c["kv_lengths"])
    paged_attention(q, *args)
    off = torch.empty(q.numel() + 4, dtype=BF, device=device)[4:].view(q.shape)   # the same form, 8 bytes off
    with pytest.raises(ValueError):
        paged_attention(off, *args)
    with pytest.raises(ValueError):
        paged_attention(q, *args, out=q)
    k = torch.zeros(5, 2, 64, dtype=BF, device=device)
    slots = torch.arange(5, device=device)
    paged_append(k, k, *args[:2], slots)
    with pytest.raises(ValueError):
        paged_append(torch.empty(k.numel() + 4, dtype=BF, device=device)[4:].view(k.shape), k, *args[:2], slots)
    with pytest.raises(ValueError):
        paged_attention(q.cpu(), *args)
    with pytest.raises(ValueError):
        paged_attention(q, args[0], args[1][:, :, :4], *args[2:])
    for kw in (dict(max_new=-1), dict(max_new=1.5), dict(gate=q[:, :4]), dict(out=q.half())):
        with pytest.raises(ValueError):
            paged_attention(q, *args, **kw)


def test_numbers_held_in_tensors_count_by_value(device):
    from lightreason_amd.paged import paged_append

    c, *rest = _case(device, 8, 2, 64, 8, [(20, 2), (24, 3)], BF, seed=17)
    scale = torch.tensor(0.25)
    for x in (0.25, 0.5):
        scale.fill_(x)
        _check(c, *rest, _run_attention(c, scale=scale), scale=x)
    k, slots, eps = torch.ones(5, 2, 64, dtype=BF, device=device), torch.arange(5, device=device), torch.tensor(0.0)
    norm = torch.zeros(64, dtype=BF, device=device)
    for x, want in ((0.0, 1.0), (3.0, 0.5)):
        eps.fill_(x)
        paged_append(k, k, c["k_cache"], c["v_cache"], slots, k_norm=norm, eps=eps)
        assert bool((c["k_cache"][0, :, :5] == want).all())


def test_threads_share_no_scratch(device):
    # Two threads' calls on one stream may have their launches mixed.
    import threading

    from lightreason_amd import _native

    mine, seen = _native.workspace(device, 1000), []
    other = threading.Thread(target=lambda: seen.append(_native.workspace(device, 1000)))
    other.start()
    other.join()
    assert _native.workspace(device, 1000).data_ptr() == mine.data_ptr() != seen[0].data_ptr()

    cases = [_case(device, 16, 2, 256, 16, [(2000, 1)] * 4, BF, seed=s)[0] for s in (1, 2)]
    want = [_run_attention(c, max_new=1) for c in cases]
    got = [[], []]

    def work(i):
        for _ in range(20):
            got[i].append(_run_attention(cases[i], max_new=1))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [len(g) for g in got] == [20, 20]
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_attention_on_two_streams_at_once(device):
    cases = [_case(device, 16, 2, 256, 16, [(3000, 1)] * 8, BF, seed=s) for s in (1, 2)]
    want = [_run_attention(c[0], max_new=1) for c in cases]
    streams = [torch.cuda.Stream(device) for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(_run_attention(c[0], max_new=1))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---- drafts -----------------------------------------------------------------------

def _blocks(device, counts, vocab, dtype, seed, noise=0.5):
    g = torch.Generator(device=device).manual_seed(seed)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    N = starts[-1]
    logits = torch.empty(N, vocab, device=device).normal_(0, 2, generator=g)
    target = torch.softmax(logits, 1).to(dtype)
    draft = torch.softmax(logits + noise * torch.empty(N, vocab, device=device).normal_(generator=g), 1)
    tokens = torch.randint(0, vocab, (N,), generator=g, device=device)
    if N > 1:
        tokens[1:] = torch.multinomial(draft, 1, generator=g)[:-1, 0]
    return dict(tokens=tokens, target=target, starts=_ints(starts, device), draft=draft.to(dtype),
                uniforms=torch.rand(N, generator=g, device=device),
                samples=torch.rand(len(counts), generator=g, device=device)), starts


def _verify(c, starts, **kw):
    from lightreason_amd.verify import verify_drafts

    draft = kw.pop("draft", c["draft"])
    got = verify_drafts(c["tokens"], c["target"], c["starts"], c["uniforms"], c["samples"], draft=draft, **kw)
    want = ref.verify(c["tokens"], c["target"], starts, c["uniforms"].tolist(), c["samples"].tolist(), draft)
    assert got[0].tolist() == want[0]
    assert got[1].tolist() == want[1]
    return want


@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8192, 8193, 50257, 151936])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify(device, dtype, vocab, with_draft):
    counts = [1, 5, 0, 2, 9, 1, 3, 17, 4]
    c, starts = _blocks(device, counts, vocab, dtype, seed=vocab)
    _verify(c, starts, draft=c["draft"] if with_draft else None)


def test_verify_long_block_and_strided_rows(device):
    c, starts = _blocks(device, [700, 1, 300], 777, torch.float32, seed=1, noise=0.01)
    c["uniforms"] *= 0.5   # long accepted runs
    wide = torch.zeros(1001, 1000, device=device)
    wide[:, 3:780] = c["target"]
    c["target"] = wide[:, 3:780]
    want = _verify(c, starts)
    assert max(want[0]) > 256


def test_verify_all_stand_and_all_fail(device):
    c, starts = _blocks(device, [4, 4], 500, torch.float32, seed=2)
    c["draft"] = c["target"].clone()
    want = _verify(c, starts)   # q = p: u q < p always
    assert want[0] == [3, 3]
    c["uniforms"].fill_(0.999)
    rows = torch.arange(7, device=device)
    c["target"][rows, c["tokens"][1:]] = 0.0
    assert _verify(c, starts)[0] == [0, 0]


def test_verify_samples_at_the_ends(device):
    c, starts = _blocks(device, [1] * 6, 4000, torch.float32, seed=3)
    c["target"][:, :100] = 0.0
    c["target"][:, 3900:] = 0.0
    c["samples"] = torch.tensor([0.0, 1.0, 0.99999994, -0.5, 2.0, math.nan], device=device)
    from lightreason_amd.verify import verify_drafts

    _, token = verify_drafts(c["tokens"], c["target"], c["starts"], c["uniforms"], c["samples"])
    assert token.tolist()[0] == token.tolist()[3] == token.tolist()[5] == 100
    assert token.tolist()[1] == token.tolist()[4] == 3899


def test_verify_rows_without_mass_and_bad_entries(device):
    c, starts = _blocks(device, [2, 2, 1, 1, 2], 300, torch.float32, seed=4)
    c["target"][0:2] = 0.0                               # no mass at all: -1
    c["draft"][2] = c["target"][2] * 2 + 1               # nothing left of p - q: drawn from p
    c["uniforms"][2] = 0.9
    c["target"][4, ::2] = math.nan                       # entries without mass
    c["target"][5, 7], c["target"][5, 9] = math.inf, -1.0
    c["tokens"][7] = 300                                 # not a token: fails
    want = _verify(c, starts)
    assert want[0][0] == 0 and want[1][0] == -1 and want[0][4] == 0


def test_verify_starts_outside_the_rows_are_idle(device):
    from lightreason_amd.verify import verify_drafts

    c, _ = _blocks(device, [3, 3], 100, torch.float32, seed=5)
    for starts in ([-1, 3, 6], [0, 3, 7], [0, 3, 2]):
        accepted, token = verify_drafts(c["tokens"], c["target"], _ints(starts, device), c["uniforms"], c["samples"])
        bad = [s < 0 or e > 6 or e <= s for s, e in zip(starts, starts[1:])]
        for b, is_bad in enumerate(bad):
            assert (token[b].item() == -1 and accepted[b].item() == 0) == is_bad


def test_verified_tokens_follow_the_target(device):
    # 40000 blocks of one draft over 5 tokens: the first output's distribution
    # is the target's, whatever the drafter's.
    from lightreason_amd.verify import verify_drafts

    B = 40000
    g = torch.Generator(device=device).manual_seed(6)
    p = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05], device=device)
    q = torch.tensor([0.1, 0.2, 0.3, 0.2, 0.2], device=device)
    tokens = torch.multinomial(q, 2 * B, replacement=True, generator=g)
    uniforms, samples = torch.rand(2 * B, generator=g, device=device), torch.rand(B, generator=g, device=device)
    accepted, token = verify_drafts(tokens, p.expand(2 * B, 5).contiguous(),
                                    _ints(list(range(0, 2 * B + 1, 2)), device), uniforms, samples,
                                    draft=q.expand(2 * B, 5).contiguous())
    first = torch.where(accepted == 1, tokens[1::2], token)
    share = torch.bincount(first, minlength=5).double() / B
    # five standard deviations of a share of 40000 draws
    assert bool(((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt()).all())


# ---- together ---------------------------------------------------------------------

class _Loop:
    """A speculative serving loop on fixed buffers: plan, append, attention,
    verify, commit over one layer; `rows` sequences of up to `room` positions."""

    def __init__(self, device, rows=5, room=8, heads=16, kv_heads=2, dim=256, page=16, vocab=2000):
        from lightreason_amd.paged import PageTable

        self.pt = PageTable(rows, 200, page, max_pages=60, device=device)
        kc, vc = self.pt.new_cache(1, kv_heads, dim)
        kc.fill_(math.nan)
        vc.fill_(math.nan)
        self.kc, self.vc = kc[0], vc[0]
        self.N = N = rows * room
        bf = dict(dtype=BF, device=device)
        self.qg, self.k, self.v = (torch.zeros(N, heads, 2 * dim, **bf), torch.zeros(N, kv_heads, dim, **bf),
                                   torch.zeros(N, kv_heads, dim, **bf))
        self.qn, self.kn = 0.1 * torch.randn(dim, **bf), 0.1 * torch.randn(dim, **bf)
        angle = torch.arange(1000, device=device)[:, None] * torch.rand(1, 32, device=device)
        angle = torch.cat([angle, angle], 1)
        self.cos, self.sin = angle.cos(), angle.sin()
        self.new = torch.zeros(rows, dtype=torch.int32, device=device)
        self.plan = self.pt.new_plan(N)
        self.q = torch.zeros(N, heads, dim, **bf)
        self.out = torch.zeros(N, heads, dim, **bf)
        self.tokens = torch.zeros(N, dtype=torch.int64, device=device)
        self.target = torch.zeros(N, vocab, device=device)
        self.draft = torch.zeros(N, vocab, device=device)
        self.uniforms, self.samples = torch.zeros(N, device=device), torch.zeros(rows, device=device)
        self.accepted = torch.zeros(rows, dtype=torch.int32, device=device)
        self.next = torch.zeros(rows, dtype=torch.int64, device=device)
        self.dim, self.page, self.room = dim, page, room

    def step(self):
        from lightreason_amd.paged import paged_append, paged_attention
        from lightreason_amd.verify import verify_drafts

        self.pt.plan(self.new, self.N, out=self.plan)
        D = self.dim
        paged_append(self.k, self.v, self.kc, self.vc, self.plan.slots, q=self.qg[:, :, :D], q_norm=self.qn,
                     k_norm=self.kn, cos=self.cos, sin=self.sin, positions=self.plan.positions, q_out=self.q)
        paged_attention(self.q, self.kc, self.vc, self.pt.table, self.plan.starts, self.plan.kv_lengths,
                        max_new=self.room, gate=self.qg[:, :, D:], out=self.out)
        verify_drafts(self.tokens, self.target, self.plan.starts, self.uniforms, self.samples, draft=self.draft,
                      accepted=self.accepted, next_tokens=self.next)
        self.pt.commit(self.plan, self.accepted)

    def fill(self, g, new):
        for t in (self.qg, self.k, self.v):
            t.normal_(generator=g)
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        logits = torch.empty_like(self.target).normal_(0, 2, generator=g)
        self.target.copy_(torch.softmax(logits, 1))
        self.draft.copy_(torch.softmax(logits + 0.4 * torch.empty_like(logits).normal_(generator=g), 1))
        self.tokens.copy_(torch.randint(0, logits.shape[1], (self.N,), generator=g, device=logits.device))
        self.tokens[1:] = torch.multinomial(self.draft, 1, generator=g)[:-1, 0]
        self.uniforms.uniform_(generator=g)
        self.samples.uniform_(generator=g)


def _loop_steps(loop, device, run, steps=6):
    """Runs the loop and checks every step against dense per-row histories."""
    g = torch.Generator(device=device).manual_seed(11)
    rng = random.Random(11)
    rows = loop.new.shape[0]
    lengths = [0] * rows
    history = [[] for _ in range(rows)]   # per row: (k row, v row) of every valid position
    results = []
    for step in range(steps):
        new = [rng.randint(1, loop.room) if step == 0 else rng.choice([0, 1, rng.randint(1, loop.room)])
               for _ in range(rows)]
        loop.fill(g, new)
        run()
        loop.pt.check()
        starts = loop.plan.starts.tolist()
        total = sum(new)
        positions = loop.plan.positions[:total].long()
        c, s = loop.cos[positions], loop.sin[positions]
        rk = ref.norm_rope(loop.k[:total], loop.kn, c, s, 1e-6).to(BF)
        rq = ref.norm_rope(loop.qg[:total, :, :loop.dim], loop.qn, c, s, 1e-6).to(BF)
        assert bool(((loop.q[:total].double() - rq.double()).abs() <= 2 * ref.half_step(BF) * rq.double().abs()
                     + 2.0 ** -16).all())
        want = ref.verify(loop.tokens, loop.target, starts, loop.uniforms.tolist(), loop.samples.tolist(), loop.draft)
        assert loop.accepted.tolist() == want[0] and loop.next.tolist() == want[1]
        for r in range(rows):
            a, n = starts[r], new[r]
            if n == 0:
                continue
            history[r] = history[r][:lengths[r]] + [(rk[a + i], loop.v[a + i].clone()) for i in range(n)]
            kv = lengths[r] + n
            blocks = loop.pt.table[r].tolist()[:-(-kv // loop.page)]
            k, v = ref.gathered(loop.kc, blocks, kv), ref.gathered(loop.vc, blocks, kv)
            assert torch.equal(v, torch.stack([x for _, x in history[r]], 1).double())
            # the 64-bit key rounded, or its neighbour where the fp32 sums fall on the other side of a border
            hk = torch.stack([x for x, _ in history[r]], 1).double()
            assert bool(((k - hk).abs() <= 2 * ref.half_step(BF) * hk.abs() + 2.0 ** -16).all())
            got = loop.out[a:a + n]
            gate = loop.qg[a:a + n, :, loop.dim:]
            o, spread, score = ref.attention(loop.q[a:a + n], loop.kc, loop.vc, [blocks], [0, n], [kv],
                                             loop.dim ** -0.5, gate)
            bound = ref.attention_bound(o, spread, score, BF, loop.dim, kv, float(v.abs().max()))
            assert bool(((got.double() - o).abs() <= bound).all())
            lengths[r] += want[0][r] + 1
        assert loop.pt.lengths.tolist() == lengths
        results.append((loop.out[:total].clone(), loop.accepted.clone(), loop.next.clone()))
    return results


def test_speculative_loop_eager_and_captured(device):
    torch.manual_seed(0)
    loop = _Loop(device)
    qn, kn, cos, sin = loop.qn, loop.kn, loop.cos, loop.sin
    eager = _loop_steps(loop, device, loop.step)
    other = _Loop(device)
    other.qn, other.kn, other.cos, other.sin = qn, kn, cos, sin
    # capture on an empty step (all counts 0), then replay with what the
    # buffers hold; the program's own eager work runs in between
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other.step()
    torch.cuda.current_stream(device).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step()
    captured = _loop_steps(other, device, graph.replay)
    for a, b in zip(eager, captured):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_two_graphs_replayed_on_two_streams(device):
    cases = [_case(device, 16, 2, 256, 16, [(2000 + s, 1)] * 6, BF, seed=s) for s in (3, 4)]
    outs = [torch.zeros(c[0]["q"].shape, dtype=BF, device=device) for c in cases]
    want = [_run_attention(c[0], max_new=1) for c in cases]
    graphs = []
    for c, out in zip(cases, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _run_attention(c[0], max_new=1, out=out)
        graphs.append(graph)
    streams = [torch.cuda.Stream(device) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)


def test_paged_layer_matches_the_contiguous_step(device):
    """paged_layer against AttentionDecode.step on the same weights: a prompt
    in a chunk of 40 and then blocks, two sequences.  Both round differently
    on the way (the step follows the Transformers forward's roundings, the
    paged operators round once), so their outputs differ by some bf16 steps of
    the values: within 2e-2 of the output's largest."""
    from lightreason_amd.attention import AttentionDecode
    from lightreason_amd.paged import PageTable, paged_layer

    g = torch.Generator(device=device).manual_seed(21)

    def normal(*shape, sigma=0.02):
        return torch.empty(shape, dtype=BF, device=device).normal_(0, sigma, generator=g)
    attn = AttentionDecode(q_proj=normal(8192, 2048), k_proj=normal(512, 2048), v_proj=normal(512, 2048),
                           o_proj=normal(2048, 4096), q_norm=normal(256, sigma=0.1), k_norm=normal(256, sigma=0.1))
    inv = 10000000.0 ** (-torch.arange(0, 64, 2, device=device).double() / 64)
    angle = torch.arange(100, device=device).double()[:, None] * inv
    angle = torch.cat([angle, angle], 1)
    cos, sin = angle.cos().to(BF), angle.sin().to(BF)
    pt = PageTable(2, 30, 16, device=device)
    kc, vc = pt.new_cache(1)
    dense = [(torch.zeros(2, 100, 256, dtype=BF, device=device), torch.zeros(2, 100, 256, dtype=BF, device=device))
             for _ in range(2)]
    lengths = [0, 0]
    for new in ([40, 9], [1, 16], [16, 1], [3, 0]):
        plan = pt.plan(_ints(new, device), sum(new) + 2)
        x = normal(plan.tokens, 2048, sigma=1.0)
        out = paged_layer(attn, x, cos, sin, kc[0], vc[0], pt, plan, max_new=max(new))
        pt.commit(plan)
        assert bool((out[sum(new):] == 0).all())
        at = 0
        for r, n in enumerate(new):
            for i in range(0, n, 16):
                m = min(16, n - i)
                p = slice(lengths[r] + i, lengths[r] + i + m)
                want = attn.step(x[at + i:at + i + m], cos[p].contiguous(), sin[p].contiguous(), *dense[r],
                                 lengths[r] + i)
                have = out[at + i:at + i + m]
                assert float((have.float() - want.float()).abs().max() / want.float().abs().max()) < 2e-2
            at += n
            lengths[r] += n
    pt.check()
