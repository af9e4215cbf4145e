"""Calls of the paged-cache operators that are settled on the host (no GPU)."""

from __future__ import annotations

import ctypes as C

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


def _rows(base, shape, strides, dim):
    return {base + t * strides[0] + h * strides[1] + d
            for t in range(shape[0]) for h in range(shape[1]) for d in range(dim)}


@pytest.mark.parametrize("which", ["q", "gate", "out"])
def test_overlapping_outputs_of_the_attention_are_refused(which):
    """Layouts in which out shares elements with q, with gate or with itself,
    told by sets of addresses, are refused before any launch (addresses in
    elements of 2 bytes; the calls that would pass are made on the GPU)."""
    import random

    from lightreason_amd import _native

    lib, rng, D, refused = _native.library(), random.Random(which), 64, 0
    for _ in range(400):
        N, H = rng.choice([1, 2, 5]), rng.choice([1, 2, 4])
        base = 1 << 20
        out_at = base + 8 * rng.randint(-60, 60)

        def strides():
            pitch = rng.choice([D, D + 8, 2 * D, 0])
            return rng.choice([(H * pitch, pitch), (H * pitch + 2 * D, pitch), (pitch, N * pitch), (2 * D, 4 * D)])
        s, o = strides(), strides()
        out = _rows(out_at, (N, H), o, D)
        if which == "out":
            shared = len(out) < N * H * D
            other = dict(q=256, q_token_stride=H * D, q_head_stride=D)
        else:
            shared = bool(out & _rows(base, (N, H), s, D))
            other = {which: 2 * base, f"{which}_token_stride": s[0], f"{which}_head_stride": s[1]}
            if which == "gate":
                other.update(q=256, q_token_stride=H * D, q_head_stride=D)
        if not shared:
            continue
        refused += 1
        a = _native.PagedAttentionArgs(
            seqs=1, tokens=N, max_new=1, heads=H, kv_heads=1, dim=D, pages=4, page=16, max_pages=4, scale=1.0,
            k_cache=256, v_cache=256, k_page_stride=1024, k_head_stride=1024, k_row_stride=64, v_page_stride=1024,
            v_head_stride=1024, v_row_stride=64, table=256, starts=256, kv_lengths=256, out=2 * out_at,
            out_token_stride=o[0], out_head_stride=o[1], **other)
        assert lib.lrmoe_paged_attention(C.addressof(a), 256, 1 << 40, None) == -1, (N, H, s, o, out_at - base)
    assert refused > 50


def test_queries_written_over_other_inputs_are_refused():
    from lightreason_amd import _native

    lib, D, N, H = _native.library(), 64, 3, 2
    far = {"q": 1 << 20, "k": 1 << 21, "v": 1 << 22, "q_out": 1 << 23}
    for kw in (dict(q_out=far["q"] + 2 * 64), dict(q_out=far["q"] - 2 * 64), dict(q_out=far["k"] + 2 * 64),
               dict(q_out=far["v"]), dict(q_out=far["q"], q_token_stride=256), dict(q_out=far["q"], q_head_stride=0)):
        args = dict(tokens=N, heads=H, kv_heads=1, dim=D, pages=4, page=16, q_token_stride=H * D, q_head_stride=D,
                    k_token_stride=D, k_head_stride=D, v_token_stride=D, v_head_stride=D, eps=1e-6, slots=256,
                    k_cache=256, v_cache=512, k_page_stride=1024, k_cache_head_stride=1024, k_row_stride=64,
                    v_page_stride=1024, v_cache_head_stride=1024, v_row_stride=64, **far)
        args.update(kw)
        a = _native.PagedAppendArgs(**args)
        assert lib.lrmoe_paged_append(C.addressof(a), None) == -1, kw


def test_appends_of_more_threads_than_a_launch_holds_are_refused():
    from lightreason_amd import _native

    lib = _native.library()
    for tokens, kv_heads, dim in ((1 << 24, 1024, 256), (1 << 24, 16, 256), (1 << 20, 256, 256), (1 << 24, 64, 64)):
        a = _native.PagedAppendArgs(
            tokens=tokens, heads=0, kv_heads=kv_heads, dim=dim, pages=4, page=16, k=256, v=256, slots=256, k_cache=256,
            v_cache=512, k_page_stride=1 << 20, k_cache_head_stride=1 << 14, k_row_stride=dim, v_page_stride=1 << 20,
            v_cache_head_stride=1 << 14, v_row_stride=dim)
        assert lib.lrmoe_paged_append(C.addressof(a), None) == -1, (tokens, kv_heads, dim)


def test_workspaces_stay_within_the_bound_of_the_header():
    import random

    from lightreason_amd import _native

    lib, rng, closest = _native.library(), random.Random(5), 0.0
    for _ in range(3000):
        kv_heads, group = rng.choice([1, 2, 4, 8, 16, 64, 1024]), rng.choice([1, 2, 3, 8, 16, 64])
        dim = rng.choice([64, 128, 256])
        heads = kv_heads * group
        if heads > 1024:
            continue
        tokens = min(int(2 ** rng.uniform(0, 20)), (1 << 28) // heads)
        seqs, max_new = int(2 ** rng.uniform(0, 12)), rng.choice([1, 2, 4, 9, 40, tokens])
        page = 1 << rng.randint(3, 10)
        a = _native.PagedAttentionArgs(seqs=seqs, tokens=tokens, max_new=max_new, heads=heads, kv_heads=kv_heads,
                                       dim=dim, pages=1, page=page, max_pages=int(2 ** rng.uniform(0, 30)) // page or 1)
        got = lib.lrmoe_paged_attention_workspace_bytes(C.addressof(a))
        rows = 32 if max_new * group <= 32 else 128
        partial = 2 * (1024 + kv_heads) + 16 if rows == 32 else 4 * (256 + kv_heads) + 16
        tiles = kv_heads * (tokens * group // rows + min(seqs, tokens))
        bound = partial * rows * (4 * dim + 8) + 36 * tiles + 16384
        assert 0 < got <= bound, (heads, kv_heads, dim, tokens, seqs, max_new, page)
        closest = max(closest, got / bound)
    assert closest > 0.95
