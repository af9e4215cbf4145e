"""Host-side refusals of the paged-cache operators and of the draft
verification (no GPU needed): the Python checks, and the C ABI's."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from lightreason_amd import _native, paged, verify

BF = torch.bfloat16


def test_structures_match_the_header():
    """Field order and sizes of the argument structures (natural alignment, no
    hidden padding: every 8-byte field follows an even number of 4-byte ones)."""
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "lrmoe.h").read_text()
    for name, struct in (("lrmoe_paged_append_args", _native.PagedAppendArgs),
                         ("lrmoe_paged_attention_args", _native.PagedAttentionArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for line in body.split(";"):
            words = re.findall(r"\w+", line)
            fields += [w for w in words if w not in ("const", "void", "int32_t", "int64_t", "float")]
        assert fields == [f for f, _ in struct._fields_]
        size = sum(C.sizeof(t) for _, t in struct._fields_)
        assert C.sizeof(struct) == size


def test_page_table_refuses_bad_sizes():
    for kw in (dict(rows=0), dict(rows=4097), dict(pages=0), dict(page=4), dict(page=24), dict(page=2048),
               dict(max_pages=0), dict(rows=2.0), dict(pages=True), dict(page=1024, max_pages=1 << 22),
               dict(page=1024, max_pages=(1 << 20) + 1)):
        args = dict(rows=2, pages=10, page=16, max_pages=None, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            paged.PageTable(args.pop("rows"), args.pop("pages"), args.pop("page"), **args)


def test_page_table_calls_refuse_host_tensors_and_other_pools():
    pt = paged.PageTable(2, 10, 16, device="cpu")
    new = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU|cpu"):
        pt.plan(new, 4)
    with pytest.raises(ValueError):
        pt.plan(new.long(), 4)
    with pytest.raises(ValueError):
        pt.plan(new[:1], 4)
    with pytest.raises(TypeError):
        pt.plan([1, 1], 4)
    with pytest.raises(ValueError):
        pt.release(torch.ones(2))
    other = paged.PageTable(3, 10, 16, device="cpu").new_plan(4)
    with pytest.raises(ValueError, match="pool"):
        pt.commit(other)


def _cache(pages=4, kv_heads=2, page=16, dim=64, dtype=BF):
    return torch.zeros(pages, kv_heads, page, dim, dtype=dtype)


def test_append_and_attention_refuse_host_tensors_and_shapes():
    k = torch.zeros(3, 2, 64, dtype=BF)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        paged.paged_append(k, k, _cache(), _cache(), slots)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        paged.paged_append(k.float(), k.float(), _cache(), _cache(), slots)
    with pytest.raises(ValueError, match="width"):
        paged.paged_append(k[:, :, :32], k[:, :, :32], _cache(), _cache(), slots)
    with pytest.raises(ValueError, match="heads, dim"):
        paged.paged_append(k[0], k, _cache(), _cache(), slots)
    table = torch.zeros(1, 4, dtype=torch.int32)
    starts = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        paged.paged_attention(k, _cache(), _cache(), table, starts, starts[1:])
    with pytest.raises(ValueError, match="width"):
        paged.paged_attention(k[:, :, :48], _cache(), _cache(), table, starts, starts[1:])



def test_strides_are_checked():
    good = torch.zeros(4, 3, 64, dtype=BF)
    paged._strided(good, "x", 8)
    paged._strided(torch.zeros(4, 3, 128, dtype=BF)[:, :, 64:], "x", 8)
    for bad in (torch.zeros(4, 3, 65, dtype=BF)[:, :, :64], torch.zeros(4, 64, 3, dtype=BF).transpose(1, 2),
                torch.zeros(4, 3, 128, dtype=BF)[:, :, 4:68]):
        with pytest.raises(ValueError, match="contiguous last dimension"):
            paged._strided(bad, "x", 8)
    # a dimension of one entry has no stride to speak of
    paged._strided(torch.zeros(1, 3, 65, dtype=BF)[:, :1, :64], "x", 8)


def test_layer_refuses_caches_of_another_pool():
    pt = paged.PageTable(2, 4, 16, device="cpu")
    plan, hidden = pt.new_plan(3), torch.zeros(3, 2048, dtype=BF)
    for pages, page in ((5, 16), (4, 32)):
        other = _cache(pages=pages, page=page, dim=256)
        with pytest.raises(ValueError, match="pool"):
            paged.paged_layer(None, hidden, None, None, other, _cache(dim=256), pt, plan)
        with pytest.raises(ValueError, match="pool"):
            paged.paged_layer(None, hidden, None, None, _cache(dim=256), other, pt, plan)


def test_verify_refuses():
    tokens = torch.zeros(4, dtype=torch.int64)
    p = torch.zeros(4, 10)
    starts = torch.tensor([0, 4], dtype=torch.int32)
    u, s = torch.zeros(4), torch.zeros(1)
    with pytest.raises(ValueError, match="GPU"):
        verify.verify_drafts(tokens, p, starts, u, s)
    with pytest.raises(ValueError):
        verify.verify_drafts(tokens, p.double(), starts, u, s)
    with pytest.raises(ValueError):
        verify.verify_drafts(tokens, p[0], starts, u, s)


def _attention_args(**kw):
    base = dict(seqs=1, tokens=1, max_new=1, heads=16, kv_heads=2, dim=256, pages=4, page=16, max_pages=4, scale=1.0,
                q=256, q_token_stride=4096, q_head_stride=256, k_cache=256, v_cache=256, k_page_stride=8192,
                k_head_stride=4096, k_row_stride=256, v_page_stride=8192, v_head_stride=4096, v_row_stride=256,
                table=256, starts=256, kv_lengths=256, out=512, out_token_stride=4096, out_head_stride=256)
    base.update(kw)
    return _native.PagedAttentionArgs(**base)


def test_abi_attention_refuses_before_any_launch():
    lib = _native.library()
    big = 1 << 40

    def call(a, ws=256, nbytes=big):
        return lib.lrmoe_paged_attention(C.addressof(a), ws, nbytes, None)
    assert lib.lrmoe_paged_attention(None, 256, big, None) == -1
    for kw in (dict(seqs=-1), dict(seqs=4097), dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(max_new=-1),
               dict(heads=0), dict(kv_heads=0), dict(heads=15), dict(heads=2048), dict(dim=96), dict(pages=0),
               dict(page=4), dict(page=48), dict(page=2048), dict(max_pages=0), dict(max_pages=1 << 28), dict(max_pages=(1 << 26) + 1),
               dict(q=0),
               dict(k_cache=0), dict(v_cache=0), dict(table=0), dict(starts=0), dict(kv_lengths=0), dict(out=0),
               dict(q=264), dict(k_cache=8), dict(v_cache=24), dict(out=8), dict(gate=8), dict(q_token_stride=4),
               dict(k_row_stride=260), dict(v_page_stride=4), dict(out_token_stride=4),
               dict(gate=256, gate_head_stride=4), dict(out=256), dict(gate=512), dict(k_row_stride=1 << 20),
               dict(v_row_stride=-8), dict(pages=1 << 30, k_page_stride=1 << 20), dict(v_page_stride=-8),
               dict(tokens=1 << 19, heads=1024, kv_heads=1)):
        assert call(_attention_args(**kw)) == -1, kw
    assert call(_attention_args(), ws=8) == -1
    need = lib.lrmoe_paged_attention_workspace_bytes(C.addressof(_attention_args()))
    if need:
        assert call(_attention_args(), nbytes=need - 1) == -2
        assert call(_attention_args(), ws=None) == -1
    assert lib.lrmoe_paged_attention_workspace_bytes(C.addressof(_attention_args(dim=3))) == 0
    assert call(_attention_args(tokens=0)) == 0 and call(_attention_args(seqs=0)) == 0


def _append_args(**kw):
    base = dict(tokens=1, heads=2, kv_heads=1, dim=64, rotary=32, pages=4, page=16, q=256, k=256, v=256,
                q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64, v_token_stride=64,
                v_head_stride=64, eps=1e-6, rope_fp32=1, cos=256, sin=256, rope_rows=4, slots=256, q_out=256,
                k_cache=256, v_cache=256, k_page_stride=1024, k_cache_head_stride=1024, k_row_stride=64,
                v_page_stride=1024, v_cache_head_stride=1024, v_row_stride=64)
    base.update(kw)
    return _native.PagedAppendArgs(**base)


def test_abi_append_refuses_before_any_launch():
    lib = _native.library()
    assert lib.lrmoe_paged_append(None, None) == -1
    for kw in (dict(tokens=-1), dict(heads=-1), dict(kv_heads=0), dict(dim=32), dict(rotary=24), dict(rotary=80),
               dict(pages=0), dict(page=12), dict(rope_rows=0), dict(k=0), dict(v=0), dict(slots=0), dict(k_cache=0),
               dict(v_cache=0), dict(q=0), dict(q_out=0), dict(cos=0), dict(sin=0), dict(k=264), dict(q_norm=8),
               dict(cos=4), dict(k_row_stride=4), dict(q_head_stride=12), dict(v_page_stride=3)):
        assert lib.lrmoe_paged_append(C.addressof(_append_args(**kw)), None) == -1, kw
    assert lib.lrmoe_paged_append(C.addressof(_append_args(tokens=0)), None) == 0


def test_abi_pool_and_verify_refuse_before_any_launch():
    lib = _native.library()
    p = 256

    def plan(rows=1, pages=4, page=16, max_pages=4, tokens=1, ptrs=(p,) * 12):
        return lib.lrmoe_page_plan(rows, pages, page, max_pages, tokens, *ptrs, None)
    for kw in (dict(rows=-1), dict(rows=4097), dict(pages=0), dict(page=4), dict(page=24), dict(max_pages=0),
               dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(max_pages=1 << 28)):
        assert plan(**kw) == -1, kw
    for i in range(12):
        assert plan(ptrs=(p,) * i + (None,) + (p,) * (11 - i)) == -1
    assert plan(rows=0) == 0
    assert lib.lrmoe_page_commit(-1, *([p] * 8), None) == -1
    for i in (0, 1, 2, 3, 5, 6, 7):
        assert lib.lrmoe_page_commit(1, *([p] * i + [None] + [p] * (7 - i)), None) == -1
    assert lib.lrmoe_page_release(1, 0, 4, *([p] * 6), None) == -1
    for i in range(6):
        assert lib.lrmoe_page_release(1, 4, 4, *([p] * i + [None] + [p] * (5 - i)), None) == -1

    def check(blocks=1, rows=2, vocab=10, type=0, tokens=p, target=p, ts=10, draft=p, ds=10, starts=p, u=p, s=p,
              acc=p, nxt=p, ws=p, nbytes=1 << 30):
        return lib.lrmoe_verify_drafts(blocks, rows, vocab, type, tokens, target, ts, draft, ds, starts, u, s, acc,
                                       nxt, ws, nbytes, None)
    for kw in (dict(blocks=-1), dict(blocks=65536), dict(rows=-1), dict(vocab=0), dict(type=3), dict(type=-1),
               dict(tokens=None), dict(target=None), dict(ts=9), dict(ds=9), dict(starts=None), dict(u=None),
               dict(s=None), dict(acc=None), dict(nxt=None), dict(ws=None), dict(ws=8), dict(target=258),
               dict(draft=257, type=1)):
        assert check(**kw) == -1, kw
    assert check(nbytes=lib.lrmoe_verify_workspace_bytes(1, 10) - 1) == -2
    assert check(blocks=0) == 0
