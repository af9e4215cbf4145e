"""Refusals of the scan's, beam search's and forks' calls on the host (no GPU)."""

from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from lightreason_amd import _native, beam, paged, scan

BF = torch.bfloat16


def test_structures_match_the_header():
    text = (Path(__file__).resolve().parents[1] / "include" / "lrmoe.h").read_text()
    for name, struct in (("lrmoe_delta_scan_args", _native.DeltaScanArgs),
                         ("lrmoe_delta_grad_args", _native.DeltaGradArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for line in body.split(";"):
            words = re.findall(r"\w+", line)
            fields += [w for w in words if w not in ("const", "void", "int32_t", "int64_t", "float")]
        assert fields == [f for f, _ in struct._fields_]
        assert C.sizeof(struct) == sum(C.sizeof(t) for _, t in struct._fields_)
    for name, value in (("LRMOE_BEAM_MAX", _native.BEAM_MAX), ("LRMOE_FORK_TENSORS", _native.FORK_TENSORS),
                        ("LRMOE_FORK_CACHES", _native.FORK_CACHES)):
        assert int(re.search(r"#define %s (\d+)" % name, text).group(1)) == value


def _scan_args(N=4, K=2, H=4, D=64, E=64, dtype=BF):
    return dict(query=torch.zeros(N, K, D, dtype=dtype), key=torch.zeros(N, K, D, dtype=dtype),
                value=torch.zeros(N, H, E, dtype=dtype), g=torch.zeros(N, H), beta=torch.zeros(N, H, dtype=dtype),
                starts=torch.tensor([0, N], dtype=torch.int32))


def test_scan_refuses_host_tensors_and_shapes():
    for call in (scan.delta_scan, lambda **x: scan.delta_step(**x, states=torch.zeros(1, 4, 64, 64))):
        with pytest.raises(ValueError, match="GPU"):
            call(**_scan_args())
        with pytest.raises(ValueError, match="bfloat16"):
            call(**_scan_args(dtype=torch.float32))
        with pytest.raises(ValueError, match="width"):
            call(**_scan_args(D=96))
        with pytest.raises(ValueError, match="key_heads"):
            call(**{**_scan_args(), "query": torch.zeros(4, 64, dtype=BF)})
        with pytest.raises(ValueError):
            call(**{**_scan_args(), "query": [1]})


def test_c_entry_points_refuse_misuse():
    lib = _native.library()
    good = dict(seqs=1, tokens=4, max_new=100, heads=4, key_heads=2, dim=64, value_dim=64, pool=1, scale=1.0,
                q=256, k=256, v=1 << 20, g=256, beta=256, starts=256, initial=256, final=256, out=1 << 24,
                q_token_stride=128, q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=256,
                v_head_stride=64, g_token_stride=4, beta_token_stride=4, out_token_stride=256, out_head_stride=64)
    ws = C.c_void_p(256)

    def call(nbytes=1 << 40, workspace=ws, **kw):
        a = _native.DeltaScanArgs(**{**good, **kw})
        return lib.lrmoe_delta_scan(C.addressof(a), workspace, nbytes, None)
    for kw in (dict(seqs=-1), dict(seqs=65537), dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(heads=0),
               dict(heads=3), dict(heads=1026), dict(key_heads=0), dict(dim=96), dict(dim=256), dict(value_dim=16),
               dict(value_dim=288), dict(value_dim=72), dict(pool=-1), dict(max_new=-1), dict(q=None), dict(k=None),
               dict(v=None), dict(g=None), dict(beta=None), dict(starts=None), dict(final=None), dict(out=None),
               dict(q=264), dict(out=(1 << 24) + 4), dict(q_token_stride=129), dict(v_head_stride=4),
               dict(k_token_stride=-8), dict(v_token_stride=1 << 23), dict(out_token_stride=2), dict(g=258),
               dict(beta=257), dict(final=264), dict(workspace=None), dict(workspace=C.c_void_p(128)),
               dict(tokens=1 << 20, heads=128, key_heads=1), dict(seqs=65536, heads=64, key_heads=2)):
        assert call(**kw) == _native.LRMOE_E_ARG, kw
    assert call(nbytes=0) == _native.LRMOE_E_WORKSPACE
    assert call(seqs=0) == 0
    # max_new is a hint: a tape is the chunked form's, which has its workspace.
    nbytes = lambda **kw: lib.lrmoe_delta_scan_workspace_bytes(C.byref(_native.DeltaScanArgs(**{**good, **kw})))
    assert nbytes(max_new=1) == 0 and nbytes(max_new=1, tape=256) == nbytes(max_new=4, tape=256) > 0
    assert call(max_new=1, tape=256, nbytes=0) == _native.LRMOE_E_WORKSPACE
    assert lib.lrmoe_delta_scan(None, ws, 1 << 40, None) == _native.LRMOE_E_ARG
    # out over what is read, and over itself
    assert call(out=1 << 20) == _native.LRMOE_E_ARG
    assert call(out=256 + 64) == _native.LRMOE_E_ARG
    assert call(out_head_stride=32) == _native.LRMOE_E_ARG
    assert call(q=1 << 26, k=1 << 27, out=(1 << 26) + 8, value_dim=128, v_token_stride=512, v_head_stride=128,
                out_token_stride=512, out_head_stride=128) == _native.LRMOE_E_ARG

    back = dict(d_out=256, tape=256, dq=256, dk=256, dv=256, dg=256, dbeta=256, d_out_token_stride=256,
                d_out_head_stride=64)

    def gradient(nbytes=1 << 40, workspace=ws, args=(), **kw):
        a = _native.DeltaScanArgs(**{**good, **dict(args)})
        d = _native.DeltaGradArgs(**{**back, **kw})
        return lib.lrmoe_delta_scan_grad(C.addressof(a), C.addressof(d), workspace, nbytes, None)
    for kw in (dict(d_out=None), dict(tape=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dg=None),
               dict(dbeta=None), dict(dq=264), dict(d_final=264), dict(d_initial=264), dict(tape=320),
               dict(d_out_token_stride=4), dict(args=dict(slots=256)), dict(args=dict(into=256)),
               dict(args=dict(fresh=256)), dict(args=dict(pool=2)), dict(args=dict(dim=32)), dict(args=dict(q=None)),
               dict(workspace=None)):
        assert gradient(**kw) == _native.LRMOE_E_ARG, kw
    assert gradient(nbytes=0) == _native.LRMOE_E_WORKSPACE
    assert gradient(args=dict(seqs=0, pool=0)) == 0

    p = C.c_void_p(256)
    assert lib.lrmoe_beam_workspace_bytes(1, 33, 10) == 0 and lib.lrmoe_beam_workspace_bytes(1, 4, 10) > 0
    for args in ((1, 0, 10, 0), (1, 33, 10, 0), (-1, 4, 10, 0), (20000, 4, 10, 0), (1, 4, 0, 0), (1, 4, 10, 3)):
        assert lib.lrmoe_beam_select(*args, p, 10, p, None, p, p, p, p, 1 << 30, None) == _native.LRMOE_E_ARG, args
    assert lib.lrmoe_beam_select(1, 4, 10, 0, p, 9, p, None, p, p, p, p, 1 << 30, None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_beam_select(1, 4, 10, 0, None, 10, p, None, p, p, p, p, 1 << 30, None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_beam_select(1, 4, 10, 0, p, 10, p, None, p, p, p, p, 8, None) == _native.LRMOE_E_WORKSPACE
    assert lib.lrmoe_beam_select(0, 4, 10, 0, None, 10, None, None, None, None, None, None, 0, None) == 0

    table = (C.c_int64 * 3)(256, 64, 64)
    assert lib.lrmoe_fork_rows(-1, p, 1, table, None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(4, None, 1, table, None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(4, p, 65, table, None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(4, p, 1, (C.c_int64 * 3)(256, 63, 64), None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(4, p, 1, (C.c_int64 * 3)(0, 64, 64), None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(1 << 20, p, 1, (C.c_int64 * 3)(256, 1 << 30, 1 << 30), None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(1 << 24, p, 1, (C.c_int64 * 3)(256, 4, 4), None) == _native.LRMOE_E_ARG
    assert lib.lrmoe_fork_rows(0, None, 1, table, None) == 0

    row = (256, 2, 2, 128, 1 << 20, 1 << 12, 1 << 11, 128)
    fork = lambda n=4, page=16, caches=1, row=row: lib.lrmoe_page_fork(n, 8, page, 4, p, p, p, p, p, p, caches,
                                                                      (C.c_int64 * 8)(*row), p, None)
    for kw in (dict(n=-1), dict(n=4097), dict(page=24), dict(caches=33), dict(caches=-1), dict(row=(0,) + row[1:]),
               dict(row=(256, 0) + row[2:]), dict(row=(256, 2, 2, 8) + row[4:]), dict(row=row[:7] + (120,)),
               dict(row=row[:4] + (-16,) + row[5:])):
        assert fork(**kw) == _native.LRMOE_E_ARG, kw
    assert fork(n=0) == 0


def test_beam_refuses_host_tensors_and_shapes():
    logits, scores = torch.zeros(8, 100), torch.zeros(2, 4)
    with pytest.raises(ValueError, match="GPU"):
        beam.beam_select(logits, scores)
    for l, s in ((logits[:7], scores), (logits.double(), scores), (logits, scores.double()), (logits[0], scores),
                 (logits, scores[0]), (torch.zeros(66, 10), torch.zeros(2, 33)), (torch.zeros(8, 0), scores),
                 (torch.zeros(65536, 1), torch.zeros(65536, 1)), ([1], scores), (logits, None)):
        with pytest.raises(ValueError):
            beam.beam_select(l, s)
    with pytest.raises(ValueError):
        beam.fork_rows(torch.zeros(3, dtype=torch.int64), [])
    with pytest.raises(ValueError, match="GPU"):
        beam.fork_rows(torch.zeros(3, dtype=torch.int32), [])
    with pytest.raises(ValueError):
        beam.fork_rows([0], [])


def test_page_fork_refuses_host_tensors_and_shapes():
    pool = paged.PageTable(2, 10, 16, device="cpu")
    with pytest.raises(ValueError):
        pool.fork(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU|cpu"):
        pool.fork(torch.zeros(2, dtype=torch.int32))


def test_gradients_off_the_alignment_are_copied():
    whole = torch.arange(64, dtype=BF)
    assert whole.data_ptr() % 16 == 0 and scan._aligned(whole) is whole
    piece = whole[3:51].view(2, 3, 8)
    assert piece.is_contiguous() and piece.contiguous().data_ptr() % 16
    for t in (piece, piece.transpose(0, 1), piece[:1, :1].expand(4, 2, 8)):
        copy = scan._aligned(t)
        assert copy.data_ptr() % 16 == 0 and copy.is_contiguous() and torch.equal(copy, t)


def test_dual_tensors_are_told_apart():
    x = [torch.zeros(2, 3), None, torch.zeros(3, dtype=torch.int32)]
    assert not scan._has_tangents(x)
    with torch.autograd.forward_ad.dual_level():
        assert not scan._has_tangents(x)
        dual = torch.autograd.forward_ad.make_dual(x[0], torch.ones(2, 3))
        assert scan._has_tangents([*x, dual]) and not dual.requires_grad
    assert not scan._has_tangents([*x, dual])


def test_scratch_and_tape_hold_a_slot_per_chunk_or_token():
    """A slot per 64 tokens and per sequence, but no more than there are tokens (of
    sequences that go in chunks: 25 each)."""
    lib = _native.library()

    def sizes(tokens, seqs, **kw):
        a = _native.DeltaScanArgs(**{**dict(seqs=seqs, tokens=tokens, max_new=tokens, heads=2, key_heads=1, dim=64,
                                            value_dim=32, pool=seqs), **kw})
        return [getattr(lib, f"lrmoe_delta_scan_{n}_bytes")(C.byref(a)) for n in ("tape", "grad_workspace", "workspace")]
    tape, grad, _ = sizes(1, 1)
    assert tape == 2 * (64 + 64) * 32 * 4
    for tokens, seqs in ((6400, 3), (8, 1000), (64, 1), (63, 1), (1000, 1000), (0, 5)):
        slots = max(1, min(tokens, tokens // 64 + seqs))
        assert sizes(tokens, seqs)[0] == tape * slots
        assert sizes(tokens, seqs)[1] <= grad * slots
    # Without a tape: 256 single tokens have no chunk, padding takes none.
    one = sizes(100, 1)[2]
    assert sizes(256, 256)[2] < 8 * one and sizes(100, 60000)[2] < 4 * one + 4 * 60000 * 2 * 2 + 256


def test_chunk_slots_never_meet():
    """The kernels' rule for a sequence's first slot, over counts around its edges."""
    import random
    rng = random.Random(3)
    first = lambda start, s, c: min(start // c, start // 64 + s)
    for token_wise in (0, 24, 40):   # (sequences of up to so many tokens have none)
        c = min(token_wise + 1, 32)
        edges = [0, 0, 1, 2, token_wise, token_wise + 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]
        for _ in range(2000):
            counts = [rng.choice(edges) for _ in range(rng.choice([1, 3, 10, 80]))]
            at, used = rng.choice([0, 1, 63, 64, 500]), 0
            tokens = at + sum(counts) + rng.choice([0, 7])
            for s, n in enumerate(counts):
                if n > token_wise:
                    assert first(at, s, c) >= used
                    used = first(at, s, c) + (n + 63) // 64
                    assert used <= first(at + n, s + 1, c)
                at += n
            assert used <= min(tokens // c, tokens // 64 + len(counts))


def test_fused_scan_tells_what_it_takes():
    class Shape:   # what is looked at of a tensor
        def __init__(self, *shape, dtype=BF, device="cuda"):
            self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)

        def dim(self):
            return len(self.shape)

    def call(B=2, T=10, K=4, H=4, D=64, E=64, **kw):
        q, k, v, g, beta = (Shape(B, T, K, D), Shape(B, T, K, D), Shape(B, T, H, E), Shape(B, T, H, dtype=torch.float32),
                            Shape(B, T, H))
        args = dict(query=q, key=k, value=v, g=g, beta=beta, initial=None)
        return scan._takes(**{**args, **kw})
    assert call() and call(E=256, H=8) and call(D=128, initial=Shape(2, 4, 128, 64, dtype=torch.float32))
    for kw in (dict(D=96), dict(D=256), dict(E=48), dict(E=288), dict(K=3), dict(T=1 << 20), dict(K=1026, H=1026),
               dict(B=65537, T=1), dict(query=Shape(2, 10, 4, 64, device="cpu")), dict(key=Shape(2, 10, 4, 64, dtype=torch.half)),
               dict(value=Shape(2, 10, 4, 64, dtype=torch.float32)), dict(query=Shape(2, 10, 4, 64, dtype=torch.float32)),
               dict(key=Shape(2, 9, 4, 64)), dict(g=Shape(2, 10, 4, dtype=torch.float32, device="cpu")),
               dict(initial=Shape(2, 4, 64, 128, dtype=torch.float32)), dict(query=Shape(10, 4, 64))):
        assert not call(**kw), kw


def test_rows_that_cannot_be_read_in_place_are_copied():
    whole = torch.randn(5 * 3 * 80 + 8).to(BF)
    good = whole[8:8 + 5 * 3 * 80].view(5, 3, 80)[:, :, :64]
    assert scan._laid_out(good) is good
    off = whole[3:3 + 5 * 3 * 64].view(5, 3, 64)
    narrow = whole[:5 * 3 * 68].view(5, 3, 68)[:, :, :64]
    turned = whole[:5 * 3 * 64].view(5, 64, 3).transpose(1, 2)
    for t in (off, narrow, turned):
        copy = scan._laid_out(t)
        assert copy is not t and copy.is_contiguous() and copy.data_ptr() % 16 == 0 and torch.equal(copy, t)
    g = torch.randn(5, 9)[:, 1:4]
    assert scan._laid_out(g) is g


def test_forks_are_cut_to_what_a_call_holds():
    text = (Path(__file__).resolve().parents[1] / "include" / "lrmoe.h").read_text()
    assert f"#define LRMOE_FORK_BYTES {_native.FORK_BYTES}\n" in text and "#define LRMOE_FORK_PIECES (1 << 24)\n" in text
    assert _native.FORK_PIECES == 1 << 24
    counts = lambda rows, layout: [(i, len(part)) for i, part in beam._fork_parts(rows, layout)]
    assert counts(4, []) == [] and counts(0, [(8, 8)] * 3) == [(0, 3)] and counts(4, [(0, 0)] * 65) == [(0, 64), (64, 1)]
    assert counts(4, [(64, 64)] * 130) == [(0, 64), (64, 64), (128, 2)]
    # 2^18 - 1 rows: 64 pieces of a row fit a call, 65 do not.
    rows, small, two = (1 << 18) - 1, (4, 4), (40000, 40000)
    assert counts(rows, [small] * 64 + [small] * 62 + [two] + [small]) == [(0, 64), (64, 63), (127, 1)]
    for rows, layout in ((rows, [two] * 70), (1 << 22, [small] * 9), (1, [(1 << 38, 1 << 38)] * 3)):
        parts = beam._fork_parts(rows, layout)
        assert [x for _, part in parts for x in part] == layout
        assert [i for i, _ in parts] == [sum(len(part) for _, part in parts[:n]) for n in range(len(parts))]
        for _, part in parts:
            assert sum(-(-b // 32768) * rows for _, b in part) < 1 << 24
    # One that fits no call, behind others, is refused before any of them.
    with pytest.raises(ValueError, match="tensor 70 has"):
        beam._fork_parts(1 << 18, [small] * 70 + [(1 << 21, 1 << 21)])
    with pytest.raises(ValueError, match="tensor 0 has"):
        beam._fork_parts(1 << 24, [(4, 4)])
