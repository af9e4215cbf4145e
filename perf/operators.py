"""Serving operators over a paged key/value cache, as cases that can be timed
and compared with plain forms: the page plan of a step (which pages and slots
its new positions take), the append of normed and rotated keys and values into
those slots, the attention of the new positions over the cache, and the
verification of drafted tokens from given random numbers.

With ``own`` false ``run`` computes each operator in elementary torch
operations; with ``own`` true it calls ``lightreason_amd.paged`` and
``lightreason_amd.verify``.  Head layouts are the 35B model's (16 query heads
over 2 key/value heads of width 256, rotary width 64) and generic ones; a
step's sequences are ragged, from one cached position to tens of thousands.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # Four chat sequences of which each adds one position: the plan before
        # every decode step of a small server.
        {"name": "plan_4", "kind": "plan", "rows": 4, "page": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 100,
         "ctx_hi": 4000, "lens": 1},
        # A full server: 1000 rows on small pages, prompts and decode steps
        # mixed, half of the positions of the widest step.
        {"name": "plan_1000", "kind": "plan", "rows": 1000, "page": 16, "new_lo": 0, "new_hi": 65, "ctx_lo": 0,
         "ctx_hi": 9000, "lens": 2},
        # Decode of eight sequences: the append of one layer.
        {"name": "append_8", "kind": "append", "seqs": 8, "heads": 16, "kv_heads": 2, "dim": 256, "rotary": 64,
         "page": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 100, "ctx_hi": 3000, "dtype": "bf16", "lens": 3},
        # Prompts of a whole prefill step, ragged.
        {"name": "append_8k", "kind": "append", "seqs": 5, "heads": 16, "kv_heads": 2, "dim": 256, "rotary": 64,
         "page": 64, "new_lo": 1200, "new_hi": 2100, "ctx_lo": 0, "ctx_hi": 2000, "dtype": "bf16", "lens": 4},
        # One chat sequence decoding: the latency of one layer's attention.
        {"name": "attn_decode_1", "kind": "attn", "seqs": 1, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "new_lo": 1, "new_hi": 1, "ctx_lo": 1000, "ctx_hi": 1000, "dtype": "bf16", "gate": True, "lens": 5},
        # A server's decode step: 64 sequences of unequal length.
        {"name": "attn_decode_64", "kind": "attn", "seqs": 64, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "new_lo": 1, "new_hi": 1, "ctx_lo": 200, "ctx_hi": 16000, "dtype": "bf16", "gate": True, "lens": 6},
        # Verify blocks of up to 8 drafted positions on small pages.
        {"name": "attn_verify_16", "kind": "attn", "seqs": 16, "heads": 16, "kv_heads": 2, "dim": 256, "page": 16,
         "new_lo": 2, "new_hi": 9, "ctx_lo": 1000, "ctx_hi": 8000, "dtype": "bf16", "gate": True, "lens": 7},
        # A prompt from an empty cache.
        {"name": "attn_prompt_2k", "kind": "attn", "seqs": 1, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "new_lo": 2048, "new_hi": 2048, "ctx_lo": 0, "ctx_hi": 0, "dtype": "bf16", "gate": True, "lens": 8},
        # One chunk of a long prompt over what is cached of it.
        {"name": "attn_chunk_4k", "kind": "attn", "seqs": 1, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "new_lo": 4096, "new_hi": 4096, "ctx_lo": 28003, "ctx_hi": 28003, "dtype": "bf16", "gate": True, "lens": 9},
        # Prompt chunks of ragged lengths in another head layout and type.
        {"name": "attn_ragged_fp16", "kind": "attn", "seqs": 9, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "new_lo": 1, "new_hi": 900, "ctx_lo": 0, "ctx_hi": 5000, "dtype": "fp16", "gate": False, "lens": 10},
        # A verify block of one sequence: four drafts and the bonus position.
        {"name": "verify_1", "kind": "verify", "seqs": 1, "vocab": 151936, "new_lo": 5, "new_hi": 5,
         "dtype": "fp32", "draft": True, "lens": 11},
        # Verify blocks of a server, unequal numbers of drafts.
        {"name": "verify_64", "kind": "verify", "seqs": 64, "vocab": 151936, "new_lo": 1, "new_hi": 8,
         "dtype": "fp32", "draft": True, "lens": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attn", "attn", "attn", "attn", "verify", "verify"])
    lens = rng.randint(100, 1 << 30)
    if kind == "plan":
        rows = _log(rng, 1, 1000)
        lo = rng.choice([0, 0, 1])
        return {"kind": kind, "rows": rows, "page": rng.choice([16, 32, 64, 128]), "new_lo": lo,
                "new_hi": max(1, _log(rng, 1, 60)), "ctx_lo": 0, "ctx_hi": _log(rng, 10, 9000), "lens": lens}
    heads, kv_heads, dim, rotary = rng.choice([(16, 2, 256, 64), (16, 2, 256, 64), (32, 8, 128, 128), (8, 8, 64, 64),
                                               (20, 4, 128, 64)])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 4000 // seqs))
        return {"kind": kind, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
                "page": page, "new_lo": rng.randint(0, 1), "new_hi": hi, "ctx_lo": 0, "ctx_hi": _log(rng, 1, 2000),
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "lens": lens}
    if kind == "attn":
        form = rng.choice(["decode", "verify", "chunk", "chunk"])
        if form == "decode":
            seqs, lo, hi = _log(rng, 1, 64), 1, 1
            ctx = _log(rng, 1, 16000)
        elif form == "verify":
            seqs, lo, hi = _log(rng, 1, 32), rng.randint(1, 3), rng.randint(4, 17)
            ctx = _log(rng, 1, 12000)
        else:
            seqs, lo = _log(rng, 1, 8), 1
            hi = _log(rng, 17, max(17, 4000 // seqs))
            ctx = _log(rng, 1, 20000 // seqs)
        return {"kind": kind, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "new_lo": lo, "new_hi": hi, "ctx_lo": ctx // 10, "ctx_hi": ctx,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "gate": rng.random() < 0.5, "lens": lens}
    return {"kind": kind, "seqs": _log(rng, 1, 64), "vocab": _log(rng, 500, 150000), "new_lo": rng.randint(1, 2),
            "new_hi": rng.randint(2, 8), "dtype": rng.choice(["fp32", "fp32", "bf16"]),
            "draft": rng.random() < 0.7, "lens": lens}


# ---- a step's sequences -----------------------------------------------------------

def lengths(case):
    """(cached, new) positions per sequence: functions of the case alone."""
    rng = random.Random(case["lens"])
    n = case.get("seqs", case.get("rows"))
    cached = [rng.randint(case.get("ctx_lo", 0), case.get("ctx_hi", 0)) for _ in range(n)]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    if sum(new) == 0:
        new[0] = 1
    return cached, new


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _block_table(lens, page, seed):
    """Pages in an arbitrary order, as a server's pool hands them out."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 3
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = max(1, max(counts)) + 1
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    return rows, pages


# ---- inputs -----------------------------------------------------------------------

def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attn": _prepare_attn,
            "verify": _prepare_verify}[case["kind"]](case, seed)


def _prepare_plan(case, seed):
    cached, new = lengths(case)
    page, rows = case["page"], len(cached)
    rng = random.Random(seed)
    # Another seed: the same multiset of sequences on other rows and pages.
    both = list(zip(cached, new))
    rng.shuffle(both)
    cached, new = [c for c, _ in both], [n for _, n in both]
    held = [-(-c // page) for c in cached]
    need = [max(h, -(-(c + n) // page)) for h, c, n in zip(held, cached, new)]
    pages = sum(need) + 40
    width = max(max(need), 1) + 2
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        if h:
            table[r, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
        at += h
    free = order[at:]
    tokens = sum(new) + 5   # a captured step is sized for more positions than it gets
    state = dict(case=case, tokens=tokens, new=_ints(new), lengths=_ints(cached), held=_ints(held),
                 table=table.cuda(), free=_ints(free + [0] * (pages - len(free))), free_count=_ints([len(free)]))
    if own:
        from lightreason_amd.paged import PageTable
        pt = PageTable(rows, pages, page, max_pages=width, device="cuda")
        pt.table.copy_(state["table"])
        pt.held.copy_(state["held"])
        pt.lengths.copy_(state["lengths"])
        pt.free_pages.copy_(state["free"])
        pt.state[:1].copy_(state["free_count"])
        state["pages"] = pt
        state["out"] = pt.new_plan(tokens)
    return state


def _prepare_append(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    cached, new = lengths(case)
    page, D, R = case["page"], case["dim"], case["rotary"]
    lens = [c + n for c, n in zip(cached, new)]
    table, pages = _block_table(lens, page, seed)
    positions = [c + i for c, n in zip(cached, new) for i in range(n)]
    slots = [table[s][(c + i) // page] * page + (c + i) % page
             for s, (c, n) in enumerate(zip(cached, new)) for i in range(n)]
    N, H, K = len(slots), case["heads"], case["kv_heads"]

    def normal(*shape):
        return torch.empty(shape, device="cuda").normal_(generator=g)

    # Rotary table of every position the model serves up to here.
    P = max(max(positions) + 1, 1)
    inv = 10000000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = torch.arange(P, dtype=torch.float64, device="cuda")[:, None] * inv[None]
    angle = torch.cat([angle, angle], dim=1)
    return dict(case=case, q_gate=normal(N, H, 2 * D).to(dt), k=normal(N, K, D).to(dt), v=normal(N, K, D).to(dt),
                q_norm=(0.1 * normal(D)).to(dt), k_norm=(0.1 * normal(D)).to(dt),
                cos=angle.cos().float(), sin=angle.sin().float(),
                positions=_ints(positions), slots=_ints(slots, torch.int64),
                k_cache=normal(pages, K, page, D).to(dt), v_cache=normal(pages, K, page, D).to(dt),
                q_out=torch.zeros(N, H, D, dtype=dt, device="cuda"))


def _prepare_attn(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    cached, new = lengths(case)
    page, D, H, K = case["page"], case["dim"], case["heads"], case["kv_heads"]
    lens = [c + n for c, n in zip(cached, new)]
    table, pages = _block_table(lens, page, seed)
    N = sum(new)

    def normal(*shape):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)

    # Normed heads: elements of unit size, so scores q.k / sqrt(D) are of unit
    # size too; a common direction makes some positions weigh more.
    k_cache = normal(pages, K, page, D)
    q = normal(N, H, D)
    q += normal(1, H, D)
    return dict(case=case, cached=cached, new=new, q=q, k_cache=k_cache, v_cache=normal(pages, K, page, D),
                gate=normal(N, H, D) if case["gate"] else None, table=_ints(table), starts=_ints(_starts(new)),
                kv_lengths=_ints(lens), max_new=max(new), out=torch.zeros(N, H, D, dtype=dt, device="cuda"))


def _prepare_verify(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    _, new = lengths(case)
    N, V = sum(new), case["vocab"]
    logits = torch.empty(N, V, device="cuda").normal_(0.0, 2.5, generator=g)
    target = torch.softmax(logits, dim=1).to(dt)
    state = dict(case=case, target=target, starts=_ints(_starts(new)), draft=None,
                 uniforms=torch.rand(N, generator=g, device="cuda"),
                 samples=torch.rand(len(new), generator=g, device="cuda"))
    # The drafter agrees with the target up to noise; its tokens are sampled
    # from its own probabilities (exponential race), or are its best ones.
    logits += torch.empty(N, V, device="cuda").normal_(0.0, 0.7, generator=g)
    if case["draft"]:
        draft = torch.softmax(logits, dim=1)
        race = torch.empty(N, V, device="cuda").exponential_(generator=g)
        drawn = (draft / race).argmax(dim=1)
        state["draft"] = draft.to(dt)
    else:
        drawn = logits.argmax(dim=1)
    # Row i's drafted token is fed at row i + 1 of its block.
    tokens = torch.randint(0, V, (N,), generator=g, device="cuda")
    tokens[1:] = drawn[:-1]
    state["tokens"] = tokens
    return state


# ---- one pass ---------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attn": _own_attn, "verify": _own_verify}[kind](state)
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn, "verify": _plain_verify}[kind](state)


def _own_plan(s):
    plan = s["pages"].plan(s["new"], s["tokens"], out=s["out"])
    return dict(starts=plan.starts, kv_lengths=plan.kv_lengths, held=plan.held, positions=plan.positions,
                slots=plan.slots, table=s["pages"].table)


def _own_append(s):
    from lightreason_amd.paged import paged_append
    D = s["case"]["dim"]
    paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q_gate"][:, :, :D], q_norm=s["q_norm"],
                 k_norm=s["k_norm"], eps=EPS, cos=s["cos"], sin=s["sin"], positions=s["positions"], q_out=s["q_out"])
    return dict(q=s["q_out"], k=s["k_cache"], v=s["v_cache"])


def _own_attn(s):
    from lightreason_amd.paged import paged_attention
    return paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["kv_lengths"],
                           max_new=s["max_new"], gate=s["gate"], out=s["out"])


def _own_verify(s):
    from lightreason_amd.verify import verify_drafts
    accepted, token = verify_drafts(s["tokens"], s["target"], s["starts"], s["uniforms"], s["samples"],
                                    draft=s["draft"])
    return dict(accepted=accepted, token=token)


def _plain_plan(s):
    page, N = s["case"]["page"], s["tokens"]
    new, old, held, table = s["new"].long(), s["lengths"].long(), s["held"].long(), s["table"]
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    starts = torch.cat([zero, torch.cumsum(new, 0)])
    total = old + new
    need = torch.maximum(held, (total + page - 1) // page)
    before = torch.cat([zero, torch.cumsum(need - held, 0)])[:-1]
    # Fresh pages, from the top of the free stack, rows in order.
    column = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (column >= held[:, None]) & (column < need[:, None])
    pick = s["free_count"].long() - 1 - (before[:, None] + column - held[:, None])
    table.copy_(torch.where(fresh, s["free"][pick.clamp(0, s["free"].numel() - 1)], table))
    index = torch.arange(N, device="cuda")
    row = torch.searchsorted(starts[1:], index, right=True)
    live = row < new.numel()
    row = row.clamp(max=new.numel() - 1)
    position = torch.where(live, old[row] + index - starts[row], zero)
    entry = table[row, position // page].long()
    slots = torch.where(live, entry * page + position % page, zero - 1)
    return dict(starts=starts.int(), kv_lengths=total.int(), held=need.int(), positions=position.int(), slots=slots,
                table=table)


def _norm_rope(x, weight, cos, sin, D, R):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * (1.0 + weight.float())
    rot, rest = x[..., :R], x[..., R:]
    half = torch.cat([-rot[..., R // 2:], rot[..., :R // 2]], dim=-1)
    return torch.cat([rot * cos[:, None] + half * sin[:, None], rest], dim=-1)


def _plain_append(s):
    D, R, page = s["case"]["dim"], s["case"]["rotary"], s["case"]["page"]
    p = s["positions"].long()
    cos, sin = s["cos"][p], s["sin"][p]
    s["q_out"].copy_(_norm_rope(s["q_gate"][:, :, :D], s["q_norm"], cos, sin, D, R))
    block, row = s["slots"] // page, s["slots"] % page
    s["k_cache"][block, :, row] = _norm_rope(s["k"], s["k_norm"], cos, sin, D, R).to(s["k_cache"].dtype)
    s["v_cache"][block, :, row] = s["v"]
    return dict(q=s["q_out"], k=s["k_cache"], v=s["v_cache"])


def _sequence(s, i, dtype):
    """Keys and values [kv_heads, length, dim] of sequence i, in order."""
    case = s["case"]
    n = s["cached"][i] + s["new"][i]
    blocks = s["table"][i, :-(-n // case["page"])].long()

    def rows(cache):
        x = cache[blocks].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])
        return x[:, :n].to(dtype).contiguous()
    return rows(s["k_cache"]), rows(s["v_cache"])


def _plain_attn(s):
    case, out = s["case"], s["out"]
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    at = 0
    for i, (c, n) in enumerate(zip(s["cached"], s["new"])):
        if n == 0:
            continue
        k, v = _sequence(s, i, torch.float32)
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (H * (c + n)))
        for a in range(0, n, step):
            b = min(n, a + step)
            q = s["q"][at + a:at + b].float().reshape(b - a, K, H // K, D).permute(1, 2, 0, 3)
            scores = torch.matmul(q.reshape(K, -1, D), kt).view(K, H // K, b - a, c + n) * D ** -0.5
            seen = torch.arange(c + n, device="cuda")[None] <= torch.arange(c + a, c + b, device="cuda")[:, None]
            scores = torch.where(seen, scores, -math.inf)
            w = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
            o = torch.matmul(w.reshape(K, -1, c + n), v).view(K, H // K, b - a, D)
            o = (o / w.sum(dim=-1, keepdim=True)).permute(2, 0, 1, 3).reshape(b - a, H, D)
            if s["gate"] is not None:
                o = o / (1.0 + torch.exp(-s["gate"][at + a:at + b].float()))
            out[at + a:at + b] = o.to(out.dtype)
        at += n
    return out


def _plain_verify(s):
    # In 64 bits: a drawn token is the first whose running sum passes a border.
    tokens, starts, target, draft = s["tokens"], s["starts"].long(), s["target"], s["draft"]
    N, V = target.shape
    zero = torch.zeros(1, dtype=torch.float64, device="cuda")
    index = torch.arange(N - 1, device="cuda")
    fed = tokens[1:]
    p = target[index, fed].double()
    q = draft[index, fed].double() if draft is not None else torch.ones_like(p)
    ok = torch.cat([s["uniforms"][:-1].double() * q < p, torch.zeros(1, dtype=torch.bool, device="cuda")])
    # Drafts of a block: its rows but the last; accepted: those before the
    # first that fails.
    row = torch.arange(N, device="cuda")
    first, last = starts[:-1, None], starts[1:, None] - 1
    fails = (row[None] >= first) & (row[None] < last) & ~ok[None]
    stop = torch.where(fails, row[None], N).amin(dim=1)
    stop = torch.minimum(stop, last[:, 0])
    accepted = stop - starts[:-1]
    full = target[stop].double()
    rejected = (stop < last[:, 0])[:, None]
    if draft is not None:
        rest = (full - draft[stop].double()).clamp(min=0.0)
    else:
        rest = full.scatter(1, tokens[(stop + 1).clamp(max=N - 1)][:, None], 0.0)
    rest = torch.where(rest.sum(dim=1, keepdim=True) > 0.0, rest, full)
    mass = torch.where(rejected, rest, full)
    running = torch.cumsum(mass, dim=1)
    border = s["samples"].double()[:, None] * running[:, -1:]
    token = (running <= border).sum(dim=1)
    # A sample that rounds up to the whole sum takes the last token with mass.
    ends = (mass > zero).long() * torch.arange(V, device="cuda")
    return dict(accepted=accepted.int(), token=torch.minimum(token, ends.amax(dim=1)))


# ---- work and the definition in 64 bits ---------------------------------------------

def work(case):
    cached, new = lengths(case)
    N = sum(new)
    if case["kind"] == "plan":
        rows, page = len(cached), case["page"]
        taken = sum(max(0, -(-(c + n) // page) - -(-c // page)) for c, n in zip(cached, new))
        return {"bytes": 4 * rows * 6 + 12 * N + 8 * taken, "flops": 10 * (rows + N)}
    if case["kind"] == "append":
        H, K, D, R = case["heads"], case["kv_heads"], case["dim"], case["rotary"]
        return {"bytes": N * (2 * 2 * D * (H + 2 * K) + 2 * 4 * R + 12), "flops": N * (H + K) * (4 * D + 4 * R)}
    if case["kind"] == "attn":
        H, K, D = case["heads"], case["kv_heads"], case["dim"]
        held = sum(c + n for c, n in zip(cached, new) if n)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
        rows = 3 if case["gate"] else 2
        return {"bytes": 2 * D * (2 * K * held + rows * H * N), "flops": 4 * D * H * pairs}
    # One probability row of each side per block, and the drafts' entries.
    size = 2 if case["dtype"] == "bf16" else 4
    sides = 2 if case["draft"] else 1
    return {"bytes": sides * size * (len(new) * case["vocab"] + N) + 12 * N + 16 * len(new),
            "flops": 3 * len(new) * case["vocab"]}


def exact(case, seed):
    return {"plan": _exact_plan, "append": _exact_append, "attn": _exact_attn,
            "verify": _exact_verify}[case["kind"]](case, seed)


def _exact_plan(case, seed):
    s = _prepare_plan(case, seed)
    page = case["page"]
    new, old, held = s["new"].tolist(), s["lengths"].tolist(), s["held"].tolist()
    table, free = s["table"].tolist(), s["free"].tolist()[:int(s["free_count"])]
    starts, total, positions, slots = [0], [], [], []
    for r, (n, c) in enumerate(zip(new, old)):
        while held[r] * page < c + n:
            table[r][held[r]] = free.pop()
            held[r] += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r][p // page] * page + p % page)
        starts.append(starts[-1] + n)
        total.append(c + n)
    pad = s["tokens"] - len(slots)
    return dict(starts=_ints(starts), kv_lengths=_ints(total), held=_ints(held), positions=_ints(positions + [0] * pad),
                slots=_ints(slots + [-1] * pad, torch.int64), table=_ints(table))


def _exact_append(case, seed):
    s = _prepare_append(case, seed)
    D, R = case["dim"], case["rotary"]
    index = s["positions"].long()
    c, n = s["cos"].double()[index][:, None, :], s["sin"].double()[index][:, None, :]

    def turned(x, weight):
        x = x.double()
        scale = 1.0 / torch.sqrt(torch.sum(x ** 2, dim=-1, keepdim=True) / D + EPS)
        y = x * scale * (weight.double() + 1.0)
        a, b = y[..., :R // 2].clone(), y[..., R // 2:R].clone()
        y[..., :R // 2] = a * c[..., :R // 2] - b * n[..., :R // 2]
        y[..., R // 2:R] = b * c[..., R // 2:] + a * n[..., R // 2:]
        return y
    block, row = s["slots"].div(case["page"], rounding_mode="floor"), s["slots"].remainder(case["page"])
    k, v = s["k_cache"].double(), s["v_cache"].double()
    k[block, :, row] = turned(s["k"], s["k_norm"])
    v[block, :, row] = s["v"].double()
    return dict(q=turned(s["q_gate"][:, :, :D], s["q_norm"]), k=k, v=v)


def _exact_attn(case, seed):
    s = _prepare_attn(case, seed)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (c, n) in enumerate(zip(s["cached"], s["new"])):
        k, v = _sequence(s, i, torch.float64)
        for h in range(H):
            kh, vh = k[h * K // H], v[h * K // H]
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                score = (s["q"][at + a:at + b, h].double() @ kh.t()) / math.sqrt(D)
                later = torch.arange(c + n, device="cuda")[None] > torch.arange(c + a, c + b, device="cuda")[:, None]
                out[at + a:at + b, h] = torch.softmax(score.masked_fill(later, -math.inf), dim=1) @ vh
        at += n
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out


def _exact_verify(case, seed):
    s = _prepare_verify(case, seed)
    _, new = lengths(case)
    target, draft, tokens = s["target"], s["draft"], s["tokens"].tolist()
    uniforms, samples = s["uniforms"].double().tolist(), s["samples"].double().tolist()
    accepted, chosen, at = [], [], 0
    for i, n in enumerate(new):
        j = 0
        while j + 1 < n:
            x = tokens[at + j + 1]
            q = float(draft[at + j, x]) if draft is not None else 1.0
            if not uniforms[at + j] * q < float(target[at + j, x]):
                break
            j += 1
        mass = target[at + j].double()
        if j + 1 < n:
            rest = mass.clone()
            if draft is not None:
                rest = torch.relu(rest - draft[at + j].double())
            else:
                rest[tokens[at + j + 1]] = 0.0
            if float(rest.sum()) > 0.0:
                mass = rest
        running = mass.cumsum(0)
        token = int(torch.searchsorted(running, samples[i] * running[-1], right=True))
        chosen.append(min(token, int(mass.nonzero()[-1])))
        accepted.append(j)
        at += n
    return dict(accepted=_ints(accepted), token=_ints(chosen, torch.int64))
