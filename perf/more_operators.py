"""Operators around the recurrent layers and beam search, as cases that can be
timed and compared with plain forms: the gated delta rule over packed
sequences (prompts), its gradient, a serving step over a pool of states
(single tokens and verify blocks), the choice of the best continuations of a
group of beams, and the beams' states and cached pages following their parents.

With ``own`` false ``run`` computes each operator in elementary torch
operations; with ``own`` true it calls ``lightreason_amd.scan``,
``lightreason_amd.beam`` and ``lightreason_amd.paged``.  Head layouts are the
35B model's (16 key heads, 32 value heads of width 128; caches of 2 heads of
width 256) and generic ones.
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
        # One long prompt through a linear-attention layer of the 35B model.
        {"name": "scan_8k", "kind": "scan", "seqs": 1, "lo": 8192, "hi": 8192, "lens": 1, "key_heads": 16, "heads": 32,
         "dim": 128, "value_dim": 128, "dtype": "bf16", "initial": False, "normalize": True},
        # Short ragged requests of a small model, continued from states.
        {"name": "scan_ragged", "kind": "scan", "seqs": 9, "lo": 1, "hi": 301, "lens": 2, "key_heads": 4, "heads": 4,
         "dim": 64, "value_dim": 64, "dtype": "fp16", "initial": True, "normalize": False},
        # A training step's packed documents through one layer, with all gradients.
        {"name": "train_4k", "kind": "train", "seqs": 5, "lo": 300, "hi": 1500, "lens": 3, "key_heads": 16, "heads": 32,
         "dim": 128, "value_dim": 128, "dtype": "bf16", "initial": False, "normalize": True},
        # A few short sequences of a small model with learned first states.
        {"name": "train_small", "kind": "train", "seqs": 3, "lo": 20, "hi": 190, "lens": 4, "key_heads": 2, "heads": 4,
         "dim": 64, "value_dim": 128, "dtype": "fp16", "initial": True, "normalize": False},
        # One sequence, one token: latency.
        {"name": "step_1", "kind": "step", "seqs": 1, "lo": 1, "hi": 1, "lens": 5, "key_heads": 16, "heads": 32,
         "dim": 128, "value_dim": 128, "dtype": "bf16", "normalize": True},
        # A full server's decode step.
        {"name": "step_256", "kind": "step", "seqs": 256, "lo": 1, "hi": 1, "lens": 6, "key_heads": 16, "heads": 32,
         "dim": 128, "value_dim": 128, "dtype": "bf16", "normalize": True},
        # One request with four beams; a finished one among them.
        {"name": "beam_4", "kind": "beam", "groups": 1, "beams": 4, "vocab": 151936, "dtype": "bf16", "done": 0.25,
         "masked": 0.0},
        # A batch of requests with eight beams each, a grammar masking most tokens of some.
        {"name": "beam_32x8", "kind": "beam", "groups": 32, "beams": 8, "vocab": 151936, "dtype": "fp32", "done": 0.1,
         "masked": 0.3},
        # States of four beams over three linear-attention layers.
        {"name": "fork_rows_4", "kind": "rows", "rows": 4, "layers": 3, "moved": 0.4, "heads": 32, "dim": 128,
         "conv": 8192},
        # All 30 linear-attention layers' states of a batch of beams.
        {"name": "fork_rows_32", "kind": "rows", "rows": 32, "layers": 30, "moved": 0.4, "heads": 32, "dim": 128,
         "conv": 8192},
        # Cached pages of one request's four beams, ten attention layers.
        {"name": "fork_pages_4", "kind": "pages", "groups": 1, "beams": 4, "layers": 10, "kv_heads": 2, "dim": 256,
         "page": 64, "lo": 900, "hi": 900, "lens": 7, "moved": 0.5, "fresh": False},
        # Prompts of eight requests given to all their beams, which hold nothing yet.
        {"name": "fork_pages_8x4", "kind": "pages", "groups": 8, "beams": 4, "layers": 10, "kv_heads": 2, "dim": 256,
         "page": 16, "lo": 300, "hi": 3000, "lens": 8, "moved": 1.0, "fresh": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["scan", "train", "step", "beam", "rows", "pages"])
    lens = rng.randrange(1 << 30)
    if kind in ("scan", "train", "step"):
        key_heads, heads, dim, value_dim = rng.choice(
            [(16, 32, 128, 128), (4, 4, 64, 64), (2, 4, 64, 128), (8, 8, 128, 64), (3, 9, 128, 128), (16, 16, 128, 128)])
        case = {"kind": kind, "lens": lens, "key_heads": key_heads, "heads": heads, "dim": dim, "value_dim": value_dim,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "normalize": rng.random() < 0.6}
        if kind == "step":
            case["hi"] = rng.choice([1, 1, 2, 4, 7, 16])
            case["seqs"] = _log(rng, 1, 256 // case["hi"])
            case["lo"] = rng.randint(1, case["hi"])
            return case
        total = _log(rng, 8, 8000 if kind == "scan" else 3600)
        case["seqs"] = _log(rng, 1, min(32, total))
        case["hi"] = max(1, total // case["seqs"])
        case["lo"] = _log(rng, 1, case["hi"])
        case["initial"] = rng.random() < 0.5
        return case
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _log(rng, 300, 151936)
        return {"kind": kind, "groups": _log(rng, 1, 256 // beams), "beams": beams, "vocab": vocab,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "done": rng.choice([0.0, 0.2]),
                "masked": rng.choice([0.0, 0.5])}
    if kind == "rows":
        return {"kind": kind, "rows": _log(rng, 2, 32), "layers": _log(rng, 1, 30), "moved": rng.uniform(0.0, 0.8),
                "heads": rng.choice([4, 32]), "dim": rng.choice([64, 128]), "conv": rng.choice([1001, 8192])}
    beams = rng.choice([2, 3, 4, 8])
    hi = _log(rng, 16, 3000)
    return {"kind": kind, "groups": _log(rng, 1, 32 // beams), "beams": beams, "layers": _log(rng, 1, 10),
            "kv_heads": rng.choice([1, 2, 4]), "dim": rng.choice([64, 128, 256]) if hi < 1500 else 128,
            "page": rng.choice([16, 64, 128]), "lo": _log(rng, 1, hi), "hi": hi, "lens": lens,
            "moved": rng.uniform(0.2, 1.0), "fresh": rng.random() < 0.4}


def lengths(case):
    rng = random.Random(case["lens"])
    out = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    out[rng.randrange(len(out))] = case["hi"]
    return out


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ---- inputs -------------------------------------------------------------------------

def prepare(case, seed):
    kind = case["kind"]
    return {"scan": _prepare_scan, "train": _prepare_scan, "step": _prepare_scan, "beam": _prepare_beam,
            "rows": _prepare_rows, "pages": _prepare_pages}[kind](case, seed)


def _prepare_scan(case, seed):
    gen = _generator(seed)
    new = lengths(case)
    N, S, H, K = sum(new), len(new), case["heads"], case["key_heads"]
    D, E, dtype = case["dim"], case["value_dim"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    # Queries, keys and values as they come out of the convolution: side by
    # side in one row per token.
    qkv = torch.nn.functional.silu(normal(N, 2 * K * D + H * E) * 1.5)
    if not case["normalize"]:
        qk = qkv[:, :2 * K * D].reshape(N, 2 * K, D)
        qkv[:, :2 * K * D] = (qk / qk.norm(dim=-1, keepdim=True)).reshape(N, -1)
    qkv = qkv.to(dtype)
    s = dict(case=case, new=new, starts=_ints([0] + torch.tensor(new).cumsum(0).tolist()),
             q=qkv[:, :K * D].view(N, K, D), k=qkv[:, K * D:2 * K * D].view(N, K, D),
             v=qkv[:, 2 * K * D:].view(N, H, E), beta=torch.sigmoid(normal(N, H)).to(dtype))
    # Decays from e^-1.6 to almost 1 a token, by head.
    rate = torch.rand(H, generator=gen, device="cuda") * 15 + 1
    step = torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    bias = step + torch.log(-torch.expm1(-step))
    s["g"] = -rate * torch.nn.functional.softplus(normal(N, H) * 0.5 + bias)
    s["initial"] = normal(S, H, D, E) * 0.3 if case.get("initial") else None
    if case["kind"] == "train":
        s["d_out"] = normal(N, H, E).to(dtype)
        s["d_final"] = normal(S, H, D, E) * 0.1
        s["leaves"] = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["v"], s["g"], s["beta"])]
        if s["initial"] is not None:
            s["leaves"].append(s["initial"].requires_grad_())
    if case["kind"] == "step":
        order = torch.randperm(2 * S, generator=gen, device="cuda").int()
        s["states"] = normal(2 * S, H, D, E) * 0.3
        s["slots"], s["into"] = order[:S].contiguous(), order[S:].contiguous()
        s["out"] = torch.zeros(N, H, E, dtype=dtype, device="cuda")
    return s


def _prepare_beam(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    G, W, V = case["groups"], case["beams"], case["vocab"]
    logits = torch.randn(G * W, V, generator=gen, device="cuda") * 2.5
    for r in range(G * W):
        if rng.random() < case["masked"]:
            # A grammar leaves some tens of tokens, or none.
            keep = torch.randint(V, (rng.choice([0, 1, 3, 40]),), generator=gen, device="cuda")
            row = torch.full((V,), -math.inf, device="cuda")
            row[keep] = logits[r, keep]
            logits[r] = row
    scores = -torch.rand(G, W, generator=gen, device="cuda") * 12.0
    for i in range(G):
        if W > 1 and rng.random() < 0.2:
            scores[i, 1:] = -math.inf   # a first step: one beam lives
    done = torch.tensor([[rng.random() < case["done"] for _ in range(W)] for _ in range(G)], device="cuda")
    return dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), scores=scores, finished=done)


def _family(rng, rows, moved):
    """Parents of rows 0 .. rows - 1: some rows keep their place, the others follow one that does."""
    keeps = [rng.random() >= moved for _ in range(rows)]
    keeps[rng.randrange(rows)] = True
    stay = [r for r in range(rows) if keeps[r]]
    return [r if keeps[r] else rng.choice(stay) for r in range(rows)]


def _prepare_rows(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    R, H, D = case["rows"], case["heads"], case["dim"]
    tensors = []
    for _ in range(case["layers"]):
        tensors.append(torch.randn(R, H, D, D, generator=gen, device="cuda"))
        tensors.append(torch.randn(R, case["conv"], 4, generator=gen, device="cuda").bfloat16())
    return dict(case=case, tensors=tensors, parents=_ints(_family(rng, R, case["moved"])))


def _page_rows(case):
    """Cached lengths and pages held, row by row: a group's beams are equally long, or its first one alone has
    anything."""
    rng = random.Random(case["lens"])
    out, held = [], []
    for _ in range(case["groups"]):
        n = _log(rng, case["lo"], case["hi"])
        for b in range(case["beams"]):
            out.append(n if b == 0 or not case["fresh"] else 0)
            held.append(-(-out[-1] // case["page"]))
    return out, held


def _page_parents(case, seed):
    rng, W = random.Random(seed), case["beams"]
    parents = []
    for i in range(case["groups"]):
        family = [0] * W if case["fresh"] else _family(rng, W, case["moved"])
        parents += [i * W + p for p in family]
    return parents


def _prepare_pages(case, seed):
    gen = _generator(seed)
    R, page = case["groups"] * case["beams"], case["page"]
    cached, held = _page_rows(case)
    width = max(held) + 2
    # Room for every row to hold what its group's longest does, and some more.
    total = case["beams"] * sum(held[::case["beams"]]) + 3
    order = torch.randperm(total, generator=gen, device="cuda").tolist()
    table = [[-1] * width for _ in range(R)]
    for r in range(R):
        for j in range(held[r]):
            table[r][j] = order.pop()
    shape = (case["layers"], total, case["kv_heads"], page, case["dim"])
    caches = [torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    s = dict(case=case, table=_ints(table), held=_ints(held), lengths=_ints(cached), parents=_ints(_page_parents(case, seed)),
             free=_ints(order + [0] * (total - len(order))), count=_ints([len(order)]), k_cache=caches[0],
             v_cache=caches[1])
    if own:
        from lightreason_amd.paged import PageTable
        pool = PageTable(R, total, page, max_pages=width)
        pool.table.copy_(s["table"])
        pool.held.copy_(s["held"])
        pool.lengths.copy_(s["lengths"])
        pool.free_pages.copy_(s["free"])
        pool.state[:1].copy_(s["count"])
        s["pool"] = pool
    return s


# ---- one pass -----------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


def _own_scan(s):
    from lightreason_amd.scan import delta_scan
    out, final = delta_scan(s["q"], s["k"], s["v"], s["g"], s["beta"], s["starts"], initial=s["initial"],
                            normalize=s["case"]["normalize"])
    return dict(out=out, final=final)


def _own_train(s):
    from lightreason_amd.scan import delta_scan
    leaves = s["leaves"]
    out, final = delta_scan(*leaves[:5], s["starts"], initial=leaves[5] if len(leaves) > 5 else None,
                            normalize=s["case"]["normalize"])
    grads = torch.autograd.grad([out, final], leaves, [s["d_out"], s["d_final"]])
    return dict(out=out.detach(), final=final.detach(), grads=list(grads))


def _own_step(s):
    from lightreason_amd.scan import delta_step
    delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["starts"], s["states"], slots=s["slots"], into=s["into"],
               normalize=s["case"]["normalize"], max_new=s["case"]["hi"], out=s["out"])
    return dict(out=s["out"], states=s["states"])


def _own_beam(s):
    from lightreason_amd.beam import beam_select
    tokens, parents, scores = beam_select(s["logits"], s["scores"], finished=s["finished"])
    return dict(tokens=tokens, parents=parents, scores=scores)


def _own_rows(s):
    from lightreason_amd.beam import fork_rows
    fork_rows(s["parents"], s["tensors"])
    return s["tensors"]


def _own_pages(s):
    pool = s["pool"]
    pool.fork(s["parents"], s["k_cache"], s["v_cache"])
    return dict(table=pool.table, held=pool.held, lengths=pool.lengths, count=pool.state[:1], k=s["k_cache"],
                v=s["v_cache"])


# ---- plain forms --------------------------------------------------------------------

def _unit(x, normalize):
    x = x.float()
    if not normalize:
        return x, None
    r = torch.rsqrt((x * x).sum(dim=-1, keepdim=True) + EPS)
    return x * r, r


def _padded(s):
    """The packed rows as [step][sequence], the longest sequence first, and how many sequences each step has."""
    new = s["new"]
    order = sorted(range(len(new)), key=lambda i: -new[i])
    starts = [sum(new[:i]) for i in range(len(new))]
    longest = new[order[0]]
    steps = [[starts[i] + t for i in order if new[i] > t] for t in range(longest)]
    counts = [len(x) for x in steps]
    return _ints(order, torch.int64), _ints([i for x in steps for i in x], torch.int64), counts


def _forward(s, first, keep):
    """The recurrence, step by step over all sequences: outputs by packed row, last states by sequence, and with
    `keep` what the gradient needs."""
    case = s["case"]
    H, K, D, E = case["heads"], case["key_heads"], case["dim"], case["value_dim"]
    N, S = s["q"].shape[0], len(s["new"])
    order, index, counts = _padded(s)
    q, q_scale = _unit(s["q"].detach(), case["normalize"])
    k, k_scale = _unit(s["k"].detach(), case["normalize"])
    scale = D ** -0.5
    wide_q, wide_k = ((x.repeat_interleave(H // K, dim=1)[index]) for x in (q * scale, k))
    v, beta = s["v"].detach().float()[index], s["beta"].detach().float()[index]
    decay = torch.exp(s["g"].detach())[index]
    state = torch.zeros(S, H, D, E, device="cuda") if first is None else first.detach()[order].clone()
    out = torch.empty(N, H, E, device="cuda")
    kept, left, at = [], [], 0
    for n in counts:
        kt, qt, vt = wide_k[at:at + n], wide_q[at:at + n], v[at:at + n]
        a, b = decay[at:at + n], beta[at:at + n]
        before = state[:n]
        faded = before * a[:, :, None, None]
        rest = vt - torch.matmul(kt[:, :, None, :], faded)[:, :, 0]
        u = rest * b[:, :, None]
        after = faded + kt[:, :, :, None] * u[:, :, None, :]
        out[at:at + n] = torch.matmul(qt[:, :, None, :], after)[:, :, 0]
        if keep:
            kept.append(before)
            left.append(rest)
            state = torch.cat([after, state[n:]]) if n < S else after
        else:
            state[:n] = after
        at += n
    packed = torch.empty_like(out)
    packed[index] = out
    final = torch.empty_like(state)
    final[order] = state
    return packed, final, dict(order=order, index=index, counts=counts, q=q, k=k, q_scale=q_scale, k_scale=k_scale,
                               wide_q=wide_q, wide_k=wide_k, beta=beta, decay=decay, kept=kept, left=left, state=state)


def _plain_scan(s):
    out, final, _ = _forward(s, s["initial"], False)
    return dict(out=out.to(s["v"].dtype), final=final)


def _plain_step(s):
    out, final, _ = _forward(s, s["states"][s["slots"].long()], False)
    s["states"][s["into"].long()] = final
    s["out"].copy_(out)
    return dict(out=s["out"], states=s["states"])


def _plain_train(s):
    case = s["case"]
    H, K, D, E = case["heads"], case["key_heads"], case["dim"], case["value_dim"]
    N = s["q"].shape[0]
    out, final, m = _forward(s, s["initial"], True)
    index, order = m["index"], m["order"]
    d_out = s["d_out"].float()[index]
    d_state = s["d_final"][order].clone()
    dq, dk = torch.empty(N, H, D, device="cuda"), torch.empty(N, H, D, device="cuda")
    dv = torch.empty(N, H, E, device="cuda")
    dg, db = torch.empty(N, H, device="cuda"), torch.empty(N, H, device="cuda")
    at, after = N, m["state"]
    for n, before, rest in zip(reversed(m["counts"]), reversed(m["kept"]), reversed(m["left"])):
        at -= n
        kt, qt = m["wide_k"][at:at + n], m["wide_q"][at:at + n]
        b, a, do = m["beta"][at:at + n, :, None], m["decay"][at:at + n], d_out[at:at + n]
        # The state after this step is the one kept before the next, but for sequences that end here.
        now = before * a[:, :, None, None]
        u = rest * b
        d_now = d_state[:n] + qt[:, :, :, None] * do[:, :, None, :]
        dq[at:at + n] = torch.matmul(now, do[:, :, :, None])[:, :, :, 0] + kt * (u * do).sum(dim=-1, keepdim=True)
        du = torch.matmul(kt[:, :, None, :], d_now)[:, :, 0]
        db[at:at + n] = (du * rest).sum(dim=-1)
        dr = du * b
        dv[at:at + n] = dr
        dk[at:at + n] = (torch.matmul(d_now, u[:, :, :, None]) - torch.matmul(now, dr[:, :, :, None]))[:, :, :, 0]
        d_now = d_now - kt[:, :, :, None] * dr[:, :, None, :]
        dg[at:at + n] = (d_now * now).sum(dim=(-1, -2))
        d_state[:n] = d_now * a[:, :, None, None]

    def heads(d, x, r):
        d = d.view(N, K, H // K, D).sum(dim=2)
        return d if r is None else r * (d - x * (x * d).sum(dim=-1, keepdim=True))

    def packed(x):
        y = torch.empty_like(x)
        y[index] = x
        return y
    dtype = s["q"].dtype
    grads = [heads(packed(dq) * D ** -0.5, m["q"], m["q_scale"]).to(dtype), heads(packed(dk), m["k"], m["k_scale"]).to(dtype),
             packed(dv).to(dtype), packed(dg), packed(db).to(dtype)]
    if s["initial"] is not None:
        first = torch.empty_like(d_state)
        first[order] = d_state
        grads.append(first)
    return dict(out=out.to(dtype), final=final, grads=grads)


def _plain_beam(s):
    # In 64 bits: candidates next to each other must not change places.
    G, W, V = s["case"]["groups"], s["case"]["beams"], s["case"]["vocab"]
    x = s["logits"].view(G, W, V).double()
    done = s["finished"]
    top = x.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    total = top + torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))
    c = torch.where(torch.isfinite(x), s["scores"].double()[:, :, None] + (x - total), -math.inf)
    only = torch.full_like(c, -math.inf)
    only[:, :, 0] = s["scores"].double()
    c = torch.where(done[:, :, None], only, c).view(G, W * V)
    place = torch.arange(W * V, device="cuda")
    values, picks = [], []
    for _ in range(W):
        best = c.amax(dim=1, keepdim=True)
        pick = torch.where(c == best, place[None], W * V).amin(dim=1, keepdim=True)
        values.append(best)
        picks.append(pick)
        c.scatter_(1, pick, -math.inf)
    value, pick = torch.cat(values, dim=1), torch.cat(picks, dim=1)
    valid = value > -math.inf
    beam, token = pick // V, pick % V
    token = torch.where(done.gather(1, beam), -1, token)
    # A beam's best continuation stays in its row, the others go to the rows left over, in order.
    rank = torch.arange(W, device="cuda")
    again = ((beam[:, :, None] == beam[:, None, :]) & valid[:, None, :] & (rank[None, :] < rank[:, None])).any(dim=2)
    stays, moves = valid & ~again, valid & again
    taken = ((beam[:, :, None] == rank) & stays[:, :, None]).any(dim=1)
    which = torch.cumsum(moves.long(), dim=1) - 1
    spare = torch.cumsum((~taken).long(), dim=1) - 1
    fits = (spare[:, None, :] == which[:, :, None]) & ~taken[:, None, :]
    target = torch.where(stays, beam, torch.where(fits, rank, 0).sum(dim=2))
    target = torch.where(valid, target, W)
    tokens = torch.full((G, W + 1), -1, dtype=torch.int64, device="cuda").scatter(1, target, token)[:, :W]
    parents = torch.cat([rank.expand(G, W), rank.new_zeros(G, 1)], dim=1).scatter(1, target, beam)[:, :W]
    scores = torch.full((G, W + 1), -math.inf, dtype=torch.float64, device="cuda").scatter(1, target, value)[:, :W]
    parents = parents + W * torch.arange(G, device="cuda")[:, None]
    return dict(tokens=tokens.contiguous(), parents=parents.int(), scores=scores.float())


def _plain_rows(s):
    parents = s["parents"].long()
    for t in s["tensors"]:
        t.copy_(t[parents])
    return s["tensors"]


def _plain_pages(s):
    case = s["case"]
    page, parents = case["page"], s["parents"].long()
    R, width = s["table"].shape
    rows = torch.arange(R, device="cuda")
    moves = parents != rows
    need = torch.where(moves, (s["lengths"][parents] + page - 1) // page, 0)
    fresh = (need - s["held"]).clamp(min=0)
    before = torch.cumsum(fresh, dim=0) - fresh
    column = torch.arange(width, device="cuda")
    new = (column[None] >= s["held"][:, None]) & (column[None] < need[:, None])
    at = s["count"].long() - 1 - before[:, None] - (column[None] - s["held"][:, None])
    s["table"].copy_(torch.where(new, s["free"][at.clamp(min=0)], s["table"]))
    s["count"].sub_(fresh.sum())
    s["held"].copy_(torch.maximum(s["held"], need))
    s["lengths"].copy_(s["lengths"][parents])
    # Every position of the rows that follow another, from the parent's page into the row's own.
    longest = int(width * page)
    p = torch.arange(longest, device="cuda")
    seen = moves[:, None] & (p[None] < s["lengths"][:, None])
    row, pos = seen.nonzero(as_tuple=True)
    to, src = s["table"][row, pos // page].long(), s["table"][parents[row], pos // page].long()
    for cache in (s["k_cache"], s["v_cache"]):
        for layer in cache:
            layer[to, :, pos % page] = layer[src, :, pos % page]
    return dict(table=s["table"], held=s["held"], lengths=s["lengths"], count=s["count"], k=s["k_cache"], v=s["v_cache"])


_own = {"scan": _own_scan, "train": _own_train, "step": _own_step, "beam": _own_beam, "rows": _own_rows,
        "pages": _own_pages}
_plain = {"scan": _plain_scan, "train": _plain_train, "step": _plain_step, "beam": _plain_beam, "rows": _plain_rows,
          "pages": _plain_pages}


# ---- work and the definition in 64 bits ---------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("scan", "train", "step"):
        N, S = sum(lengths(case)), case["seqs"]
        H, K, D, E = case["heads"], case["key_heads"], case["dim"], case["value_dim"]
        tokens = N * (2 * (2 * K * D + H * E) + 6 * H)
        out, states = 2 * N * H * E, 4 * S * H * D * E
        if kind == "step":
            return {"bytes": tokens + out + 2 * states, "flops": 6 * D * E * H * N}
        first = states if case["initial"] else 0
        if kind == "scan":
            return {"bytes": tokens + out + states + first, "flops": 6 * D * E * H * N}
        # Forward, then the inputs again with the outputs' gradients, and the inputs' gradients.
        return {"bytes": 3 * tokens + 2 * out + 2 * states + 3 * first, "flops": 18 * D * E * H * N}
    if kind == "beam":
        R = case["groups"] * case["beams"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": R * (size * case["vocab"] + 21), "flops": 4 * R * case["vocab"]}
    if kind == "rows":
        row = case["layers"] * (4 * case["heads"] * case["dim"] ** 2 + 8 * case["conv"])
        # Which rows move is the seed's: their mean.
        return {"bytes": int(2 * row * case["moved"] * (case["rows"] - 1)), "flops": 0}
    cached, _ = _page_rows(case)
    moved = 1.0 if case["fresh"] else case["moved"]
    positions = moved * (case["beams"] - 1) * sum(cached[::case["beams"]])
    return {"bytes": int(2 * 4 * case["layers"] * case["kv_heads"] * case["dim"] * positions), "flops": 0}


def exact(case, seed):
    return {"scan": _exact_scan, "train": _exact_train, "step": _exact_step, "beam": _exact_beam, "rows": _exact_rows,
            "pages": _exact_pages}[case["kind"]](case, seed)


def _sequence(case, leaves, i, a, b, state, groups):
    """Tokens a .. b - 1 of a sequence, one after another, in 64 bits."""
    q, k, v, g, beta = (t[a:b] for t in leaves)
    if case["normalize"]:
        q = q / torch.sqrt(torch.sum(q ** 2, dim=-1, keepdim=True) + EPS)
        k = k / torch.sqrt(torch.sum(k ** 2, dim=-1, keepdim=True) + EPS)
    q = q.repeat_interleave(groups, dim=1) / math.sqrt(case["dim"])
    k = k.repeat_interleave(groups, dim=1)
    out = []
    for t in range(b - a):
        # (I - beta k k^T) e^g S + beta k v^T, written out.
        held = state * g[t].exp()[:, None, None]
        seen = (held * k[t][:, :, None]).sum(dim=1)
        change = beta[t][:, None] * (v[t] - seen)
        state = torch.addcmul(held, k[t][:, :, None], change[:, None, :])
        out.append((state * q[t][:, :, None]).sum(dim=1))
    return torch.stack(out), state


def _exact_sequences(s, first):
    case = s["case"]
    leaves = [s[n].detach().double() for n in ("q", "k", "v", "g", "beta")]
    outs, finals, at = [], [], 0
    for i, n in enumerate(s["new"]):
        out, final = _sequence(case, leaves, i, at, at + n, first[i].double(), case["heads"] // case["key_heads"])
        outs.append(out)
        finals.append(final)
        at += n
    return torch.cat(outs), torch.stack(finals)


def _zeros(case):
    return torch.zeros(case["seqs"], case["heads"], case["dim"], case["value_dim"], device="cuda")


def _exact_scan(case, seed):
    s = _prepare_scan(case, seed)
    out, final = _exact_sequences(s, _zeros(case) if s["initial"] is None else s["initial"])
    return dict(out=out, final=final)


def _exact_step(case, seed):
    s = _prepare_scan(case, seed)
    states = s["states"].double()
    out, final = _exact_sequences(s, s["states"][s["slots"].long()])
    states[s["into"].long()] = final
    return dict(out=out, states=states)


def _exact_train(case, seed):
    s = _prepare_scan(case, seed)
    groups, block = case["heads"] // case["key_heads"], 32
    first = _zeros(case) if s["initial"] is None else s["initial"]
    leaves = [s[n].detach().double() for n in ("q", "k", "v", "g", "beta")]
    grads = [torch.zeros_like(t) for t in leaves]
    outs, finals, firsts, at = [], [], [], 0
    for i, n in enumerate(s["new"]):
        # States at block borders, then the blocks backwards by automatic differentiation.
        state, borders = first[i].detach().double(), []
        with torch.no_grad():
            for a in range(at, at + n, block):
                borders.append((a, state))
                out, state = _sequence(case, leaves, i, a, min(a + block, at + n), state, groups)
                outs.append(out)
        finals.append(state)
        d_state = s["d_final"][i].double()
        for a, before in reversed(borders):
            b = min(a + block, at + n)
            parts = [t[a:b].clone().requires_grad_() for t in leaves]
            before = before.clone().requires_grad_()
            out, after = _sequence(case, parts, i, 0, b - a, before, groups)
            got = torch.autograd.grad([out, after], parts + [before], [s["d_out"][a:b].double(), d_state])
            for whole, part in zip(grads, got):
                whole[a:b] = part
            d_state = got[5]
        firsts.append(d_state)
        at += n
    if s["initial"] is not None:
        grads.append(torch.stack(firsts))
    return dict(out=torch.cat(outs), final=torch.stack(finals), grads=grads)


def _exact_beam(case, seed):
    s = _prepare_beam(case, seed)
    G, W, V = case["groups"], case["beams"], case["vocab"]
    done, scores = s["finished"].tolist(), s["scores"].double().tolist()
    tokens, parents, values = [], [], []
    for i in range(G):
        found = []
        for w in range(W):
            if done[i][w]:
                if scores[i][w] > -math.inf:
                    found.append((-scores[i][w], w * V, w, -1))
                continue
            row = s["logits"][i * W + w].double()
            finite = torch.isfinite(row).nonzero()[:, 0]
            if len(finite) == 0 or scores[i][w] == -math.inf:
                continue
            logp = scores[i][w] + row[finite] - torch.logsumexp(row[finite], dim=0)
            value, order = torch.sort(logp, descending=True, stable=True)
            for x, t in zip(value[:W].tolist(), finite[order[:W]].tolist()):
                found.append((-x, w * V + t, w, t))
        found = sorted(found)[:W]
        rows = [None] * W
        for entry in found:
            if rows[entry[2]] is None:
                rows[entry[2]] = entry
        empty = [w for w in range(W) if rows[w] is None]
        for entry in found:
            if rows[entry[2]] is not entry:
                rows[empty.pop(0)] = entry
        tokens.append([-1 if e is None else e[3] for e in rows])
        parents.append([i * W + (w if e is None else e[2]) for w, e in enumerate(rows)])
        values.append([-math.inf if e is None else -e[0] for e in rows])
    return dict(tokens=_ints(tokens, torch.int64), parents=_ints(parents), scores=_ints(values, torch.float64))


def _exact_rows(case, seed):
    s = _prepare_rows(case, seed)
    return [torch.stack([t[p] for p in s["parents"].tolist()]) for t in s["tensors"]]


def _exact_pages(case, seed):
    s = _prepare_pages(case, seed)
    page = case["page"]
    table, held, cached = s["table"].tolist(), s["held"].tolist(), s["lengths"].tolist()
    free = s["free"].tolist()[:int(s["count"])]
    for r, p in enumerate(s["parents"].tolist()):
        if p == r:
            continue
        while held[r] * page < cached[p]:
            table[r][held[r]] = free.pop()
            held[r] += 1
        cached[r] = cached[p]
        for j in range(-(-cached[p] // page)):
            n = min(page, cached[p] - j * page)
            for cache in (s["k_cache"], s["v_cache"]):
                cache[:, table[r][j], :, :n] = cache[:, table[p][j], :, :n]
    return dict(table=_ints(table), held=_ints(held), lengths=_ints(cached), count=_ints([len(free)]), k=s["k_cache"],
                v=s["v_cache"])
