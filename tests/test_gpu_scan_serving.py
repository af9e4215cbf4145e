"""The recurrent layers' operators, the page pool and beam search together, as a
server uses them, and ``fused_scan`` under a Transformers model, on an MI355X.

A search over a model of one recurrent and one full-attention layer: prompts of
one beam per group, forks to the others, then steps in which every beam takes
its token, the best continuations are chosen from the layers' outputs and the
dead beams' rows follow their parents.  Each row's outputs are checked against
its whole history recomputed in float64 (tests/scan_ref.py's bounds for the
recurrence; attention within one rounding of its weights and of its result), the
choices against the plain search of tests/test_gpu_beam.py on the same
logits."""

from __future__ import annotations

import math

import pytest
import torch

import scan_ref as R
from lightreason_amd.beam import beam_select, fork_rows
from lightreason_amd.paged import PageTable, paged_append, paged_attention
from lightreason_amd.scan import delta_scan, delta_step, fused_scan
from test_gpu_beam import _select

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
VOCAB, HEADS, KEY_HEADS, DIM, GROUPS, BEAMS = 97, 4, 2, 64, 3, 4


class Search:
    """Tables of what each token brings to the layers, and the state of a search."""

    def __init__(self, device):
        self.device = device
        x = R.inputs([VOCAB], KEY_HEADS, HEADS, DIM, DIM, BF, 90, device=device)
        self.table = {n: x[n] for n in ("query", "key", "value", "g", "beta")}
        gen = torch.Generator().manual_seed(91)
        self.attn = [torch.randn(VOCAB, h, DIM, generator=gen).to(BF).to(device) for h in (HEADS, 2, 2)]
        self.head = torch.randn(2 * HEADS * DIM, VOCAB, generator=gen).to(device) * 0.4
        rows = GROUPS * BEAMS
        self.pool = PageTable(rows, 80, 16, max_pages=8, device=device)
        self.caches = self.pool.new_cache(1, 2, DIM)
        self.states = torch.zeros(rows, HEADS, DIM, DIM, device=device)
        self.slots = torch.randperm(rows, generator=gen).to(torch.int32).to(device)   # row r's state
        self.inverse = torch.argsort(self.slots.long())

    def layers(self, tokens, new, count, max_new, fresh=None):
        """A step of `count` packed tokens, new[r] of row r: the layers' outputs."""
        plan = self.pool.plan(new, count)
        x = {n: t[tokens] for n, t in self.table.items()}
        rec = delta_step(**x, starts=plan.starts, states=self.states, slots=self.slots, fresh=fresh, max_new=max_new,
                         out=torch.zeros(count, HEADS, DIM, dtype=BF, device=self.device))
        q, k, v = (t[tokens] for t in self.attn)
        paged_append(k, v, self.caches[0][0], self.caches[1][0], plan.slots)
        att = paged_attention(q, self.caches[0][0], self.caches[1][0], self.pool.table, plan.starts, plan.kv_lengths,
                              max_new=max_new, out=torch.zeros_like(q))
        self.pool.commit(plan)
        return rec, att

    def logits(self, rec, att):
        return torch.cat([rec.flatten(1), att.flatten(1)], dim=1).float() @ self.head

    def choose(self, logits, scores, finished):
        tokens, parents, scores = beam_select(logits, scores, finished=finished)
        # The states lie in slots: a row's parent is its parent's slot.
        flat = parents.view(-1)
        by_slot = self.slots[flat[self.inverse].long()]
        fork_rows(by_slot, [self.states])
        self.pool.fork(flat, *self.caches)
        return tokens, parents, scores

    def check(self, histories, rec, att, rows):
        """Outputs at the last token of each row against the row's history."""
        lengths = [len(histories[r]) for r in rows]
        tokens = torch.tensor([t for r in rows for t in histories[r]], device=self.device)
        x = {n: t[tokens] for n, t in self.table.items()}
        x["starts"] = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=self.device)
        zero = torch.zeros(len(rows), HEADS, DIM, DIM, device=self.device)
        out, final, size = R.rule(x, zero)
        b_out, b_final = R.bounds(x, out, size)
        last = x["starts"][1:].long() - 1
        R.check("recurrent", rec, out[last], b_out[last])
        R.check("states", self.states[self.slots.long()][rows], final, b_final)
        q, k, v = (t[tokens].double() for t in self.attn)
        for i, (a, b) in enumerate(zip(x["starts"].tolist(), x["starts"].tolist()[1:])):
            for h in range(HEADS):
                w = torch.softmax(k[a:b, h // 2] @ q[b - 1, h] * DIM ** -0.5, 0)
                want = w @ v[a:b, h // 2]
                bound = 3 * R.half(BF) * (w @ v[a:b, h // 2].abs())
                assert ((att[i, h].double() - want).abs() <= bound).all()


def _run(device, graph):
    s = Search(device)
    rows = GROUPS * BEAMS
    prompts = [[(7 * g + 3 * i) % VOCAB for i in range(n)] for g, n in enumerate((70, 5, 21))]
    new = torch.zeros(rows, dtype=torch.int32, device=device)
    for g, p in enumerate(prompts):
        new[g * BEAMS] = len(p)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    fresh = torch.ones(rows, dtype=torch.bool, device=device)
    rec, att = s.layers(tokens, new, len(tokens), None, fresh)
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0).to(device) - 1
    first = [g * BEAMS for g in range(GROUPS)]
    histories = {r: list(p) for r, p in zip(first, prompts)}
    s.check(histories, rec[ends], att[ends], first)
    # The first step: the group's one beam has logits, the others follow it.
    logits = torch.zeros(rows, VOCAB, device=device)
    logits[first] = s.logits(rec[ends], att[ends])
    scores = torch.full((GROUPS, BEAMS), -math.inf, device=device)
    scores[:, 0] = 0.0
    finished = torch.zeros(GROUPS, BEAMS, dtype=torch.bool, device=device)
    tokens, parents, scores = s.choose(logits, scores, finished)
    assert torch.equal(tokens.cpu(), _select(logits, torch.where(torch.arange(BEAMS, device=device) == 0, 0.0, -math.inf)
                                             .expand(GROUPS, BEAMS))[0])
    every = list(range(rows))
    held = dict(tokens=tokens.view(-1).clone(), scores=scores.clone())
    ones = torch.ones(rows, dtype=torch.int32, device=device)

    def step():
        rec, att = s.layers(held["tokens"], ones, rows, 1)
        logits = s.logits(rec, att)
        given = held["scores"].clone()
        tokens, parents, scores = s.choose(logits, held["scores"], finished)
        fed = held["tokens"].clone()
        held["tokens"].copy_(tokens.view(-1))
        held["scores"].copy_(scores)
        return rec, att, logits, given, fed, tokens, parents, scores
    for r, p in enumerate(parents.view(-1).tolist()):
        histories[r] = list(prompts[p // BEAMS])
    replay = None
    for i in range(6):
        if graph and i == 2:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=stream):
                results = step()
            torch.cuda.current_stream().wait_stream(stream)
            replay = captured
        before = s.states.clone()
        if replay is not None:
            replay.replay()
            torch.cuda.synchronize()
        else:
            results = step()
        rec, att, logits, given, fed, tokens, parents, scores = results
        want = _select(logits, given)
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(parents.cpu().long(), want[1])
        assert not torch.equal(before, s.states)
        s.pool.check()
        # Histories: the fed token joins a row's, then rows follow their parents.
        for r in every:
            histories[r] = histories[r] + [int(fed[r])]
        moved = parents.view(-1).tolist()
        old = dict(histories)
        for r in every:
            histories[r] = list(old[moved[r]])
        # Outputs were those of the rows before the fork; states and pages are
        # checked behind it, at the parents' outputs.
        flat = torch.tensor(moved, device=device)
        s.check(histories, rec[flat], att[flat], every)
        assert s.pool.lengths.tolist() == [len(histories[r]) for r in every]
    return scores


def test_beam_search_over_states_and_pages(device):
    _run(device, graph=False)


def test_beam_search_step_in_a_graph(device):
    _run(device, graph=True)


def test_a_prompt_in_pieces_is_the_whole_prompt(device):
    """scan of all, or steps of chunks of any length over a pool: the same states
    within the bounds of both."""
    x = R.inputs([200], 2, 4, 128, 64, BF, 77)
    pool = torch.zeros(1, 4, 128, 64, device=device)
    outs, at = [], 0
    for n in (1, 70, 16, 64, 2, 47):
        y = {k: v[at:at + n] for k, v in x.items() if k != "starts"}
        y["starts"] = torch.tensor([0, n], dtype=torch.int32, device=device)
        outs.append(delta_step(**y, states=pool, max_new=n))
        at += n
    zero = torch.zeros_like(pool)
    out, final, size = R.rule(x, zero)
    b_out, b_final = R.bounds(x, out, size)
    R.check("in pieces", torch.cat(outs), out, b_out)
    R.check("in pieces", pool, final, b_final)
    whole, last = delta_scan(**x)
    R.check("whole", whole, out, b_out)
    R.check("whole", last, final, b_final)


# ---- under a Transformers model ----------------------------------------------------

@pytest.fixture(scope="module")
def model(device):
    from transformers import Qwen3_5MoeTextConfig
    from transformers.models.qwen3_5_moe.modeling_qwen3_5_moe import Qwen3_5MoeForCausalLM

    torch.manual_seed(515)
    cfg = Qwen3_5MoeTextConfig(num_hidden_layers=4, num_experts=4, num_experts_per_tok=2, vocab_size=512)
    m = Qwen3_5MoeForCausalLM(cfg).to(device=device, dtype=BF)
    return cfg, m


def test_fused_scan_runs_every_linear_layer(model, device, monkeypatch):
    """Each layer's call gets the rule's result for its own inputs; the stock
    function is back afterwards; gradients reach every weight."""
    from transformers.models.qwen3_5_moe import modeling_qwen3_5_moe as module

    import lightreason_amd.scan as scan

    cfg, m = model
    calls = []

    def spy(*args, **kw):
        result = delta_scan(*args, **kw)
        calls.append(([a.detach() for a in args], kw, [r.detach() for r in result]))
        return result
    monkeypatch.setattr(scan, "delta_scan", spy)
    ids = torch.randint(0, 512, (2, 75), generator=torch.Generator().manual_seed(3)).to(device)
    mixers = [layer.linear_attn for layer in m.model.layers if getattr(layer, "linear_attn", None) is not None]
    stock = module.torch_chunk_gated_delta_rule
    with fused_scan(m):
        loss = m(ids, labels=ids, use_cache=False).loss
    assert module.torch_chunk_gated_delta_rule is stock
    assert len(calls) == len(mixers) == 3
    for args, kw, (out, final) in calls:
        x = dict(zip(("query", "key", "value", "g", "beta", "starts"), args))
        zero = torch.zeros_like(final)
        want, last, size = R.rule(x, zero, normalize=kw["normalize"])
        b_out, b_final = R.bounds(x, want, size, normalize=kw["normalize"])
        R.check("layer", out, want, b_out)
        R.check("layer", final, last, b_final)
    loss.backward()
    for mixer in mixers:
        for name, p in mixer.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    m.zero_grad(set_to_none=True)


@torch.no_grad()
def test_fused_scan_and_fused_delta_fill_one_cache(model, device):
    """A prompt through fused_scan, then cached tokens through fused_delta: the
    recurrent states are fp32, of the module's shape, and the steps use them."""
    from transformers.cache_utils import DynamicCache

    from lightreason_amd.delta import _live, fused_delta

    cfg, m = model
    ids = torch.randint(0, 512, (1, 40), generator=torch.Generator().manual_seed(4)).to(device)
    with fused_scan(m), fused_delta(m):
        cache = DynamicCache(config=cfg)
        m(ids[:, :36], past_key_values=cache, use_cache=True)
        states = [_live(layer.recurrent_states).clone() for layer in cache.layers if hasattr(layer, "recurrent_states")]
        for i in range(36, 40):
            logits = m(ids[:, i:i + 1], past_key_values=cache, use_cache=True).logits
    after = [_live(layer.recurrent_states) for layer in cache.layers if hasattr(layer, "recurrent_states")]
    assert len(states) == 3
    for a, b in zip(states, after):
        assert a.shape == (1, 32, 128, 128) and not torch.equal(a, b) and torch.isfinite(b).all()
    assert torch.isfinite(logits).all()


def _layers_of(rule):
    """A model of one linear-attention layer whose module's rule is ``rule``."""
    import sys
    import types

    module = types.ModuleType("lrmoe_test_layers")
    module.torch_chunk_gated_delta_rule = rule
    Mixer = type("Mixer", (), {"__module__": module.__name__})
    sys.modules[module.__name__] = module
    layer = types.SimpleNamespace(linear_attn=Mixer())
    return module, types.SimpleNamespace(model=types.SimpleNamespace(layers=[layer]))


def _layer_call(D, E, device, dtype=BF, T=70):
    x = R.inputs([2 * T], 3, 3, D, E, dtype, 92)
    return {n: t.unflatten(0, (2, T)) for n, t in x.items() if n != "starts"}


@pytest.mark.parametrize("case", ["width 96", "values of 48", "fp32", "several types", "cu_seqlens", "tangents"])
def test_fused_scan_leaves_other_calls_to_the_stock_rule(device, case):
    given = []

    def stock(query, key, value, g, beta, chunk_size=64, initial_state=None, output_final_state=False,
              use_qk_l2norm_in_kernel=False, **kwargs):
        given.append((query, key, value, g, beta, initial_state, kwargs))
        return "stock", None
    module, model = _layers_of(stock)
    x = _layer_call(96 if case == "width 96" else 64, 48 if case == "values of 48" else 64, device,
                    torch.float32 if case == "fp32" else BF)
    more = {}
    if case == "several types":
        x["value"] = x["value"].half()
    if case == "cu_seqlens":
        more["cu_seqlens"] = torch.tensor([0, 70], device=device)
    with torch.autograd.forward_ad.dual_level(), fused_scan(model):
        if case == "tangents":
            x["value"] = torch.autograd.forward_ad.make_dual(x["value"], torch.ones_like(x["value"]))
        assert module.torch_chunk_gated_delta_rule is not stock
        assert module.torch_chunk_gated_delta_rule(**x, output_final_state=True, **more)[0] == "stock"
    assert module.torch_chunk_gated_delta_rule is stock and len(given) == 1
    assert all(a is b for a, b in zip(given[0], (x[n] for n in ("query", "key", "value", "g", "beta"))))
    assert given[0][5] is None and given[0][6].keys() == more.keys()


def test_fused_scan_copies_rows_that_cannot_be_read_in_place(device):
    def stock(*args, **kw):
        raise AssertionError("not native")
    module, model = _layers_of(stock)
    x = _layer_call(64, 64, device)
    first = R.states(2, 3, 64, 64, 4)
    with fused_scan(model):
        want = module.torch_chunk_gated_delta_rule(**x, initial_state=first, output_final_state=True)
        y = dict(x)
        for n in ("query", "key", "value"):   # off any alignment; strides of 68; heads' elements apart
            t = x[n]
            y[n] = {"query": torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape),
                    "key": torch.cat([t, t[..., :4]], -1)[..., :64],
                    "value": t.transpose(2, 3).contiguous().transpose(2, 3)}[n]
        y["g"], y["beta"] = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x["g"], x["beta"]))
        shifted = torch.cat([first.new_zeros(1), first.flatten()])[1:].view(first.shape)
        got = module.torch_chunk_gated_delta_rule(**y, initial_state=shifted, output_final_state=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@torch.no_grad()
def test_a_prompts_cached_states_are_the_scans(model, device, monkeypatch):
    """What fused_scan leaves in the cache, bit for bit, and what it should be."""
    from transformers.cache_utils import DynamicCache

    import lightreason_amd.scan as scan
    from lightreason_amd.delta import _live

    cfg, m = model
    calls = []

    def spy(*args, **kw):
        calls.append((args, kw, delta_scan(*args, **kw)))
        return calls[-1][2]
    monkeypatch.setattr(scan, "delta_scan", spy)
    ids = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(5)).to(device)
    with fused_scan(m):
        cache = DynamicCache(config=cfg)
        m(ids, past_key_values=cache, use_cache=True)
    states = [_live(layer.recurrent_states) for layer in cache.layers if hasattr(layer, "recurrent_states")]
    assert len(states) == len(calls) == 3
    for state, (args, kw, (out, final)) in zip(states, calls):
        assert torch.equal(state, final)
        x = dict(zip(("query", "key", "value", "g", "beta", "starts"), args))
        want, last, size = R.rule(x, torch.zeros_like(final), normalize=kw["normalize"])
        R.check("state", state, last, R.bounds(x, want, size, normalize=kw["normalize"])[1])
