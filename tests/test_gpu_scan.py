"""The gated delta rule over packed sequences (scan.delta_scan and delta_step)
on an MI355X against the recurrence in float64 (tests/scan_ref.py, where the
bounds are derived)."""

from __future__ import annotations

import pytest
import torch

import scan_ref as R
from lightreason_amd.scan import delta_scan, delta_step

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _compare(name, x, got, initial, **kw):
    out, final, size = R.rule(x, initial, **kw)
    b_out, b_final = R.bounds(x, out, size, **kw)
    R.check(name + " out", got[0], out, b_out)
    R.check(name + " final", got[1], final, b_final)


@pytest.mark.parametrize("lengths", [[1], [2, 0, 1], [17], [63, 64, 65], [0, 130], [300, 5], [129, 0, 0, 256]])
@pytest.mark.parametrize("layout", [(2, 4, 128, 128, BF), (3, 3, 64, 64, FP), (1, 3, 64, 96, BF), (2, 2, 128, 32, FP),
                                    (1, 6, 64, 256, BF), (2, 10, 128, 32, FP)])
def test_scan_of_packed_sequences(device, lengths, layout):
    K, H, D, E, dtype = layout
    print(f"[scan] {lengths} {layout}", flush=True)
    x = R.inputs(lengths, K, H, D, E, dtype, 11 + sum(lengths))
    initial = R.states(len(lengths), H, D, E, 5)
    got = delta_scan(**x, initial=initial)
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    _compare("given state", x, got, initial)
    _compare("from zero", x, delta_scan(**x), torch.zeros_like(initial))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lengths", [[1, 3], [70, 9]])
def test_normalized_inputs_scale_and_fp32_beta(device, dtype, lengths):
    x = R.inputs(lengths, 2, 4, 128, 64, dtype, 3, unit=False, beta_dtype=torch.float32)
    initial = R.states(len(lengths), 4, 128, 64, 6)
    kw = dict(normalize=True, scale=0.5)
    _compare("normalized", x, delta_scan(**x, initial=initial, **kw), initial, **kw)


@pytest.mark.parametrize("n", [5, 70])
def test_fp16_below_its_normal_range(device, n):
    """Keys that are subnormal in fp16 against large queries and states."""
    x = R.inputs([n], 2, 2, 64, 64, FP, 17)
    x["key"].copy_((x["key"].double() * 2.0 ** -16).to(FP))
    assert 0 < x["key"].abs().max() < torch.finfo(FP).tiny
    initial = R.states(1, 2, 64, 64, 2)
    kw = dict(normalize=False, scale=2.0 ** 12)
    _compare("subnormal", x, delta_scan(**x, initial=initial, **kw), initial, **kw)
    # From zero, the outputs are of the keys alone.
    x["g"].zero_()
    out, _ = delta_scan(**x, scale=2.0 ** 16)
    want, _, _ = R.rule(x, torch.zeros_like(initial), scale=2.0 ** 16)
    R.check("of keys", out, want, R.half(FP) * want.abs() + 2.0 ** -16 * want.abs().max())


def test_rows_of_no_sequence_are_zero(device):
    x = R.inputs([5, 0, 70], 2, 2, 64, 64, BF, 8, lead=3, tail=40)
    out, final = delta_scan(**x)
    assert not out[:3].any() and not out[78:].any() and out[3:78].any()
    _compare("inside", x, (out, final), R.states(3, 2, 64, 64, 1) * 0)
    none = delta_scan(*(x[n] for n in ("query", "key", "value", "g", "beta")), x["starts"][:1])
    assert not none[0].any() and none[1].shape == (0, 2, 64, 64)
    short = {n: x[n][:0] for n in ("query", "key", "value", "g", "beta")}
    initial = R.states(2, 2, 64, 64, 2)
    out, final = delta_scan(**short, starts=torch.zeros(3, dtype=torch.int32, device=device), initial=initial)
    assert out.shape == (0, 2, 64) and torch.equal(final, initial)


def test_starts_out_of_order_make_a_sequence_empty(device):
    x = R.inputs([4, 6, 5], 2, 2, 64, 64, BF, 9)
    initial = R.states(3, 2, 64, 64, 2)
    want = delta_scan(**x, initial=initial)
    for bad in ([0, 4, 2, 2], [0, 4, 4 + 1000, 3], [-1, 4, 10, 9], [-5, -3, 10, 9]):
        x["starts"] = torch.tensor(bad, dtype=torch.int32, device=device)
        out, final = delta_scan(**x, initial=initial)
        assert torch.isfinite(out).all() and torch.isfinite(final).all()
        empty = [s for s in range(3) if not 0 <= bad[s] <= bad[s + 1] <= 15]
        for s in empty:
            assert torch.equal(final[s], initial[s])
        if 0 not in empty:
            assert torch.equal(final[0], want[1][0])


@pytest.mark.parametrize("n", [6, 150])
def test_what_is_not_finite_reaches_later_tokens_only(device, n):
    """Values of every input that are not finite, at one token of one sequence:
    the tokens before it and the other sequences keep their values."""
    for name in ("query", "key", "value", "g", "beta"):
        for value in (float("nan"), float("inf")):
            x = R.inputs([n, 7], 2, 4, 64, 64, BF, 10)
            want = delta_scan(**x)
            y = {k: v.clone() for k, v in x.items()}
            at = n // 2
            y[name][at] = value
            print(f"[scan] {name} {value} at {at}", flush=True)
            out, final = delta_scan(**y)
            R.check("before", out[:at], want[0][:at], 2 * R.half(BF) * want[0][:at].double().abs() + 2.0 ** -14)
            assert torch.equal(out[n:], want[0][n:]) and torch.equal(final[1], want[1][1])
            if value != value:
                assert torch.isnan(out[at].float()).any()
            if name == "query":
                R.check("last state", final, want[1], torch.tensor(2.0 ** -14))


def test_decays_of_zero_and_steps_without_weight(device):
    """g = -inf forgets, g = 0 keeps, beta = 0 only reads."""
    for n in (9, 140):
        x = R.inputs([n], 2, 2, 64, 64, BF, 12)
        initial = R.states(1, 2, 64, 64, 3)
        x["g"][n // 3] = float("-inf")
        x["g"][n // 2:] = 0.0
        x["beta"][n // 2 + 1] = 0.0
        x["beta"][-1] = 1.0
        _compare("edges", x, delta_scan(**x, initial=initial), initial)
        x["beta"].zero_()
        x["g"].zero_()
        _compare("reads only", x, delta_scan(**x, initial=initial), initial)


def test_a_step_without_weight_before_growth(device):
    """What beta = 0 leaves out stays out, however much a state grows after it."""
    for n in (9, 140):
        x = R.inputs([n], 2, 2, 64, 64, BF, 14)
        at = n // 2
        x["beta"][:at + 1] = 0.0
        x["beta"][-1] = 0.0
        x["value"][at] = 100.0
        x["g"][at + 1] = 30.0
        out, final = delta_scan(**x)
        # A state of zero, until the first step with a weight.
        assert not out[:at + 1].any()
        want = {k: v[at + 1:] for k, v in x.items() if k != "starts"}
        want["starts"] = torch.tensor([0, n - at - 1], dtype=torch.int32, device=device)
        _compare("after", want, (out[at + 1:], final), R.states(1, 2, 64, 64, 1) * 0)


def test_repeated_keys(device):
    """The same key again and again: nothing cancels in the chunk's inverse."""
    x = R.inputs([200], 1, 2, 128, 64, BF, 13)
    x["key"][:] = x["key"][:1].clone()
    x["beta"].fill_(1.0)
    x["g"].fill_(-1e-3)
    _compare("repeated", x, delta_scan(**x), R.states(1, 2, 128, 64, 1) * 0)


# ---- steps over a pool ------------------------------------------------------------

@pytest.mark.parametrize("lengths,max_new", [([1], 1), ([1] * 7, 1), ([4, 1, 0, 16, 2], 16), ([200, 1, 1, 3], None)])
@pytest.mark.parametrize("layout", [(2, 4, 128, 128, BF), (2, 2, 64, 64, FP)])
def test_step_over_slots(device, lengths, max_new, layout):
    K, H, D, E, dtype = layout
    S = len(lengths)
    x = R.inputs(lengths, K, H, D, E, dtype, 21)
    pool = R.states(2 * S + 1, H, D, E, 4)
    order = torch.randperm(2 * S + 1, generator=torch.Generator().manual_seed(S)).to(torch.int32).to(device)
    slots, into = order[:S].contiguous(), order[S:2 * S].contiguous()
    fresh = torch.zeros(S, dtype=torch.bool, device=device)
    fresh[S // 2] = True
    first = pool[slots.long()].clone()
    first[fresh] = 0.0
    # In place.
    held = pool.clone()
    out = delta_step(**x, states=held, slots=slots, fresh=fresh, max_new=max_new)
    _compare("in place", x, (out, held[slots.long()]), first)
    rest = [i for i in range(2 * S + 1) if i not in slots.tolist()]
    assert torch.equal(held[rest], pool[rest])
    # Into other slots: the old states stay.
    held = pool.clone()
    given = torch.full_like(out, 7.0)
    got = delta_step(**x, states=held, slots=slots, into=into, fresh=fresh, max_new=max_new, out=given)
    assert got is given and torch.equal(given, out)
    _compare("into", x, (given, held[into.long()]), first)
    rest = [i for i in range(2 * S + 1) if i not in into.tolist()]
    assert torch.equal(held[rest], pool[rest])
    # Without slots: sequence s has slot s.
    held = pool.clone()
    out = delta_step(**x, states=held, max_new=max_new)
    _compare("in order", x, (out, held[:S]), pool[:S])


@pytest.mark.parametrize("n", [3, 100])
def test_resting_rows_and_rows_of_no_sequence_stay(device, n):
    x = R.inputs([n, n, 2], 2, 2, 64, 64, BF, 31, lead=2, tail=9)
    pool = R.states(3, 2, 64, 64, 4)
    for bad in (-1, 3, 2**31 - 1, -2**31):
        slots = torch.tensor([1, bad, 0], dtype=torch.int32, device=device)
        held, out = pool.clone(), torch.full((2 * n + 13, 2, 64), 7.0, dtype=BF, device=device)
        delta_step(**x, states=held, slots=slots, out=out)
        assert (out[:2] == 7.0).all() and (out[-9:] == 7.0).all() and (out[2 + n:2 + 2 * n] == 7.0).all()
        assert torch.equal(held[2], pool[2]) and not torch.equal(held[:2], pool[:2])
        assert not (out[2:2 + n] == 7.0).all() and not (out[2 + 2 * n:4 + 2 * n] == 7.0).all()


@pytest.mark.parametrize("n", [2, 90])
def test_strided_outputs_and_views(device, n):
    x = R.inputs([n, 1], 2, 4, 64, 64, BF, 33)
    pool = R.states(2, 4, 64, 64, 4)
    want_pool = pool.clone()
    want = delta_step(**x, states=want_pool)
    wide = torch.full((n + 1, 4, 128), 7.0, dtype=BF, device=device)
    heads_first = {k: v.transpose(0, 1).contiguous().transpose(0, 1) if k in ("query", "key", "value") else v
                   for k, v in x.items()}
    wider_g = torch.zeros(n + 1, 9, device=device)
    wider_g[:, 2:6] = x["g"]
    heads_first["g"] = wider_g[:, 2:6]
    got = delta_step(**heads_first, states=pool, out=wide[:, :, 64:])
    assert torch.equal(got, want) and torch.equal(pool, want_pool)
    assert (wide[:, :, :64] == 7.0).all()


@pytest.mark.parametrize("n", [1, 80])
def test_captured_steps_follow_the_slots(device, n):
    """Graphs of in-place steps, replayed with the program's own work between."""
    x = R.inputs([n, 0, n], 2, 2, 64, 64, BF, 41)
    pool = R.states(4, 2, 64, 64, 4)
    slots = torch.tensor([3, 0, 1], dtype=torch.int32, device=device)
    eager = pool.clone()
    out = torch.zeros(2 * n, 2, 64, dtype=BF, device=device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        delta_step(**x, states=pool.clone(), slots=slots, out=out.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            delta_step(**x, states=pool, slots=slots, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(4):
        if i == 2:
            slots.copy_(torch.tensor([0, 1, 2], dtype=torch.int32))
        want = delta_step(**x, states=eager, slots=slots)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, eager)


def test_two_streams(device):
    """Calls on two streams at once have scratch of their own."""
    cases = [(R.inputs([300, 40], 2, 4, 128, 64, BF, 50 + i), R.states(2, 4, 128, 64, i)) for i in range(2)]
    want = [delta_scan(**x, initial=s) for x, s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, (x, s) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = delta_scan(**x, initial=s)
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])


def test_slots_past_32_bits(device):
    """A pool of more than 2^31 elements."""
    H, D, E = 32, 128, 128
    pool = torch.empty(4100, H, D, E, device=device)
    assert pool[4099].storage_offset() > 2**31
    for lengths in ([1, 2], [70, 1]):
        x = R.inputs(lengths, 16, H, D, E, BF, 60)
        pool[4098:] = R.states(2, H, D, E, 9)
        first = pool[4098:].clone()
        slots = torch.tensor([4099, 4098], dtype=torch.int32, device=device)
        out = delta_step(**x, states=pool, slots=slots)
        _compare("far slots", x, (out, pool[slots.long()]), first.flip(0))
    del pool
    torch.cuda.empty_cache()


def test_many_short_sequences(device):
    """More sequences than a wave has lanes, twice over."""
    lengths = [(7 * i) % 4 for i in range(4500)]
    x = R.inputs(lengths, 1, 1, 64, 32, BF, 70)
    pool = R.states(4500, 1, 64, 32, 9)
    first = pool.clone()
    out = delta_step(**x, states=pool, max_new=None)
    few = [0, 1, 63, 64, 65, 1000, 4095, 4096, 4499]
    starts = x["starts"].tolist()
    for s in few:
        y = {k: v[starts[s]:starts[s + 1]] for k, v in x.items() if k != "starts"}
        y["starts"] = torch.tensor([0, lengths[s]], dtype=torch.int32, device=device)
        _compare(f"sequence {s}", y, (out[starts[s]:starts[s + 1]], pool[s:s + 1]), first[s:s + 1])


def test_a_step_of_long_and_short_sequences(device):
    """Prompts among single tokens: either form's sequences in one call, in place."""
    lengths = [1, 1, 500, 1, 24, 25, 40, 41, 0, 1, 64, 3, 130]
    x = R.inputs(lengths, 2, 8, 128, 128, BF, 80)
    pool = R.states(len(lengths), 8, 128, 128, 9)
    first = pool.clone()
    out = delta_step(**x, states=pool)
    _compare("mixed", x, (out, pool), first)


def test_a_long_sequence_of_slow_decays(device):
    """4000 tokens whose state hardly fades."""
    x = R.inputs([4000], 1, 2, 64, 32, BF, 81, decay=(1e-6, 1e-4))
    _compare("slow", x, delta_scan(**x), R.states(1, 2, 64, 32, 1) * 0)


def test_growing_states(device):
    """Positive log decays within fp32's range, token by token and in chunks."""
    for n in (10, 80):
        x = R.inputs([n], 1, 2, 64, 32, BF, 82)
        x["g"].fill_(0.05)
        initial = R.states(1, 2, 64, 32, 1)
        out, final, size = R.rule(x, initial)
        b_out, b_final = R.bounds(x, out, size)
        # An error grows as the state does, e^(0.05 n) at most.
        grow = 2.718281828 ** (0.05 * n)
        got = delta_scan(**x, initial=initial)
        R.check("growing out", got[0], out, b_out * grow)
        R.check("growing final", got[1], final, b_final * grow)


def test_heads_and_tokens_in_any_order_and_repeated_rows(device):
    """Expanded rows (stride 0) and heads that are stored first."""
    x = R.inputs([90], 2, 4, 64, 64, BF, 83)
    y = dict(x)
    y["query"] = x["query"][:1].expand(90, 2, 64)
    y["value"] = x["value"].transpose(0, 1).contiguous().transpose(0, 1)
    y["beta"] = x["beta"][:1].expand(90, 4)
    _compare("expanded", y, delta_scan(**y), R.states(1, 4, 64, 64, 1) * 0)


def test_counts_around_the_edges_of_chunks_and_forms(device):
    """Slots of one sequence right behind another's, empty ones and short ones between,
    in few heads (from 25 tokens on in chunks) and in many (from 41)."""
    lengths = [25, 0, 65, 1, 26, 24, 64, 0, 0, 41, 40, 129, 42, 63, 3, 32, 33, 128]
    for H in (2, 64):
        x = R.inputs(lengths, 2, H, 64, 32, BF, 84, lead=5)
        initial = R.states(len(lengths), H, 64, 32, 5)
        _compare(f"{H} heads", x, delta_scan(**x, initial=initial), initial)


def test_a_batch_padded_with_empty_sequences(device):
    x = R.inputs([70, 30, 1] + [0] * 3000, 2, 2, 64, 64, BF, 85)
    initial = R.states(3003, 2, 64, 64, 5)
    got = delta_scan(**x, initial=initial)
    _compare("padded", x, got, initial)
    assert torch.equal(got[1][3:], initial[3:])


@pytest.mark.parametrize("n", [6, 70])
def test_values_next_to_the_end_of_fp32(device, n):
    """u above bf16's largest number, and u e^G above fp32's with a key that is
    small: outputs and states are finite."""
    x = R.inputs([n], 2, 2, 64, 32, BF, 88, beta_dtype=torch.float32)
    for t in ("query", "key", "value", "g"):
        x[t].zero_()
    x["beta"].fill_(1.0)
    x["key"][n - 3, :, 0], x["query"][n - 2:, :, 0] = 1.0, 1.0
    x["value"][n - 3] = torch.finfo(BF).max
    x["beta"][n - 3] = 1.0025
    initial = R.states(1, 2, 64, 32, 1) * 0
    u = torch.finfo(BF).max * float(x["beta"][n - 3, 0])
    assert 3.3962e38 < u < torch.finfo(torch.float32).max
    got = delta_scan(**x, initial=initial, scale=2.0 ** -20)
    want, last, _ = R.rule(x, initial, scale=2.0 ** -20)
    R.check("large u out", got[0], want, R.half(BF) * want.abs() + 4 * 2.0 ** -24 * want.abs())
    R.check("large u state", got[1], last, 4 * 2.0 ** -24 * last.abs())
    # A key of 2^-20, then growth by e^5.
    x["key"].mul_(2.0 ** -20)
    x["value"].mul_(2.0 ** -1)
    x["g"][n - 1] = 5.0
    assert u / 2 * 2.718 ** 5 > torch.finfo(torch.float32).max
    got = delta_scan(**x, initial=initial)
    want, last, _ = R.rule(x, initial)
    # (The factor e^5: the exponential's own step and its argument's, 5 2^-24, as a factor.)
    R.check("grown out", got[0], want, R.half(BF) * want.abs() + 16 * 2.0 ** -24 * want.abs())
    R.check("grown state", got[1], last, 16 * 2.0 ** -24 * last.abs())
