"""The gradient of scan.delta_scan on an MI355X against automatic
differentiation of the recurrence in float64 and against differences."""

from __future__ import annotations

import math

import pytest
import torch

import scan_ref as R
from lightreason_amd.scan import delta_scan

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAMES = ("query", "key", "value", "g", "beta")


def _reference(x, initial, d_out, d_final, normalize, scale):
    leaves = [x[n].detach().double().requires_grad_() for n in NAMES]
    first = initial.detach().double().requires_grad_()
    q, k, v, g, beta = leaves
    H, K, D = v.shape[1], q.shape[1], q.shape[2]
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + R.EPS) for t in (q, k))
    q, k = q.repeat_interleave(H // K, 1), k.repeat_interleave(H // K, 1)
    scale = D ** -0.5 if scale is None else scale
    starts, total = x["starts"].tolist(), 0.0
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        S = first[s]
        for t in range(a, b):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None, :]
            total = total + (scale * (S * q[t][:, :, None]).sum(1) * d_out[t].double()).sum()
        total = total + (S * d_final[s].double()).sum()
    return torch.autograd.grad(total, leaves + [first])


def _gradients(x, initial, d_out, d_final, **kw):
    leaves = [x[n].detach().requires_grad_() for n in NAMES] + [initial.detach().requires_grad_()]
    out, final = delta_scan(*leaves[:5], x["starts"], initial=leaves[5], **kw)
    return torch.autograd.grad([out, final], leaves, [d_out, d_final]), (out, final)


def _check(x, initial, seed=0, normalize=False, scale=None):
    gen = torch.Generator().manual_seed(seed)
    d_out = torch.randn(x["value"].shape, generator=gen).to(x["value"].dtype).to(initial.device)
    d_final = (torch.randn(initial.shape, generator=gen) * 0.3).to(initial.device)
    got, _ = _gradients(x, initial, d_out, d_final, normalize=normalize, scale=scale)
    want = _reference(x, initial, d_out, d_final, normalize, scale)
    D, n = x["query"].shape[2], max(1, int((x["starts"][1:] - x["starts"][:-1]).max()))
    for name, a, b in zip(NAMES + ("initial",), got, want):
        assert a.dtype == (x[name] if name != "initial" else initial).dtype and a.shape == b.shape
        # Per number: its own rounding.  Over a tensor: factors in two bf16 parts
        # (2^-16 each, three factors in a product of products) and sums of up to
        # dim + 192 terms in fp32 (2^-24 each), over a sequence of n tokens, as a
        # random walk with 8 standard deviations, relative to the largest
        # gradient; the decays' gradient sums 64 rows once more.
        walk = 8 * (3 * 2.0 ** -16 + math.sqrt(D + 192) * 2.0 ** -24) * math.sqrt(max(n, 64) / 16)
        h = 2.0 ** -24 if a.dtype == torch.float32 else R.half(a.dtype)
        R.check(f"d{name}", a, b, h * b.abs() + walk * b.abs().max() + 2.0 ** -24)
    return got


@pytest.mark.parametrize("lengths", [[1], [2, 0, 1], [17], [63, 64, 65], [0, 130], [200, 5]])
@pytest.mark.parametrize("layout", [(2, 4, 128, 128, BF), (3, 3, 64, 64, FP), (1, 3, 64, 96, BF), (2, 2, 128, 32, FP),
                                    (1, 6, 64, 256, BF), (2, 10, 128, 32, FP)])
def test_gradients_of_packed_sequences(device, lengths, layout):
    K, H, D, E, dtype = layout
    print(f"[scan] {lengths} {layout}", flush=True)
    x = R.inputs(lengths, K, H, D, E, dtype, 110 + sum(lengths))
    _check(x, R.states(len(lengths), H, D, E, 5))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lengths", [[1, 3], [70, 9]])
def test_gradients_through_norms_scale_and_fp32_beta(device, dtype, lengths):
    x = R.inputs(lengths, 2, 4, 128, 64, dtype, 3, unit=False, beta_dtype=torch.float32)
    _check(x, R.states(len(lengths), 4, 128, 64, 6), normalize=True, scale=0.5)


def test_against_differences(device):
    """A step along the gradient's inputs moves the outputs' weighted sum by the
    gradient's product with it."""
    x = R.inputs([90, 30], 2, 4, 64, 64, BF, 7, beta_dtype=torch.float32)
    initial = R.states(2, 4, 64, 64, 6)
    gen = torch.Generator().manual_seed(1)
    d_out = torch.randn(x["value"].shape, generator=gen).to(BF).to(device)
    d_final = torch.randn(initial.shape, generator=gen).to(device)
    got, _ = _gradients(x, initial, d_out, d_final)

    def total(y, first):
        out, final, _ = R.rule(y, first)
        return float((out * d_out.double()).sum() + (final * d_final.double()).sum())
    for name, grad in zip(NAMES + ("initial",), got):
        base = initial if name == "initial" else x[name]
        way = torch.randn(base.shape, generator=gen, dtype=torch.float64).to(device)
        eps = 1e-5
        moved = []
        for sign in (1, -1):
            y = {k: v.double() if k != "starts" else v for k, v in x.items()}
            first = initial.double()
            if name == "initial":
                first = first + sign * eps * way
            else:
                y[name] = y[name] + sign * eps * way
            moved.append(total(y, first))
        slope = (moved[0] - moved[1]) / (2 * eps)
        mine = float((grad.double() * way).sum())
        # Each gradient is off by its rounding, of either sign: 6 standard
        # deviations of their sum, and the differences' own error.
        h = 2.0 ** -16 if grad.dtype == torch.float32 else R.half(grad.dtype)
        bound = 6 * h * float((grad.double() * way).norm()) + 1e-5 * abs(slope) + 1e-4
        print(f"[scan] {name}: slope {slope:.5f}, gradient {mine:.5f}, bound {bound:.2e}", flush=True)
        assert abs(slope - mine) <= bound


def test_no_first_state_unused_outputs_and_some_inputs(device):
    x = R.inputs([40, 70], 2, 4, 64, 64, BF, 8)
    leaves = [x[n].detach().requires_grad_() for n in NAMES]
    zero = torch.zeros(2, 4, 64, 64, device=device)
    d_out = torch.randn(x["value"].shape, generator=torch.Generator().manual_seed(3)).to(BF).to(device)
    out, final = delta_scan(*leaves, x["starts"])
    got = torch.autograd.grad(out, leaves, d_out, retain_graph=True)
    want, _ = _gradients(x, zero, d_out, torch.zeros_like(zero))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # Again from the same tape, an expanded gradient, and the states' alone.
    for a, b in zip(torch.autograd.grad(out, leaves, d_out, retain_graph=True), got):
        assert torch.equal(a, b)
    ones = torch.autograd.grad(out.float().sum(), leaves, retain_graph=True)
    same = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
    for a, b in zip(ones, same):
        assert torch.equal(a, b)
    alone = torch.autograd.grad(final.sum(), leaves)
    want, _ = _gradients(x, zero, torch.zeros_like(out), torch.ones_like(zero))
    for a, b in zip(alone, want):
        assert torch.equal(a, b)
    # Only some inputs, and none.
    g = x["g"].detach().requires_grad_()
    out, _ = delta_scan(x["query"], x["key"], x["value"], g, x["beta"], x["starts"])
    only, = torch.autograd.grad(out, g, d_out)
    assert torch.equal(only, got[3])
    with torch.no_grad():
        assert not delta_scan(*leaves, x["starts"])[0].requires_grad


def test_rows_of_no_sequence_have_no_gradient(device):
    x = R.inputs([5, 0, 70], 2, 4, 64, 64, BF, 8, lead=3, tail=40)
    got = _check(x, R.states(3, 4, 64, 64, 2))
    for a in got[:5]:
        assert not a[:3].any() and not a[78:].any() and a[3:78].any()
    none = {n: x[n].detach().requires_grad_() for n in NAMES}
    out, final = delta_scan(*none.values(), x["starts"][:1])
    for a in torch.autograd.grad(out.sum() + final.sum(), list(none.values())):
        assert not a.any()
    initial = R.states(2, 4, 64, 64, 2).requires_grad_()
    empty = [x[n][:0].detach().requires_grad_() for n in NAMES]
    out, final = delta_scan(*empty, torch.zeros(3, dtype=torch.int32, device=device), initial=initial)
    grads = torch.autograd.grad(final.sum(), empty + [initial])
    assert (grads[5] == 1.0).all() and all(t.numel() == 0 for t in grads[:5])


def test_gradient_where_beta_and_decays_are_at_their_ends(device):
    for n in (9, 100):
        x = R.inputs([n], 2, 2, 64, 64, BF, 12)
        x["beta"][n // 3:n // 2] = 0.0
        x["beta"][-1] = 1.0
        x["g"][n // 2:n // 2 + 3] = 0.0
        x["g"][n // 4] = -60.0
        _check(x, R.states(1, 2, 64, 64, 3))


def test_forward_with_and_without_a_tape_are_the_same(device):
    x = R.inputs([150, 33], 2, 4, 128, 64, BF, 14)
    initial = R.states(2, 4, 128, 64, 3)
    plain = delta_scan(**x, initial=initial)
    taped = delta_scan(**x, initial=initial.clone().requires_grad_())
    assert torch.equal(plain[0], taped[0]) and torch.equal(plain[1], taped[1])


def test_more_sequences_than_a_wave_has_lanes(device):
    lengths = [(11 * i) % 71 for i in range(90)]
    x = R.inputs(lengths, 1, 2, 64, 32, BF, 18)
    _check(x, R.states(90, 2, 64, 32, 3))


def test_offsets_past_32_bits(device):
    """One sequence of more than 2^31 values against its halves one after the
    other, which makes the same chunks: the same bits, gradients too."""
    N, K, H, D, half = 2**19 + 100, 2, 32, 128, 2**18
    gen = torch.Generator(device=device).manual_seed(19)
    row = torch.empty(N, (2 * K + H) * D, dtype=BF, device=device).normal_(generator=gen)
    q, k, v = row[:, :K * D].view(N, K, D), row[:, K * D:2 * K * D].view(N, K, D), row[:, 2 * K * D:].view(N, H, D)
    assert v.numel() > 2**31
    g = -torch.rand(N, H, generator=gen, device=device)
    beta = torch.rand(N, H, generator=gen, device=device)
    leaves = [t.requires_grad_() for t in (q.detach(), k.detach(), v.detach(), g, beta)]
    d_out = torch.empty(N, H, D, dtype=BF, device=device).normal_(generator=gen)
    starts = lambda n: torch.tensor([0, n], dtype=torch.int32, device=device)
    out, final = delta_scan(*leaves, starts(N), normalize=True)
    whole = torch.autograd.grad([out, final], leaves, [d_out, torch.ones_like(final)])
    out, final = out.detach(), final.detach()
    torch.cuda.empty_cache()
    for i, t in enumerate(whole):
        assert torch.isfinite(t).all(), NAMES[i]
    first, last = [t[:half] for t in leaves], [t[half:] for t in leaves]
    out1, middle = delta_scan(*first, starts(half), normalize=True)
    out2, end = delta_scan(*last, starts(N - half), initial=middle, normalize=True)
    assert torch.equal(out[:half], out1) and torch.equal(out[half:], out2) and torch.equal(final, end)
    got = torch.autograd.grad([out1, out2, end], first + last, [d_out[:half], d_out[half:], torch.ones_like(end)])
    for i, name in enumerate(NAMES):
        print(f"[scan] d{name}", flush=True)
        assert torch.equal(whole[i][:half], got[i]) and torch.equal(whole[i][half:], got[5 + i]), name
    del out, out1, out2, whole, got
    torch.cuda.empty_cache()


def test_saved_tensors_kept_on_the_host(device):
    """Hooks that hand the inputs back in another layout."""
    x = R.inputs([70, 20], 2, 4, 64, 64, BF, 16)
    leaves = [x[n].detach().requires_grad_() for n in NAMES]
    assert not leaves[0].is_contiguous()
    d_out = torch.randn(x["value"].shape, generator=torch.Generator().manual_seed(3)).to(BF).to(device)
    want = torch.autograd.grad(delta_scan(*leaves, x["starts"])[0], leaves, d_out)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().cpu(), lambda t: t.to(device)):
        out, _ = delta_scan(*leaves, x["starts"])
    for a, b in zip(torch.autograd.grad(out, leaves, d_out), want):
        assert torch.equal(a, b)


def test_a_training_step_in_a_graph(device):
    """Forward and backward captured, replayed on changing inputs between the
    program's own eager steps."""
    x = R.inputs([70, 20], 2, 4, 64, 64, BF, 15)
    leaves = [x[n].detach().clone().requires_grad_() for n in NAMES]
    d_out = torch.randn(x["value"].shape, generator=torch.Generator().manual_seed(3)).to(BF).to(device)

    def step(inputs):
        out, final = delta_scan(*inputs, x["starts"])
        return [out.detach(), final.detach(), *torch.autograd.grad(out, inputs, d_out)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(leaves)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(4):
        y = R.inputs([70, 20], 2, 4, 64, 64, BF, 30 + i)
        with torch.no_grad():
            for leaf, n in zip(leaves, NAMES):
                leaf.copy_(y[n])
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("lead", [1, 3, 8])
def test_gradients_that_begin_at_any_element(device, lead):
    """Results that are joined to something else: their gradients are pieces of a
    longer one, contiguous and off any alignment."""
    x = R.inputs([70, 20], 2, 4, 64, 64, BF, 17)
    leaves = [x[n].detach().requires_grad_() for n in NAMES]
    gen = torch.Generator().manual_seed(4)
    out, final = delta_scan(*leaves, x["starts"])
    weight = torch.randn(lead + out.numel(), generator=gen).to(BF).to(device)
    more = torch.randn(lead + final.numel(), generator=gen).to(device)
    want = torch.autograd.grad([out, final], leaves, [weight[lead:].view_as(out).clone(),
                                                      more[lead:].view_as(final).clone()], retain_graph=True)
    joined = [torch.cat([w.new_zeros(lead), t.flatten()]) for w, t in ((weight, out), (more, final))]
    for a, b in zip(torch.autograd.grad(joined, leaves, [weight, more]), want):
        assert torch.equal(a, b)


def test_saved_tensors_kept_in_pieces_of_a_longer_one(device):
    """Hooks that hand everything back off its alignment, in its own layout or
    another."""
    x = R.inputs([70, 20], 2, 4, 64, 64, BF, 18)
    d_out = torch.randn(x["value"].shape, generator=torch.Generator().manual_seed(3)).to(BF).to(device)
    for leaves in ([x[n].detach().requires_grad_() for n in NAMES],
                   [x[n].detach().clone(memory_format=torch.contiguous_format).requires_grad_() for n in NAMES]):
        want = torch.autograd.grad(delta_scan(*leaves, x["starts"])[0], leaves, d_out)

        def unpack(t):
            return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            out, _ = delta_scan(*leaves, x["starts"])
        for a, b in zip(torch.autograd.grad(out, leaves, d_out), want):
            assert torch.equal(a, b)


def test_forward_mode_derivatives_are_refused(device):
    """A result without a tangent would be a derivative of zero."""
    x = R.inputs([70, 3], 2, 4, 64, 64, BF, 19)
    want = delta_scan(**x)
    initial = R.states(2, 4, 64, 64, 3)
    for name in NAMES + ("initial",):
        with torch.autograd.forward_ad.dual_level():
            base = initial if name == "initial" else x[name]
            dual = torch.autograd.forward_ad.make_dual(base, torch.ones_like(base))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    delta_scan(**{**x, name: dual})
            got = delta_scan(**x)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("n", [9, 140])
def test_steps_without_weight_before_growth(device, n):
    """A beta of 0 is exactly 0 with a tape too: what it leaves out stays out,
    however much a state grows after it, and its value's gradient is 0; its own
    gradient is that of w."""
    x = R.inputs([n], 2, 2, 64, 64, BF, 14)
    at = n // 2
    x["beta"][:at + 1] = 0.0
    x["beta"][-1] = 0.0
    x["value"][at] = 100.0
    x["g"][at + 1] = 30.0
    initial = R.states(1, 2, 64, 64, 1) * 0
    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    out, final = (t.detach() for t in delta_scan(*leaves, x["starts"]))
    assert not out[:at + 1].any()
    if n > 40:   # (shorter ones go token by token without a tape, which rounds elsewhere)
        plain = delta_scan(**x)
        assert torch.equal(out, plain[0]) and torch.equal(final, plain[1])
    # A state of zero, until the first step with a weight.
    after = {k: v[at + 1:] for k, v in x.items() if k != "starts"}
    after["starts"] = torch.tensor([0, n - at - 1], dtype=torch.int32, device=device)
    want, last, size = R.rule(after, initial)
    b_out, b_final = R.bounds(after, want, size)
    R.check("after out", out[at + 1:], want, b_out)
    R.check("after final", final, last, b_final)
    got = _check(x, initial)
    assert not got[2][:at + 1].any() and not got[2][-1].any() and got[2][at + 1:-1].any()


def test_gradients_of_a_padded_batch_and_of_single_tokens(device):
    """Slots of sequences that are empty, or of one token each."""
    for lengths in ([70, 30, 1] + [0] * 500, [1, 2, 1, 0, 1, 3, 1, 1, 65, 1, 64, 1]):
        x = R.inputs(lengths, 2, 2, 64, 64, BF, 86)
        got = _check(x, R.states(len(lengths), 2, 64, 64, 5))
        assert got[5].shape[0] == len(lengths)


def test_a_training_step_leaves_no_memory_behind(device):
    """Scratch of whole sequences goes back to torch, the backward pass's on its own
    thread too."""
    x = R.inputs([3000], 2, 4, 128, 128, BF, 87)
    leaves = [x[n].detach().requires_grad_() for n in NAMES]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(2):
        out, final = delta_scan(*leaves, x["starts"])
        grads = torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])
        del out, final, grads
    assert torch.cuda.memory_allocated() - before < 1 << 20
