"""The gated delta rule of the 35B model's linear-attention layers over packed
sequences: prompts, training, and the steps of a server.

* ``delta_scan(query, key, value, g, beta, starts)`` -- whole sequences, from a
  first state or from zero, to outputs and last states
  (``lrmoe_delta_scan``).
* ``delta_step(..., states, slots=, into=)`` -- a step of prompts, decode
  positions and verify blocks over a pool of states in HBM, as
  ``paged.paged_attention`` serves the full-attention layers of the same step
  (its ``starts`` are a ``paged.PagePlan``'s).
* ``fused_scan(model)`` -- a context manager under which every linear-attention
  layer of a Transformers model runs its prompts and its training through
  ``delta_scan``; inside ``delta.fused_delta`` the steps after a prompt are
  native too.

``delta.delta_rule`` and ``delta.DeltaMixer`` serve one sequence of 1..16 tokens
with the rounding points of the Transformers forward (edge35b/
delta_decode.py:38-55); here a call holds any number of tokens of any number of
sequences, key heads are shared by value heads, and the recurrence runs in fp32
with one rounding, of the outputs.

Nothing reads a device value on the host: every call can be captured into a HIP
graph.  There is no CPU path: the calls raise when liblrmoe.so is missing.
"""

from __future__ import annotations

import ctypes as C
import sys
from contextlib import contextmanager

import torch
from torch.autograd import forward_ad

from . import _native
from .paged import _TYPES, _int, _on, _ptr, _require, _stream, _strided, _strides

HEAD_DIMS = (64, 128)


def _rows(t, name, tokens, dtype, dev):
    """A [tokens, heads, width] tensor whose rows the kernels can read."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, width]")
    _require(t, name, (dtype,), (tokens, *t.shape[1:]), dev, contiguous=False)
    _strided(t, name, 8)


def _per_head(t, name, dtypes, shape, dev):
    _require(t, name, dtypes, shape, dev, contiguous=False)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs a contiguous last dimension")


def _beyond(N, S, K, H, D, E) -> str | None:
    """What of these sizes the kernels cannot do, if anything."""
    if D not in HEAD_DIMS:
        return f"query must have a head width of 64 or 128, got {D}"
    if K < 1:
        return "query has no heads"
    if H < 1 or H % K:
        return f"value must have a multiple of the {K} key heads, got {H}"
    if E % 32 or not 32 <= E <= 256:
        return f"value must have a head width that is a multiple of 32 up to 256, got {E}"
    if S > 65536 or N > 1 << 20 or N * H > 1 << 26 or H > 1024 or S * H * E > 1 << 27:
        return (f"at most 65536 sequences, 2^20 tokens, 1024 heads, tokens * heads of 2^26 and sequences * heads * "
                f"width of 2^27, got {S}, {N}, {H}, {N * H} and {S * H * E}")
    return None


def _check(query, key, value, g, beta, starts, normalize, scale):
    """Checks what every call has; returns the argument structure with sizes
    and strides, and the device."""
    if not isinstance(query, torch.Tensor) or query.dim() != 3:
        raise ValueError("query must be [tokens, key_heads, dim]")
    N, K, D = query.shape
    dtype, dev = query.dtype, query.device
    if dtype not in _TYPES:
        raise ValueError(f"query must be bfloat16 or float16, got {dtype}")
    if (text := _beyond(0, 0, K, K, D, 32)) is not None:
        raise ValueError(text)
    if dev.type != "cuda":
        raise ValueError(f"query must be on a GPU, got {dev}")
    _strided(query, "query", 8)
    _rows(key, "key", N, dtype, dev)
    if tuple(key.shape) != (N, K, D):
        raise ValueError(f"key must have shape {(N, K, D)}, got {tuple(key.shape)}")
    _rows(value, "value", N, dtype, dev)
    H, E = value.shape[1:]
    if (text := _beyond(0, 0, K, H, D, E)) is not None:
        raise ValueError(text)
    _per_head(g, "g", (torch.float32,), (N, H), dev)
    _per_head(beta, "beta", (torch.float32, dtype), (N, H), dev)
    if not isinstance(starts, torch.Tensor) or starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError("starts must be int32 [seqs + 1]")
    S = starts.shape[0] - 1
    _require(starts, "starts", (torch.int32,), (S + 1,), dev)
    if (text := _beyond(N, S, K, H, D, E)) is not None:
        raise ValueError(text)
    a = _native.DeltaScanArgs(seqs=S, tokens=N, max_new=N, heads=H, key_heads=K, dim=D, value_dim=E,
                              fp16=int(dtype == torch.float16), normalize=int(bool(normalize)),
                              beta_fp32=int(beta.dtype == torch.float32), scale=D ** -0.5 if scale is None else scale)
    a.q_token_stride, a.q_head_stride = _strides(query)
    a.k_token_stride, a.k_head_stride = _strides(key)
    a.v_token_stride, a.v_head_stride = _strides(value)
    (a.g_token_stride,), (a.beta_token_stride,) = _strides(g), _strides(beta)
    if N == 0:   # (any strides)
        for name in ("q", "k", "v"):
            setattr(a, f"{name}_token_stride", 0)
            setattr(a, f"{name}_head_stride", 0)
    return a, dev


def _addresses(a, query, key, value, g, beta, starts):
    if a.tokens:
        a.q, a.k, a.v, a.g, a.beta = (t.data_ptr() for t in (query, key, value, g, beta))
    a.starts = starts.data_ptr()


def _scratch(a) -> int:
    return int(_native.library().lrmoe_delta_scan_workspace_bytes(C.addressof(a)))


def _launch(a, dev, nbytes, scratch=None):
    """``scratch``: where the call's memory comes from, the thread's own by
    default.  That stays; whole sequences and their gradient, of any length and the
    latter on a thread of autograd's, take theirs from torch for the call."""
    with _on(dev):
        ws = (scratch or _native.workspace)(dev, nbytes) if nbytes else None
        _native.call("lrmoe_delta_scan", C.addressof(a), _ptr(ws), nbytes, _stream(dev))


def _for_the_call(dev, nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


# ---- whole sequences ------------------------------------------------------------

def delta_scan(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               starts: torch.Tensor, *, initial: torch.Tensor | None = None, normalize: bool = False,
               scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over packed sequences: query, key [tokens,
    key_heads, dim] and value [tokens, heads, value_dim] (bf16 or fp16; dim 64
    or 128, value_dim a multiple of 32 up to 256; value head h reads key head
    h // (heads // key_heads)), g [tokens, heads] fp32 (log decay), beta
    [tokens, heads] (fp32 or the tensors' type), ``starts`` [seqs + 1] int32 on
    the device: sequence s is tokens starts[s] .. starts[s + 1] - 1, its first
    state ``initial[s]`` ([seqs, heads, dim, value_dim] fp32; None: zero).  Per
    token, all in fp32:

        S = exp(g) S;  u = beta (v - S^T k);  S = S + k u^T;  out = scale S^T q

    ``normalize`` divides q and k by sqrt(sum x^2 + 1e-6) first; ``scale``
    defaults to dim ** -0.5.  Returns (out [tokens, heads, value_dim], the last
    states [seqs, heads, dim, value_dim] fp32).  A sequence without tokens
    passes its state on; rows of no sequence are 0.  ``starts`` never decrease
    and lie within [0, tokens] (a batch is padded with their last value): a
    sequence whose own do not counts as empty, and what such a call gives for
    the others is not defined.  What is not finite reaches only later tokens of
    its sequence; the columns that meet it are done again token by token (one of
    a prompt of 8192: 11 ms instead of 0.3).  Longer sequences go in chunks and
    short ones token by token, by their own counts, the call's heads and
    sequences and whether a gradient is wanted: both are fp32, with sums in
    another order, so that a result may round the other way among other
    neighbours.  Tensors may be strided views with a contiguous last dimension
    and strides that are multiples of 8.

    Gradients flow to query, key, value, g, beta and initial, once (no second
    and no forward-mode derivatives: inputs with tangents are refused); they
    take the same bits every time.  For them the call keeps the states before
    every 64 tokens and v - S^T k: 4 (dim + 64) value_dim bytes a head for every
    64 tokens, and once more for every sequence (in all no more than for every
    token).  The gradient of a sequence with values that are not finite is not
    defined.  A captured training step takes its gradients with
    torch.autograd.grad, or from leaves of which no eager graph lives (torch's
    rule for every captured backward pass)."""
    if scale is not None:
        scale = float(scale)
    tensors = (query, key, value, g, beta, starts, initial)
    key_, form = _native.checked(_SCANS, tensors, normalize, scale)
    if form is None:
        a, dev = _check(query, key, value, g, beta, starts, normalize, scale)
        shape = (a.seqs, a.heads, a.dim, a.value_dim)
        if initial is not None:
            _require(initial, "initial", (torch.float32,), shape, dev)
        a.pool, a.clear = a.seqs, 1
        a.out_token_stride, a.out_head_stride = a.heads * a.value_dim, a.value_dim
        form = a, dev, shape
        _native.remember(_SCANS, key_, form)
    if _has_tangents(tensors):
        raise NotImplementedError("delta_scan has no forward-mode derivatives")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _DeltaScan.apply(form, *tensors)
    return _scan(form, tensors)[:2]


def _has_tangents(tensors) -> bool:
    """Whether any tensor is a dual one of torch.autograd.forward_ad, which does not
    show in requires_grad.  (Outside its levels, with a torch that tells, 5 us
    less a call.)"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


_SCANS: dict = {}   # arguments of a form (types, shapes, strides) that was checked, without the addresses


def _scan(form, tensors, taped=False):
    """(out, final, tape): the tape only where it is asked for."""
    template, dev, shape = form
    query, key, value, g, beta, starts, initial = tensors
    a = _native.DeltaScanArgs.from_buffer_copy(template)
    out = torch.empty(value.shape, dtype=value.dtype, device=dev)
    if a.seqs == 0:
        return out.zero_(), torch.empty(shape, dtype=torch.float32, device=dev), None
    final = torch.empty(shape, dtype=torch.float32, device=dev)
    _addresses(a, query, key, value, g, beta, starts)
    a.initial, a.final, a.out = _ptr(initial), final.data_ptr(), out.data_ptr()
    tape = None
    if taped:
        nbytes = int(_native.library().lrmoe_delta_scan_tape_bytes(C.addressof(a)))
        tape = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        a.tape = tape.data_ptr()
    _launch(a, dev, _scratch(a), _for_the_call)
    return out, final, tape


def _aligned(t: torch.Tensor, to: int = 16) -> torch.Tensor:
    """t, or a contiguous copy where it begins off the kernels' alignment (one that
    is contiguous by its strides stays where it is under ``contiguous``)."""
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % to else t


class _DeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, form, *tensors):
        out, final, tape = _scan(form, tensors, taped=True)
        ctx.form = form
        ctx.strides = [t.stride() for t in tensors[:5]]
        ctx.first = tensors[6] is not None
        ctx.save_for_backward(*tensors[:6], *(() if tape is None else (tape,)))
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_final):
        template, dev, shape = ctx.form
        query, key, value, g, beta, starts, *tape = ctx.saved_tensors
        need = ctx.needs_input_grad   # (form, query, key, value, g, beta, starts, initial)
        if not tape:   # no sequences
            zeros = [torch.zeros_like(t) if n else None for t, n in zip((query, key, value, g, beta), need[1:6])]
            first = torch.empty(shape, dtype=torch.float32, device=dev) if ctx.first and need[7] else None
            return None, *zeros, None, first
        a = _native.DeltaScanArgs.from_buffer_copy(template)
        if any(t.stride() != s or t.data_ptr() % 16 and t.dim() == 3
               for t, s in zip((query, key, value, g, beta), ctx.strides)):
            # Hooks on saved tensors (those that keep them on the host) have laid them out anew.
            query, key, value, g, beta = (_aligned(t.contiguous()) for t in (query, key, value, g, beta))
            a.q_token_stride, a.q_head_stride = _strides(query)
            a.k_token_stride, a.k_head_stride = _strides(key)
            a.v_token_stride, a.v_head_stride = _strides(value)
            (a.g_token_stride,), (a.beta_token_stride,) = _strides(g), _strides(beta)
        _addresses(a, query, key, value, g, beta, starts)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (query, key, value, g, beta)]
        first = torch.empty(shape, dtype=torch.float32, device=dev) if ctx.first and need[7] else None
        tape = _aligned(tape[0], 256)
        d = _native.DeltaGradArgs(tape=tape.data_ptr(), d_initial=_ptr(first))
        # Of a gradient that torch hands in, expanded, transposed or cut from a longer
        # one at any element, a plain copy is taken.
        if d_out.stride(-1) != 1 or any(x % 8 or not 0 <= x < 1 << 23 for x in d_out.stride()[:-1]):
            d_out = d_out.contiguous()
        d_out, d_final = _aligned(d_out), _aligned(d_final.contiguous())
        d.d_out_token_stride, d.d_out_head_stride = _strides(d_out)
        d.d_final = d_final.data_ptr()
        if a.tokens:
            d.d_out, d.dq, d.dk, d.dv, d.dg, d.dbeta = (t.data_ptr() for t in (d_out, *grads))
        with _on(dev):
            nbytes = int(_native.library().lrmoe_delta_scan_grad_workspace_bytes(C.addressof(a)))
            ws = _for_the_call(dev, nbytes)
            _native.call("lrmoe_delta_scan_grad", C.addressof(a), C.addressof(d), ws.data_ptr(), ws.numel(),
                         _stream(dev))
        return None, *(t if n else None for t, n in zip(grads, need[1:6])), None, first


# ---- steps over a pool of states ------------------------------------------------

@torch.no_grad()
def delta_step(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               starts: torch.Tensor, states: torch.Tensor, *, slots: torch.Tensor | None = None,
               into: torch.Tensor | None = None, fresh: torch.Tensor | None = None, normalize: bool = False,
               scale: float | None = None, max_new: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``delta_scan`` for a serving step over a pool ``states`` [pool, heads,
    dim, value_dim] fp32: sequence s goes on from the state in slot
    ``slots[s]`` ([seqs] int32; default s), or from zero where ``fresh[s]``
    ([seqs] bool or uint8), and leaves its state in slot ``into[s]`` (default:
    where it was read; another one keeps the old state, for a verify block of
    which only some drafts may stand).  Returns ``out`` [tokens, heads,
    value_dim].

    A sequence whose slot lies outside the pool (-1: a row that rests) is left
    out; rows of no sequence and of those stay as they were in ``out`` (whatever
    memory held where it is not given).  No two sequences of a call write one
    slot, and none writes a slot that another reads.  ``max_new`` -- at least
    every sequence's count of tokens, default ``tokens`` -- only chooses the
    kernel, whose sums may round the other way: give it where the counts are
    known to be small.  ``out`` shares no
    element with query, key and value (refused).  No gradient is recorded."""
    if scale is not None:
        scale = float(scale)
    tensors = (query, key, value, g, beta, starts, states, slots, into, fresh, out)
    key_, form = _native.checked(_STEPS, tensors, normalize, scale, max_new)
    if form is None:
        form = _check_step(*tensors, normalize, scale, max_new)
        _native.remember(_STEPS, key_, form)
    template, dev, nbytes = form
    if out is None:
        out = torch.empty(value.shape, dtype=value.dtype, device=dev)
    if template.seqs == 0:
        return out
    a = _native.DeltaScanArgs.from_buffer_copy(template)
    _addresses(a, query, key, value, g, beta, starts)
    a.initial = a.final = states.data_ptr()
    a.slots, a.into, a.fresh = _ptr(slots), _ptr(slots if into is None else into), _ptr(fresh)
    if a.tokens:
        a.out = out.data_ptr()
    _launch(a, dev, nbytes)
    return out


_STEPS: dict = {}   # as _SCANS


def _check_step(query, key, value, g, beta, starts, states, slots, into, fresh, out, normalize, scale, max_new):
    a, dev = _check(query, key, value, g, beta, starts, normalize, scale)
    if not isinstance(states, torch.Tensor) or states.dim() != 4 or states.shape[0] < 1:
        raise ValueError("states must be [pool, heads, dim, value_dim]")
    _require(states, "states", (torch.float32,), (states.shape[0], a.heads, a.dim, a.value_dim), dev)
    a.pool = states.shape[0]
    if slots is None and a.pool < a.seqs:
        raise ValueError(f"states must have a slot for each of the {a.seqs} sequences, or give slots")
    for name, t in (("slots", slots), ("into", into)):
        if t is not None:
            _require(t, name, (torch.int32,), (a.seqs,), dev)
    if fresh is not None:
        _require(fresh, "fresh", (torch.bool, torch.uint8), (a.seqs,), dev)
    if max_new is not None:
        a.max_new = min(_int(max_new, "max_new", 0, 2**31 - 1), a.tokens)
    if out is not None:
        _require(out, "out", (value.dtype,), tuple(value.shape), dev, contiguous=False)
        _strided(out, "out", 8)
        a.out_token_stride, a.out_head_stride = _strides(out)
    else:
        a.out_token_stride, a.out_head_stride = a.heads * a.value_dim, a.value_dim
    return a, dev, _scratch(a)


# ---- under a Transformers model -------------------------------------------------

def _takes(query, key, value, g, beta, initial) -> bool:
    """Whether ``delta_scan`` does a layer's call, of [batch, tokens, heads, width]."""
    if query.device.type != "cuda" or query.dtype not in _TYPES or any(t.dim() != 4 for t in (query, key, value)):
        return False
    batch, tokens, K, D = query.shape
    H, E = value.shape[2:]
    return (key.dtype == value.dtype == query.dtype and key.shape == query.shape
            and value.shape[:2] == query.shape[:2] and g.shape == beta.shape == value.shape[:3]
            and all(t.device == query.device for t in (key, value, g, beta))
            and (initial is None or initial.device == query.device and initial.shape == (batch, H, D, E))
            and _beyond(batch * tokens, batch, K, H, D, E) is None
            and not _has_tangents((query, key, value, g, beta, initial)))


def _laid_out(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where the kernels cannot read its rows in place."""
    if t.stride(-1) != 1:
        return t.clone(memory_format=torch.contiguous_format)
    if t.dim() == 2:
        return t
    if any(x % 8 or x >= 1 << 23 for x in _strides(t)):
        return t.clone(memory_format=torch.contiguous_format)
    return _aligned(t)


@contextmanager
def fused_scan(model):
    """Run the recurrence of every linear-attention layer's prompt and training
    forward as one ``delta_scan`` call for the duration of the block, gradients
    included: what the layers hand to ``torch_chunk_gated_delta_rule`` of their
    Transformers module, any batch and any length.  (The function is the
    module's, so other models of the class run through it meanwhile.)  What
    ``delta_scan`` does not do runs as before: tensors on the CPU, of another type
    than bf16 and fp16 or of several, widths and sizes beyond its own, calls with
    ``cu_seqlens`` and forward-mode derivatives.  Rows that it could not read in
    place are copied."""
    name = "torch_chunk_gated_delta_rule"
    def native(original):
        def rule(query, key, value, g, beta, chunk_size=64, initial_state=None, output_final_state=False,
                 use_qk_l2norm_in_kernel=False, **kwargs):
            if kwargs.get("cu_seqlens") is not None or not _takes(query, key, value, g, beta, initial_state):
                return original(query, key, value, g=g, beta=beta, chunk_size=chunk_size, initial_state=initial_state,
                                output_final_state=output_final_state, use_qk_l2norm_in_kernel=use_qk_l2norm_in_kernel,
                                **kwargs)
            batch, tokens = query.shape[:2]
            starts = torch.arange(batch + 1, dtype=torch.int32, device=query.device) * tokens
            beta = beta if beta.dtype == query.dtype else beta.float()
            rows = [x.reshape(batch * tokens, *x.shape[2:]) for x in (query, key, value, g.float(), beta)]
            first = None if initial_state is None else _aligned(initial_state.float().contiguous())
            out, final = delta_scan(*map(_laid_out, rows), starts, initial=first, normalize=use_qk_l2norm_in_kernel)
            return out.view(batch, tokens, *out.shape[1:]), final if output_final_state else None

        rule.lrmoe_native = True
        return rule

    mixers = [getattr(layer, "linear_attn", None) for layer in model.model.layers]
    modules = [sys.modules[m] for m in sorted({type(x).__module__ for x in mixers if x is not None})]
    for module in modules:
        if not hasattr(module, name):
            raise ValueError(f"{module.__name__} has no {name}")
    restore = [(module, getattr(module, name)) for module in modules]
    try:
        for module, original in restore:
            setattr(module, name, native(original))
        yield
    finally:
        for module, original in restore:
            setattr(module, name, original)
