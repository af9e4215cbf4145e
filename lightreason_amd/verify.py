"""Verify-width integration: speculative-verify blocks of 1-16 positions
through the MoE stack, one captured HIP graph per width, and the width
controller of the reference's DFlash verify loop.

The reference verifies a drafter's block of `count` positions with one
target forward (edge35b/dflash_probe.py:111-120), whose MoE layers take the
grouped path for 2-16 positions (edge35b/block_experts.py:89-139: routes
[T, 8], weights [T, 8], an inverse map per token), and in its adaptive mode
changes the width between blocks (dflash_probe.py:144-148).  Here a block's
MoE stack is one ``moe_chain`` launch per 48 layers (the whole decode layer
-- router, bucketing, experts, combine, shared expert, RMSNorm and residual
-- for every layer), captured once per width so that a verify pass is one
graph replay whatever width the controller picks.
"""

from __future__ import annotations

import torch

from . import _native
from .moe import DECODE_MAX_TOKENS, HIDDEN, TOPK, Workspace, moe_chain


class WidthController:
    """The adaptive verify width of edge35b/dflash_probe.py:144-148: start at
    ``start``; after a block verified at the full width (count == width),
    widen by ``step`` (at most ``limit``, the drafter's block size) when at
    least width - 1 positions were committed, narrow by ``step`` (at least
    ``floor``) when at most width // 2 were, and hold otherwise."""

    def __init__(self, start: int = 8, floor: int = 4, limit: int = 16, step: int = 4):
        if not 1 <= floor <= start <= limit <= DECODE_MAX_TOKENS or step < 1:
            raise ValueError(f"need 1 <= floor <= start <= limit <= {DECODE_MAX_TOKENS} and step >= 1")
        self.width, self.floor, self.limit, self.step = start, floor, limit, step

    def block(self, remaining: int) -> int:
        """Positions of the next block when `remaining` outputs are left
        under the cap (dflash_probe.py:111)."""
        return max(0, min(self.width, remaining))

    def update(self, count: int, committed: int) -> int:
        """Adjust after a block of `count` positions that committed
        `committed` outputs; returns the new width."""
        if count == self.width:
            if committed >= self.width - 1:
                self.width = min(self.width + self.step, self.limit)
            elif committed <= self.width // 2:
                self.width = max(self.floor, self.width - self.step)
        return self.width


class VerifyGraphs:
    """The MoE stack (``layers``: LayerWeights, RMSNorm + residual when they
    carry norm weights) for verify blocks of each width in ``widths``, each
    captured as one HIP graph over static buffers.  ``verify(hidden)`` copies
    a [T, 2048] block in, replays width T's graph and returns its static
    output (valid until the next verify of that width); ``routes(T)`` gives
    that replay's per-layer routes ([L, T, 8] indices and weights).  All
    widths share one workspace and run on the capturing stream in call
    order."""

    def __init__(self, layers, widths=range(1, DECODE_MAX_TOKENS + 1), device=None):
        self.layers = list(layers)
        if not self.layers:
            raise ValueError("VerifyGraphs needs at least one layer")
        self.device = torch.device(device) if device is not None else self.layers[0].router.device
        self.widths = sorted(set(int(w) for w in widths))
        if not self.widths or self.widths[0] < 1 or self.widths[-1] > DECODE_MAX_TOKENS:
            raise ValueError(f"verify widths must lie in 1..{DECODE_MAX_TOKENS}")
        self.workspace = Workspace(self.device, DECODE_MAX_TOKENS)
        self.pool = torch.cuda.graph_pool_handle()
        self.graphs = {}
        L = len(self.layers)
        stream = torch.cuda.Stream(self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(stream):
            for w in self.widths:
                static = dict(
                    hidden=torch.zeros((w, HIDDEN), dtype=torch.bfloat16, device=self.device),
                    out=torch.empty((w, HIDDEN), dtype=torch.bfloat16, device=self.device),
                    indices=torch.empty((L, w, TOPK), dtype=torch.int64, device=self.device),
                    weights=torch.empty((L, w, TOPK), dtype=torch.bfloat16, device=self.device))
                run = self._runner(static)
                run()  # eager once: any one-time setup happens outside the capture
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, pool=self.pool, stream=stream):
                    run()
                self.graphs[w] = (graph, static)
        torch.cuda.current_stream(self.device).wait_stream(stream)

    def _runner(self, static):
        def run():
            moe_chain(static["hidden"], self.layers, out=static["out"], indices=static["indices"],
                      weights=static["weights"], workspace=self.workspace)
        return run

    def verify(self, hidden: torch.Tensor, *, check: bool = True) -> torch.Tensor:
        """Replay the block's width graph.  ``check`` (default) reads the
        workspace status word afterwards (a host synchronisation) and raises
        RuntimeError when a bounded wait of the chain kernel expired (its
        outputs are invalid: another kernel kept workgroups off the GPU);
        ``check=False`` leaves the status to ``status()``."""
        width = hidden.shape[0]
        entry = self.graphs.get(width)
        if entry is None:
            raise ValueError(f"no verify graph of width {width} (captured: {self.widths})")
        if hidden.shape != (width, HIDDEN) or hidden.dtype != torch.bfloat16 or hidden.device != self.device:
            raise ValueError(f"hidden must be bf16 [{width}, {HIDDEN}] on {self.device}")
        graph, static = entry
        static["hidden"].copy_(hidden)
        graph.replay()
        if check:
            self.workspace.check("VerifyGraphs.verify")
        return static["out"]

    def routes(self, width: int):
        _, static = self.graphs[width]
        return static["indices"], static["weights"]

    def status(self) -> int:
        """Status word of the last replay (reads the device)."""
        return self.workspace.status()


# ---- which drafts stand ---------------------------------------------------------

_PROBABILITIES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _rows_of(t: torch.Tensor, name: str, shape, dtype, device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on {device}")
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} needs a contiguous last dimension")
    if len(shape) == 2 and shape[0] > 1 and t.stride(0) < shape[1]:
        raise ValueError(f"{name} needs rows that do not overlap")


def verify_drafts(tokens: torch.Tensor, target: torch.Tensor, starts: torch.Tensor, uniforms: torch.Tensor,
                  samples: torch.Tensor, *, draft: torch.Tensor | None = None, accepted: torch.Tensor | None = None,
                  next_tokens: torch.Tensor | None = None):
    """Which drafted tokens of each verify block stand, and the token after
    them (``lrmoe_verify_drafts``): the rejection rule under which the
    outputs follow the target's distribution whatever the drafter proposes.

    ``tokens`` [rows] int64 are the fed tokens of every block, the last
    committed one first, then its drafts; ``starts`` [blocks + 1] int32 the
    blocks' first rows (a ``paged.PagePlan``'s, or a caller's own); ``target`` [rows, vocab] the
    target's probabilities after each fed token, ``draft`` [rows, vocab] the
    drafter's of the same positions (fp32, bf16 or fp16; None for a drafter
    that proposes its best token).  Draft i stands while uniforms[row i] * q <
    p.  The next token is drawn from max(p - q, 0) at the first draft that
    fails (from p where nothing is left), or from p at the last row: the first
    whose running sum in 64 bits passes ``samples[b]`` of the total.
    ``uniforms`` [rows] and ``samples`` [blocks] are fp32 in [0, 1).

    Returns (accepted [blocks] int32, next_tokens [blocks] int64); a block
    without rows gives (0, -1), a row of probabilities without mass -1.  A
    block of one row is plain sampling.  ``PageTable.commit(plan, accepted)``
    takes the result into the page pool where a step's positions are all of
    decode rows and verify blocks.  Every row of a block after its first counts
    as a draft, so a prompt is a block of its last position alone (a chunk
    whose prompt goes on: of none), and the step is committed with
    ``commit(plan, accepted, starts=starts)``."""
    tensors = (tokens, target, starts, uniforms, samples, draft, accepted, next_tokens)
    key, form = _native.checked(_VERIFIES, tensors)
    if form is None:
        form = _check_verify(*tensors)
        _native.remember(_VERIFIES, key, form)
    blocks, rows, vocab, kind, dev, nbytes, target_stride, draft_stride = form
    if accepted is None:
        accepted = torch.empty(blocks, dtype=torch.int32, device=dev)
    if next_tokens is None:
        next_tokens = torch.empty(blocks, dtype=torch.int64, device=dev)
    if blocks == 0:
        return accepted, next_tokens
    with _native.on_device(dev):
        scratch = _native.workspace(dev, nbytes)
        _native.call("lrmoe_verify_drafts", blocks, rows, vocab, kind, tokens.data_ptr(), target.data_ptr(),
                     target_stride, None if draft is None else draft.data_ptr(), draft_stride, starts.data_ptr(),
                     uniforms.data_ptr(), samples.data_ptr(), accepted.data_ptr(), next_tokens.data_ptr(),
                     scratch.data_ptr(), scratch.numel(), _native.current_stream(dev))
    return accepted, next_tokens


_VERIFIES: dict = {}   # forms (types, shapes, strides) that were checked


def _check_verify(tokens, target, starts, uniforms, samples, draft, accepted, next_tokens):
    """Checks the arguments of verify_drafts; returns what the call derives
    from them."""
    if not isinstance(target, torch.Tensor) or target.dim() != 2 or target.dtype not in _PROBABILITIES:
        raise ValueError("target must be fp32, bf16 or fp16 [rows, vocab]")
    rows, vocab = target.shape
    dev = target.device
    if dev.type != "cuda":
        raise ValueError(f"target must be on a GPU, got {dev}")
    if vocab < 1:
        raise ValueError("the vocabulary is empty")
    _rows_of(target, "target", (rows, vocab), target.dtype, dev)
    if draft is not None:
        _rows_of(draft, "draft", (rows, vocab), target.dtype, dev)
    if not isinstance(starts, torch.Tensor) or starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError("starts must be int32 [blocks + 1]")
    blocks = starts.shape[0] - 1
    if blocks > 65535:
        raise ValueError(f"at most 65535 blocks, got {blocks}")
    for name, t, shape, dtype in (("starts", starts, (blocks + 1,), torch.int32),
                                  ("tokens", tokens, (rows,), torch.int64),
                                  ("uniforms", uniforms, (rows,), torch.float32),
                                  ("samples", samples, (blocks,), torch.float32)):
        _rows_of(t, name, shape, dtype, dev)
    for name, t, dtype in (("accepted", accepted, torch.int32), ("next_tokens", next_tokens, torch.int64)):
        if t is not None:
            _rows_of(t, name, (blocks,), dtype, dev)
    nbytes = 0 if blocks == 0 else int(_native.library().lrmoe_verify_workspace_bytes(blocks, vocab))
    return (blocks, rows, vocab, _PROBABILITIES[target.dtype], dev, nbytes, max(target.stride(0), vocab),
            0 if draft is None else max(draft.stride(0), vocab))
