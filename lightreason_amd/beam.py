"""Beam search on the GPU: the choice of each group's best continuations and the
rows of states that follow their parents.

* ``beam_select(logits, scores)`` -- the best of all beams' continuations, their
  tokens, parents and scores (``lrmoe_beam_select``), placed so that a beam which
  goes on stays in its row.
* ``fork_rows(parents, tensors)`` -- rows of states (``scan.delta_step``'s pools,
  conv states, whatever a beam carries) become copies of their parents'
  (``lrmoe_fork_rows``); ``paged.PageTable.fork`` does it for the rows of a page
  pool and their caches.

``verify.verify_drafts`` draws from probabilities; this searches.  The reference
decodes greedily and has no counterpart.

Nothing reads a device value on the host: every call can be captured into a HIP
graph.  There is no CPU path: the calls raise when liblrmoe.so is missing.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _native

_LOGITS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@torch.no_grad()
def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, finished: torch.Tensor | None = None):
    """The ``beams`` best continuations of each group: ``logits`` [groups *
    beams, vocab] (fp32, bf16 or fp16; rows may be strided) of every beam's next
    token, ``scores`` [groups, beams] fp32 the beams' scores (sums of log
    probabilities; -inf for a beam that is dead: before the first step all but
    one of a group), ``finished`` [groups, beams] bool or uint8 marks beams that
    have ended: such a beam competes as it is.

    Beam w's continuation by token t scores ``scores[w] + log_softmax(
    logits[w])[t]``.  Exponentials and their sums over 2048 logits are in fp32, what
    joins and compares them in 64 bits: a beam's continuations keep the order of
    their logits, those of two beams closer than the sums' error (about 1e-7; 2^-18 at
    most) may change places.  Equal scores go to the lower beam, a beam's own by its
    logits, then to the lower token.  Logits that are not finite take no part.

    Returns (tokens [groups, beams] int64, parents [groups, beams] int32, scores
    [groups, beams] fp32).  Parents are rows 0 .. groups * beams - 1.  The best
    continuation of a beam takes the beam's own row (its parent is itself),
    further ones the rows of beams that died, in order of their scores, so
    ``fork_rows(parents.view(-1), ...)`` moves as little as can be; rows are not
    sorted by score.  A finished beam has token -1; a row for which nothing is
    left token -1, score -inf and itself as parent."""
    tensors = (logits, scores, finished)
    key, form = _native.checked(_SELECTS, tensors)
    if form is None:
        form = _check_select(*tensors)
        _native.remember(_SELECTS, key, form)
    groups, beams, vocab, kind, stride, nbytes, dev = form
    tokens = torch.empty((groups, beams), dtype=torch.int64, device=dev)
    parents = torch.empty((groups, beams), dtype=torch.int32, device=dev)
    best = torch.empty((groups, beams), dtype=torch.float32, device=dev)
    if groups == 0:
        return tokens, parents, best
    with _native.on_device(dev):
        ws = _native.workspace(dev, nbytes)
        _native.call("lrmoe_beam_select", groups, beams, vocab, kind, logits.data_ptr(), stride, scores.data_ptr(),
                     None if finished is None else finished.data_ptr(), tokens.data_ptr(), parents.data_ptr(),
                     best.data_ptr(), ws.data_ptr(), ws.numel(), _native.current_stream(dev))
    return tokens, parents, best


_SELECTS: dict = {}   # forms (types, shapes, strides) that were checked


def _check_select(logits, scores, finished):
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError("scores must be fp32 [groups, beams]")
    groups, beams = scores.shape
    if not 1 <= beams <= _native.BEAM_MAX or groups * beams > 65535:
        raise ValueError(f"a group has 1..{_native.BEAM_MAX} beams and a call at most 65535, got {groups} x {beams}")
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _LOGITS:
        raise ValueError("logits must be fp32, bf16 or fp16 [groups * beams, vocab]")
    rows, vocab = logits.shape
    dev = logits.device
    if rows != groups * beams:
        raise ValueError(f"logits must have {groups * beams} rows, got {rows}")
    if not 1 <= vocab <= 1 << 30:
        raise ValueError(f"the vocabulary must have 1..2^30 tokens, got {vocab}")
    if dev.type != "cuda":
        raise ValueError(f"logits must be on a GPU, got {dev}")
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits need a contiguous last dimension and rows that do not overlap")
    if scores.device != dev or not scores.is_contiguous():
        raise ValueError(f"scores must be contiguous on {dev}")
    if finished is not None and (not isinstance(finished, torch.Tensor)
                                 or finished.dtype not in (torch.bool, torch.uint8)
                                 or finished.shape != scores.shape or finished.device != dev
                                 or not finished.is_contiguous()):
        raise ValueError(f"finished must be bool or uint8 {tuple(scores.shape)}, contiguous on {dev}")
    nbytes = int(_native.library().lrmoe_beam_workspace_bytes(groups, beams, vocab)) if groups else 0
    stride = logits.stride(0) if rows > 1 else vocab
    return groups, beams, vocab, _LOGITS[logits.dtype], stride, nbytes, dev


@torch.no_grad()
def fork_rows(parents: torch.Tensor, tensors) -> None:
    """In place, row r of every tensor becomes a copy of row ``parents[r]``
    ([rows] int32, ``beam_select``'s, flattened): dimension 0 of each tensor of
    the list counts rows, the others are contiguous within a row (any type;
    states of several layers as one tensor per layer).  A row that is its own
    parent stays; so does one whose parent lies outside 0 .. rows - 1 or is not
    its own parent.  Tensors must not overlap.  A call that is refused has moved
    nothing."""
    if isinstance(tensors, torch.Tensor):
        tensors = (tensors,)
    tensors = tuple(tensors)
    given = (parents, *tensors)
    key, form = _native.checked(_FORKS, given)
    if form is None:
        form = _check_rows(parents, tensors)
        _native.remember(_FORKS, key, form)
    rows, dev, parts = form
    if rows == 0:
        return
    with _native.on_device(dev):
        stream = _native.current_stream(dev)
        for i, table in parts:
            n = len(table) // 3
            table = (C.c_int64 * len(table)).from_buffer_copy(table)
            table[::3] = [t.data_ptr() for t in tensors[i:i + n]]
            _native.call("lrmoe_fork_rows", rows, parents.data_ptr(), n, C.addressof(table), stream)


_FORKS: dict = {}   # as _SELECTS


def _check_rows(parents, tensors):
    if not isinstance(parents, torch.Tensor) or parents.dim() != 1 or parents.dtype != torch.int32:
        raise ValueError("parents must be int32 [rows]")
    rows, dev = parents.shape[0], parents.device
    if dev.type != "cuda":
        raise ValueError(f"parents must be on a GPU, got {dev}")
    if not parents.is_contiguous():
        raise ValueError("parents must be contiguous")
    layout = []
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor) or t.dim() < 1 or t.shape[0] != rows or t.device != dev:
            raise ValueError(f"tensor {i} must have {rows} rows on {dev}")
        if rows and not t[0].is_contiguous():
            raise ValueError(f"tensor {i} must be contiguous within a row")
        nbytes = t.element_size() * (t.numel() // rows if rows else 0)
        stride = t.stride(0) * t.element_size() if rows > 1 else nbytes
        if stride < nbytes:
            raise ValueError(f"tensor {i} has rows that overlap")
        layout.append((stride, nbytes))
    # The parts' first tensors, and the calls' tables but for the addresses.
    return rows, dev, [(i, (C.c_int64 * (3 * len(part)))(*[x for row in part for x in (0, *row)]))
                       for i, part in _fork_parts(rows, layout)]


def _fork_parts(rows, layout):
    """(first, layouts) of the tensors of each library call: up to FORK_TENSORS of
    them, and pieces that a call can count.  Refused is what does not fit one,
    before anything is copied."""
    parts, room = [], 0
    for i, (stride, nbytes) in enumerate(layout):
        pieces = -(-nbytes // _native.FORK_BYTES) * rows
        if pieces >= _native.FORK_PIECES:
            raise ValueError(f"tensor {i} has {pieces} pieces of {_native.FORK_BYTES} bytes, at most "
                             f"{_native.FORK_PIECES - 1} fit a call")
        if not parts or len(parts[-1][1]) == _native.FORK_TENSORS or pieces >= room:
            parts.append((i, []))
            room = _native.FORK_PIECES
        parts[-1][1].append((stride, nbytes))
        room -= pieces
    return parts
