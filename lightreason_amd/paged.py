"""Serving several sequences over a paged key/value cache: what a step of
prompts, decode positions and verify blocks needs around the full-attention
layers of the 35B model, for any head layout of width 64, 128 or 256.

* ``PageTable`` -- a pool of pages shared by rows (sequences), its state on
  the device: ``plan`` turns the rows' new position counts into block table
  entries, slots and offsets (``lrmoe_page_plan``), ``commit`` takes a plan
  into the pool (with the verified counts of a speculative step), ``release``
  returns finished rows' pages, ``fork`` copies rows' pages to other rows
  (``lrmoe_page_fork``).
* ``paged_append`` -- per-head q/k RMSNorm, rotary embedding and the append of
  keys and values into their slots (``lrmoe_paged_append``).
* ``paged_attention`` -- the causal attention of the new positions over the
  cache, sigmoid gate included (``lrmoe_paged_attention``).
* ``paged_layer`` -- a whole full-attention layer of the 35B model on a plan:
  the projections of an ``AttentionDecode`` around the two.

``attention.AttentionDecode.step`` serves one sequence of 1..16 positions on
a contiguous cache; here a step holds any number of positions of up to 4096
sequences.  The reference serves one sequence on the Transformers cache and
has no counterpart.

Nothing reads a device value on the host: every call can be captured into a
HIP graph whose replays follow the counts and lengths on the device.  There
is no CPU path: the calls raise when liblrmoe.so is missing.  They serve only:
no gradient is recorded, whatever their inputs require.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import torch

from . import _native

HEAD_DIMS = (64, 128, 256)
_TYPES = (torch.bfloat16, torch.float16)


_stream = _native.current_stream
_on = _native.on_device


def _require(t: torch.Tensor, name: str, dtypes, shape, device=None, contiguous: bool = True) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on {device or 'a GPU'}, got {t.device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _strided(t: torch.Tensor, name: str, multiple: int) -> None:
    """Last dimension contiguous, the others at a multiple of `multiple`
    elements, as the kernels' vector accesses need."""
    bad = t.shape[-1] > 1 and t.stride(-1) != 1
    bad |= any(n > 1 and s % multiple for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    if bad or t.data_ptr() % (2 * multiple):
        raise ValueError(f"{name} needs a contiguous last dimension, strides that are multiples of {multiple} elements "
                         f"and {2 * multiple}-byte alignment, got strides {tuple(t.stride())}")


def _strides(t: torch.Tensor):
    """Strides of all but the last dimension (of dimensions of one entry: 0)."""
    return [s if n > 1 else 0 for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _int(value, name: str, low: int, high: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or not low <= value <= high:
        raise ValueError(f"{name} must be an int in [{low}, {high}], got {value!r}")
    return value


# ---- the pool -------------------------------------------------------------------

@dataclass
class PagePlan:
    """Outputs of ``PageTable.plan``, all on the device.  Row r's new positions
    are entries ``starts[r] .. starts[r + 1] - 1`` of the step; entries past
    ``starts[rows]`` have slot -1."""

    tokens: int                 # entries of the step
    starts: torch.Tensor        # [rows + 1] int32
    kv_lengths: torch.Tensor    # [rows] int32: cached positions with the new ones
    held: torch.Tensor          # [rows] int32: pages then
    positions: torch.Tensor     # [tokens] int32
    slots: torch.Tensor         # [tokens] int64: page * page_size + offset
    info: torch.Tensor          # [4] int32: status bits, positions, fresh pages, number
    pool: "PageTable | None" = field(default=None, repr=False, compare=False)


class PageTable:
    """``pages`` pages of ``page`` positions shared by ``rows`` sequences of at
    most ``max_pages`` pages each (no more than 2^30 positions).  ``table``
    [rows, max_pages], ``held`` and ``lengths`` [rows], ``free_pages`` [pages]
    and ``state`` [4] (free pages, epoch, status bits, plans made in this
    epoch) are int32 device tensors.

    A step is ``plan`` -> its kernels -> ``commit``.  A plan changes nothing
    that rows hold until it is committed, so it may be made again, but every
    plan writes its fresh pages into ``table``: the last one made is the one
    whose kernels and commit may follow.  An earlier one, and one from before
    another commit or release, is refused at its commit (status)."""

    def __init__(self, rows: int, pages: int, page: int, *, max_pages: int | None = None, device="cuda"):
        self.rows = _int(rows, "rows", 1, _native.PAGE_MAX_ROWS)
        self.pages = _int(pages, "pages", 1, 2**31 - 1)
        self.page = _int(page, "page", 8, 1024)
        if page & (page - 1):
            raise ValueError(f"page must be a power of two, got {page}")
        self.max_pages = _int(pages if max_pages is None else max_pages, "max_pages", 1,
                              _native.PAGE_MAX_POSITIONS // page)
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.full((rows, self.max_pages), -1, **i32)
        self.held = torch.zeros(rows, **i32)
        self.lengths = torch.zeros(rows, **i32)
        self.free_pages = torch.arange(pages - 1, -1, -1, **i32)
        self.state = torch.tensor([pages, 0, 0, 0], **i32)
        self.device = self.table.device

    def new_cache(self, layers: int, kv_heads: int = 2, head_dim: int = 256, dtype=torch.bfloat16):
        """Key and value caches [layers, pages, kv_heads, page, head_dim] for
        this pool (uninitialised)."""
        shape = (layers, self.pages, kv_heads, self.page, head_dim)
        return tuple(torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))

    def new_plan(self, tokens: int) -> PagePlan:
        """Empty outputs of a plan of up to ``tokens`` positions."""
        _int(tokens, "tokens", 0, 1 << 24)
        i32 = dict(dtype=torch.int32, device=self.device)
        return PagePlan(tokens, torch.zeros(self.rows + 1, **i32), torch.zeros(self.rows, **i32),
                        torch.zeros(self.rows, **i32), torch.zeros(tokens, **i32),
                        torch.full((tokens,), -1, dtype=torch.int64, device=self.device), torch.zeros(4, **i32), self)

    def plan(self, new_tokens: torch.Tensor, tokens: int, *, out: PagePlan | None = None) -> PagePlan:
        """The plan of a step in which row r gets ``new_tokens[r]`` positions
        ([rows] int32 on the device; 0 for a row that rests), ``tokens`` >=
        their sum (what the step's tensors are sized for).  Fresh pages come
        from the top of the free stack, rows in order.  A step that does not
        fit is refused as a whole: its ``info[0]`` holds the status bits, its
        starts are all 0, and nothing it feeds writes anything."""
        if out is not None and (out.pool not in (None, self) or out.tokens != tokens
                                or out.starts.shape[0] != self.rows + 1 or out.starts.device != self.device):
            raise ValueError(f"out must be a plan of this pool for {tokens} positions")
        _require(new_tokens, "new_tokens", (torch.int32,), (self.rows,), self.device)
        if out is None:
            out = self.new_plan(tokens)
        out.pool = self
        with _on(self.device):
            _native.call("lrmoe_page_plan", self.rows, self.pages, self.page, self.max_pages, tokens,
                         new_tokens.data_ptr(), self.lengths.data_ptr(), self.held.data_ptr(),
                         self.free_pages.data_ptr(), self.state.data_ptr(), self.table.data_ptr(),
                         out.starts.data_ptr(), out.kv_lengths.data_ptr(), out.held.data_ptr(),
                         out.positions.data_ptr(), out.slots.data_ptr(), out.info.data_ptr(), _stream(self.device))
        return out

    def commit(self, plan: PagePlan, accepted: torch.Tensor | None = None, *,
               starts: torch.Tensor | None = None) -> None:
        """Take a plan into the pool: lengths = plan.kv_lengths, or, with
        ``accepted`` ([rows] int32, from ``verify.verify_drafts``), lengths
        grown by accepted + 1 per row that took part (the last committed token
        and the drafts that stand; the rest of the block is overwritten by the
        next step).  A refused or stale plan changes only the status.

        A step that holds prompts too is verified over blocks of its own,
        ``starts`` [rows + 1] int32 (those that ``verify_drafts`` took): every
        position of a verify block, the last one of a prompt, none of a chunk
        whose prompt goes on.  Give them here as well: only the drafts of a
        block, its rows after the first, can fall; every other position
        stays."""
        if accepted is not None:
            _require(accepted, "accepted", (torch.int32,), (self.rows,), self.device)
        if plan.pool is not self:
            raise ValueError("the plan is not of this pool")
        name, blocks = "lrmoe_page_commit", ()
        if starts is not None:
            if accepted is None:
                raise ValueError("starts come with accepted")
            _require(starts, "starts", (torch.int32,), (self.rows + 1,), self.device)
            name, blocks = "lrmoe_page_commit_drafts", (starts.data_ptr(),)
        with _on(self.device):
            _native.call(name, self.rows, plan.starts.data_ptr(), plan.kv_lengths.data_ptr(), plan.held.data_ptr(),
                         plan.info.data_ptr(), _ptr(accepted), *blocks, self.lengths.data_ptr(), self.held.data_ptr(),
                         self.state.data_ptr(), _stream(self.device))

    def release(self, mask: torch.Tensor) -> None:
        """Return the pages of the rows with mask[r] ([rows] bool or uint8 on
        the device) to the free stack and empty those rows."""
        _require(mask, "mask", (torch.bool, torch.uint8), (self.rows,), self.device)
        with _on(self.device):
            _native.call("lrmoe_page_release", self.rows, self.pages, self.max_pages, mask.data_ptr(),
                         self.table.data_ptr(), self.lengths.data_ptr(), self.held.data_ptr(),
                         self.free_pages.data_ptr(), self.state.data_ptr(), _stream(self.device))

    def fork(self, parents: torch.Tensor, *caches: torch.Tensor) -> None:
        """Rows take over their parents' cached positions: row r with
        ``parents[r]`` ([rows] int32 on the device, as ``beam.beam_select``
        gives them, flattened) other than r gets that row's length, the fresh
        pages it needs and, in each of ``caches`` ([layers, pages, kv_heads,
        page, dim] or one layer [pages, kv_heads, page, dim]; all of the pool's
        key and value caches), copies of its pages.  A parent must be its own
        parent.  A fork that does not fit, or whose parents are not so, changes
        nothing but the status (``check``).  Plans made before are refused at
        their commit."""
        key, form = _native.checked(_FORKS, (parents, *caches), self.rows, self.pages, self.page, self.device)
        if form is None:
            form = self._check_fork(parents, caches)
            _native.remember(_FORKS, key, form)
        table = (C.c_int64 * (8 * len(caches) + 1))()
        for i, (cache, layout) in enumerate(zip(caches, form)):
            table[8 * i] = cache.data_ptr()
            table[8 * i + 1:8 * i + 8] = layout
        with _on(self.device):
            scratch = _native.workspace(self.device, 4 * (self.rows + 1))
            _native.call("lrmoe_page_fork", self.rows, self.pages, self.page, self.max_pages, parents.data_ptr(),
                         self.table.data_ptr(), self.lengths.data_ptr(), self.held.data_ptr(),
                         self.free_pages.data_ptr(), self.state.data_ptr(), len(caches), C.addressof(table),
                         scratch.data_ptr(), _stream(self.device))

    def _check_fork(self, parents, caches):
        _require(parents, "parents", (torch.int32,), (self.rows,), self.device)
        if len(caches) > _native.FORK_CACHES:
            raise ValueError(f"at most {_native.FORK_CACHES} caches, got {len(caches)}")
        form = []
        for i, t in enumerate(caches):
            if not isinstance(t, torch.Tensor) or t.dim() not in (4, 5) or t.device != self.device:
                raise ValueError(f"cache {i} must be [pages, kv_heads, page, dim] or one of those per layer on "
                                 f"{self.device}")
            c = t if t.dim() == 5 else t[None]
            layers, pages, heads, page, dim = c.shape
            if (pages, page) != (self.pages, self.page) or min(layers, heads, dim) < 1:
                raise ValueError(f"cache {i} must have {self.pages} pages of {self.page} positions, got {tuple(t.shape)}")
            size = t.element_size()
            strides = [size * x for x in _strides(c)]
            if (dim > 1 and c.stride(4) != 1) or dim * size % 16 or any(x % 16 or x < 0 for x in strides):
                raise ValueError(f"cache {i} needs a contiguous last dimension and rows and strides of multiples of 16 "
                                 "bytes")
            form.append((layers, heads, dim * size, *strides))
        return form

    def status(self) -> int:
        """Status bits of the commits and releases so far (reads the device)."""
        return int(self.state[2].item())

    def check(self, what: str = "page table") -> None:
        """Raise for the status (reads the device: synchronises)."""
        bits = self.status()
        texts = [text for bit, text in ((_native.PAGE_STATUS_TOKENS, "more new positions than the step has room for"),
                                        (_native.PAGE_STATUS_ROW, "a row longer than its pages, or a bad length"),
                                        (_native.PAGE_STATUS_POOL, "the pool is out of pages"),
                                        (_native.PAGE_STATUS_STALE, "a plan older than the pool, or than another plan, "
                                                                    "was committed"))
                 if bits & bit]
        if texts:
            raise RuntimeError(f"{what}: " + "; ".join(texts))


_FORKS: dict = {}   # forms of fork's arguments (types, shapes, strides) that were checked


# ---- append ---------------------------------------------------------------------

def _caches(k_cache, v_cache, kv_heads, dim, dtype, dev):
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be [pages, kv_heads, page, dim], got {tuple(k_cache.shape)}")
    pages, page = k_cache.shape[0], k_cache.shape[2]
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _require(t, name, (dtype,), (pages, kv_heads, page, dim), dev, contiguous=False)
        _strided(t, name, 8)
    if not 8 <= page <= 1024 or page & (page - 1):
        raise ValueError(f"a page must hold a power of two of 8..1024 positions, got {page}")
    if pages < 1:
        raise ValueError("the cache has no pages")
    return pages, page


def _heads(t, name, tokens, dim, dtype, dev):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, dim]")
    _require(t, name, (dtype,), (tokens, t.shape[1], dim), dev, contiguous=False)
    _strided(t, name, 8)
    return t.shape[1]


def _dims(t, name):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, dim]")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if t.shape[2] not in HEAD_DIMS:
        raise ValueError(f"{name} must have a head width of 64, 128 or 256, got {t.shape[2]}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU, got {t.device}")
    return t.shape[0], t.shape[1], t.shape[2], t.dtype, t.device


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                 *, q: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Append k, v [tokens, kv_heads, dim] to the caches [pages, kv_heads,
    page, dim] at ``slots`` [tokens] int64, and return the queries
    ([tokens, heads, dim] into ``q_out``) when ``q`` is given.

    Keys and queries are RMS-normed per head with ``k_norm`` / ``q_norm``
    [dim] (applied as 1 + w) when given, then their first ``rotary`` elements
    rotated with ``cos``, ``sin`` [rows, rotary] (fp32 or the tensors' type;
    row ``positions[t]``, or row t), all in fp32 and rounded once.  Inputs and
    caches may be strided views with a contiguous last dimension (the 35B
    model's q and gate come interleaved from one projection).  A token whose
    slot lies outside the pool (-1: padding) is left out, its q_out row too
    (whatever memory held where q_out is not given); tokens must not share a
    slot.  ``q_out`` may be a contiguous ``q`` itself;
    else it shares no element with ``q``, ``k`` or ``v`` (refused), nor the
    caches with each other or an input."""
    tensors = (k, v, k_cache, v_cache, slots, q, q_norm, k_norm, cos, sin, positions, q_out)
    eps = float(eps)   # a number, whatever held it: forms are kept by value
    key, form = _native.checked(_APPENDS, tensors, eps)
    if form is None:
        form = _check_append(*tensors, eps)
        _native.remember(_APPENDS, key, form)
    template, dev, q_shape = form
    if q_shape is not None and q_out is None:
        q_out = torch.empty(q_shape, dtype=q.dtype, device=dev)
    if template is None:   # no tokens
        return q_out
    a = _native.PagedAppendArgs.from_buffer_copy(template)
    a.k, a.v, a.k_cache, a.v_cache = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.slots, a.positions = slots.data_ptr(), _ptr(positions)
    a.q, a.q_out, a.q_norm, a.k_norm = _ptr(q), _ptr(q_out), _ptr(q_norm), _ptr(k_norm)
    a.cos, a.sin = _ptr(cos), _ptr(sin)
    with _on(dev):
        _native.call("lrmoe_paged_append", C.addressof(a), _stream(dev))
    return q_out


_APPENDS: dict = {}   # arguments of a form (types, shapes, strides) that was checked, without the addresses


def _check_append(k, v, k_cache, v_cache, slots, q, q_norm, k_norm, cos, sin, positions, q_out, eps):
    """Checks the arguments of paged_append; returns the filled-in structure
    but for the addresses (None without tokens), the device, and q_out's
    shape."""
    N, K, D, dtype, dev = _dims(k, "k")
    _strided(k, "k", 8)
    if _heads(v, "v", N, D, dtype, dev) != K:
        raise ValueError(f"v must have the {K} heads of k")
    pages, page = _caches(k_cache, v_cache, K, D, dtype, dev)
    _require(slots, "slots", (torch.int64,), (N,), dev)
    heads = 0
    if q is not None:
        heads = _heads(q, "q", N, D, dtype, dev)
        if q_out is not None:
            _require(q_out, "q_out", (dtype,), (N, heads, D), dev)
            _strided(q_out, "q_out", 8)
    elif q_out is not None or q_norm is not None:
        raise ValueError("q_out and q_norm come with q")
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None:
            _require(t, name, (dtype,), (D,), dev)
            _strided(t, name, 8)
    if (cos is None) != (sin is None):
        raise ValueError("give both cos and sin or neither")
    rotary = rows = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape[1] % 16 or not 16 <= cos.shape[1] <= D:
            raise ValueError(f"cos must be [rows, rotary], rotary a multiple of 16 up to {D}, got {tuple(cos.shape)}")
        rows, rotary = cos.shape
        _require(cos, "cos", (torch.float32, dtype), (rows, rotary), dev)
        _require(sin, "sin", (cos.dtype,), (rows, rotary), dev)
        if positions is not None:
            _require(positions, "positions", (torch.int32,), (N,), dev)
        elif rows != N:
            raise ValueError(f"without positions cos must have one row per token ({N}), got {rows}")
        if rows == 0 and N > 0:
            raise ValueError("cos has no rows")
    elif positions is not None:
        raise ValueError("positions come with cos and sin")
    q_shape = (N, heads, D) if q is not None else None
    if N == 0:
        return None, dev, q_shape
    a = _native.PagedAppendArgs(tokens=N, heads=heads, kv_heads=K, dim=D, rotary=rotary, pages=pages, page=page,
                                fp16=int(dtype == torch.float16), eps=eps,
                                rope_fp32=int(cos is not None and cos.dtype == torch.float32), rope_rows=rows)
    if q is not None:
        a.q_token_stride, a.q_head_stride = _strides(q)
    a.k_token_stride, a.k_head_stride = _strides(k)
    a.v_token_stride, a.v_head_stride = _strides(v)
    a.k_page_stride, a.k_cache_head_stride, a.k_row_stride = _strides(k_cache)
    a.v_page_stride, a.v_cache_head_stride, a.v_row_stride = _strides(v_cache)
    return a, dev, q_shape


# ---- attention ------------------------------------------------------------------

def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                    starts: torch.Tensor, kv_lengths: torch.Tensor, *, max_new: int | None = None,
                    scale: float | None = None, gate: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a step's positions over a paged cache: q [tokens,
    heads, dim] (bf16 or fp16), caches [pages, kv_heads, page, dim], ``table``
    [seqs, max_pages], ``starts`` [seqs + 1] and ``kv_lengths`` [seqs] int32
    (a ``PageTable``'s table and its plan's outputs, or a caller's own).
    Token t of sequence s, n of them in the step, sees cached positions
    0 .. kv_lengths[s] - n + t; heads share key/value head h // (heads //
    kv_heads); ``scale`` defaults to dim ** -0.5.  With ``gate`` [tokens,
    heads, dim] the result is multiplied by sigmoid(gate).

    Softmax and sums are in fp32.  The weights are rounded to the tensors' type
    before they meet the values, as in the Transformers forward; bf16 ones meet
    them as two bf16 numbers where ``max_new * heads // kv_heads`` is at most 32
    (decode and short verify steps), so that the result is as good as its own
    rounding.  A row that sees nothing is 0;
    what a row does not see cannot change it (infinities and NaN no more than
    its last bits: rows next to some that see such values are summed in
    another order);
    tokens outside starts[0] .. starts[seqs] - 1 stay as they were in ``out``
    (whatever memory held where it is not given), and all do when ``starts`` are not ascending within [0, tokens].  A table
    entry in use outside the pool makes its sequence's rows NaN (those of
    earlier positions may keep their values).  ``out`` may share a buffer with
    ``q`` and ``gate`` but no element with them or between its own rows
    (refused), nor with anything else that is read.

    ``max_new`` -- at least every sequence's n, default ``tokens`` -- only
    chooses the kernel (and the weights' rounding): give it where the counts
    are known to be small."""
    tensors = (q, k_cache, v_cache, table, starts, kv_lengths, gate, out)
    if scale is not None:
        scale = float(scale)
    key, form = _native.checked(_ATTENTIONS, tensors, max_new, scale)
    if form is None:
        form = _check_attention(*tensors, max_new, scale)
        _native.remember(_ATTENTIONS, key, form)
    template, dev, nbytes = form
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if template is None:   # no tokens or no sequences
        return out
    a = _native.PagedAttentionArgs.from_buffer_copy(template)
    a.q, a.k_cache, a.v_cache, a.gate = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _ptr(gate)
    a.table, a.starts, a.kv_lengths = table.data_ptr(), starts.data_ptr(), kv_lengths.data_ptr()
    a.out = out.data_ptr()
    with _on(dev):
        ws = _native.workspace(dev, nbytes)
        _native.call("lrmoe_paged_attention", C.addressof(a), ws.data_ptr(), ws.numel(), _stream(dev))
    return out


_ATTENTIONS: dict = {}   # as _APPENDS


def _check_attention(q, k_cache, v_cache, table, starts, kv_lengths, gate, out, max_new, scale):
    """Checks the arguments of paged_attention; returns the filled-in
    structure but for the addresses (None when there is nothing to do), the
    device, and the bytes of workspace."""
    N, H, D, dtype, dev = _dims(q, "q")
    _strided(q, "q", 8)
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4 or k_cache.shape[1] < 1 or H % k_cache.shape[1]:
        raise ValueError(f"k_cache must be [pages, kv_heads, page, dim] with kv_heads a divisor of {H}")
    K = k_cache.shape[1]
    pages, page = _caches(k_cache, v_cache, K, D, dtype, dev)
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.shape[1] < 1:
        raise ValueError("table must be [seqs, max_pages]")
    S, width = table.shape
    _require(table, "table", (torch.int32,), (S, width), dev)
    _require(starts, "starts", (torch.int32,), (S + 1,), dev)
    _require(kv_lengths, "kv_lengths", (torch.int32,), (S,), dev)
    for name, t in (("gate", gate), ("out", out)):
        if t is not None and _heads(t, name, N, D, dtype, dev) != H:
            raise ValueError(f"{name} must have the {H} heads of q")
    max_new = N if max_new is None else _int(max_new, "max_new", 0, 2**31 - 1)
    if N == 0 or S == 0:
        return None, dev, 0
    a = _native.PagedAttentionArgs(seqs=S, tokens=N, max_new=min(max_new, N), heads=H, kv_heads=K, dim=D, pages=pages,
                                   page=page, max_pages=width, fp16=int(dtype == torch.float16),
                                   scale=D ** -0.5 if scale is None else scale)
    a.q_token_stride, a.q_head_stride = _strides(q)
    if gate is not None:
        a.gate_token_stride, a.gate_head_stride = _strides(gate)
    a.k_page_stride, a.k_head_stride, a.k_row_stride = _strides(k_cache)
    a.v_page_stride, a.v_head_stride, a.v_row_stride = _strides(v_cache)
    if out is not None:
        a.out_token_stride, a.out_head_stride = _strides(out)
    else:
        a.out_token_stride, a.out_head_stride = H * D, D
    nbytes = int(_native.library().lrmoe_paged_attention_workspace_bytes(C.addressof(a)))
    if nbytes == 0:
        raise ValueError("paged_attention: sizes past what one call takes")
    return a, dev, nbytes


@torch.no_grad()
def paged_layer(attn, hidden: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor, pages: PageTable, plan: PagePlan, *, max_new: int | None = None) -> torch.Tensor:
    """One full-attention layer of the 35B model for a step: ``attn`` (an
    ``attention.AttentionDecode``), ``hidden`` [plan.tokens, 2048] bf16 (the
    normed rows), ``cos``, ``sin`` [rows, 64] of every position served,
    ``k_cache``, ``v_cache`` one layer of ``pages.new_cache``.  Returns the
    module's output [plan.tokens, 2048]; rows past the plan's positions are
    0.  The projections are library products; norms, rotation, append,
    attention and gate are two launches and a merge."""
    from .attention import HEAD_DIM, HEADS, HIDDEN, KV_HEADS

    N = plan.tokens
    if plan.pool is not pages:
        raise ValueError("the plan is not of this pool")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 4 or t.shape[0] != pages.pages or t.shape[2] != pages.page:
            raise ValueError(f"{name} must be [{pages.pages}, {KV_HEADS}, {pages.page}, {HEAD_DIM}] as the pool's, got "
                             f"{tuple(t.shape)}")
    _require(hidden, "hidden", (torch.bfloat16,), (N, HIDDEN), attn.device)
    q_gate = torch.nn.functional.linear(hidden, attn.q_proj).view(N, HEADS, 2 * HEAD_DIM)
    k = torch.nn.functional.linear(hidden, attn.k_proj).view(N, KV_HEADS, HEAD_DIM)
    v = torch.nn.functional.linear(hidden, attn.v_proj).view(N, KV_HEADS, HEAD_DIM)
    q = paged_append(k, v, k_cache, v_cache, plan.slots, q=q_gate[:, :, :HEAD_DIM], q_norm=attn.q_norm,
                     k_norm=attn.k_norm, eps=attn.eps, cos=cos, sin=sin, positions=plan.positions)
    out = torch.zeros((N, HEADS, HEAD_DIM), dtype=torch.bfloat16, device=attn.device)
    paged_attention(q, k_cache, v_cache, pages.table, plan.starts, plan.kv_lengths, max_new=max_new,
                    gate=q_gate[:, :, HEAD_DIM:], out=out)
    return torch.nn.functional.linear(out.view(N, HEADS * HEAD_DIM), attn.o_proj)
