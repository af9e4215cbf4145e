"""ctypes binding of liblrmoe.so (include/lrmoe.h).

The library is the only compute path: when it is missing or the device is
not gfx950 every entry point raises; there is no fallback.
"""

from __future__ import annotations

import ctypes as C
import threading
from contextlib import nullcontext
from functools import lru_cache
from operator import attrgetter, methodcaller
from pathlib import Path

import torch

LIBRARY = Path(__file__).resolve().parent / "liblrmoe.so"

LRMOE_OK = 0
LRMOE_E_ARG = -1
LRMOE_E_WORKSPACE = -2
LRMOE_E_DEVICE = -3
WS_STATUS_OFFSET = 4
STATUS_BAD_EXPERT = 1
STATUS_REPEATED_EXPERT = 2
STATUS_CODEC_ROW = 4
STATUS_TIMEOUT = 8       # a bounded cross-workgroup wait of the decode kernel expired: outputs invalid

STATIC_MAX_TOKENS = 16  # tokens per lrmoe_moe_layer_static call
CHAIN_PTRS = 8           # int64 addresses per layer in a chain's layer table
CHAIN_MAX_LAYERS = 48    # layers per lrmoe_moe_chain call
CODEC_TABLE_COLUMNS = 10  # int64 per expert in a decode codec table (4 addresses, 48 flag bytes)

_P = C.c_void_p
_I = C.c_int
_SIGNATURES = {
    "lrmoe_version": ([], C.c_char_p),
    "lrmoe_error_string": ([_I], C.c_char_p),
    "lrmoe_device_check": ([], _I),
    "lrmoe_workspace_bytes": ([_I], C.c_size_t),
    "lrmoe_route_topk": ([_P, _I, _P, _P, _P, C.c_float, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_bucket": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_moe_experts": ([_P, _I, _P, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_moe_layer": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_gather_tiles": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "lrmoe_moe_layer_static": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _P, _P], _I),
    "lrmoe_moe_chain": ([_P, _I, _I, _P, C.c_float, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_codec_pack": ([_P, C.c_int64, _I, _P, _P, _P, _P], _I),
    "lrmoe_codec_unpack": ([_P, _P, C.c_int64, _I, _P, _P], _I),
    "lrmoe_gather": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "lrmoe_matvec": ([_P, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "lrmoe_ordered_sum": ([_P, _P, _P, _P, _P, _I, _P], _I),
    "lrmoe_gate_silu": ([_P, _P, _P, _I, _I, _P], _I),
    "lrmoe_project": ([_P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
    "lrmoe_swiglu_rows": ([_P, _P, _I, _P], _I),
    "lrmoe_add_rmsnorm": ([_P, _P, _I, _P, C.c_float, _P, _P, _P], _I),
    "lrmoe_block_combine": ([_P, _P, _P, _P, _P, _I, _I, _P], _I),
    "lrmoe_fill_normal_bf16": ([_P, C.c_int64, C.c_uint64, C.c_uint64, C.c_double, C.c_int64, _P], _I),
    "lrmoe_timing_enable": ([_I, _I], _I),
    "lrmoe_timing_collect": ([_I, C.POINTER(C.c_double), C.POINTER(_I)], _I),
    "lrmoe_read_bandwidth": ([_P, C.c_int64, _I, _P, C.POINTER(C.c_double), _P], _I),
    "lrmoe_delta_workspace_bytes": ([_I], C.c_size_t),
    "lrmoe_delta_rule": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P], _I),
    "lrmoe_delta_mixer": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _I, _P, _P, _P, _P,
                           C.c_size_t, _P], _I),
    "lrmoe_delta_mixer_step": ([_P, _I, _P, C.c_float, _P, _P, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _I,
                                _P, _P, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_attn_workspace_bytes": ([_I], C.c_size_t),
    "lrmoe_attn_decode": ([_P, _I, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _P, _I, _I, _P, _P, C.c_size_t,
                           _P], _I),
    "lrmoe_attn_decode_at": ([_P, _I, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _P, _I, _P, _P, _P,
                              C.c_size_t, _P], _I),
    "lrmoe_attn_decode_step": ([_P, _I, _P, C.c_float, _P, _P, _P, _P, _P, _P, C.c_float, _P, _P, _P, _P, _I, _I,
                                _P, _P, _P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_page_plan": ([_I] * 5 + [_P] * 13, _I),
    "lrmoe_page_commit": ([_I] + [_P] * 9, _I),
    "lrmoe_page_commit_drafts": ([_I] + [_P] * 10, _I),
    "lrmoe_page_release": ([_I] * 3 + [_P] * 7, _I),
    "lrmoe_paged_append": ([_P, _P], _I),
    "lrmoe_paged_attention_workspace_bytes": ([_P], C.c_size_t),
    "lrmoe_paged_attention": ([_P, _P, C.c_size_t, _P], _I),
    "lrmoe_page_fork": ([_I] * 4 + [_P] * 6 + [_I] + [_P] * 3, _I),
    "lrmoe_delta_scan_workspace_bytes": ([_P], C.c_size_t),
    "lrmoe_delta_scan": ([_P, _P, C.c_size_t, _P], _I),
    "lrmoe_delta_scan_tape_bytes": ([_P], C.c_size_t),
    "lrmoe_delta_scan_grad_workspace_bytes": ([_P], C.c_size_t),
    "lrmoe_delta_scan_grad": ([_P, _P, _P, C.c_size_t, _P], _I),
    "lrmoe_beam_workspace_bytes": ([_I] * 3, C.c_size_t),
    "lrmoe_beam_select": ([_I] * 4 + [_P, C.c_int64] + [_P] * 6 + [C.c_size_t, _P], _I),
    "lrmoe_fork_rows": ([_I, _P, _I, _P, _P], _I),
    "lrmoe_verify_workspace_bytes": ([_I, _I], C.c_size_t),
    "lrmoe_verify_drafts": ([_I] * 4 + [_P, _P, C.c_int64, _P, C.c_int64] + [_P] * 6 + [C.c_size_t, _P], _I),
}


def _fields(kinds: str):
    """ctypes fields from "type: name name; ..." in the header's order."""
    types = {"i": C.c_int32, "l": C.c_int64, "f": C.c_float, "p": C.c_void_p}
    groups = [part.split(":") for part in kinds.split(";")]
    return [(name, types[kind.strip()]) for kind, names in groups for name in names.split()]


class PagedAppendArgs(C.Structure):
    """lrmoe_paged_append_args."""

    _fields_ = _fields(
        "i: tokens heads kv_heads dim rotary pages page fp16; p: q k v;"
        "l: q_token_stride q_head_stride k_token_stride k_head_stride v_token_stride v_head_stride;"
        "p: q_norm k_norm; f: eps; i: rope_fp32; p: cos sin positions; i: rope_rows pad;"
        "p: slots q_out k_cache v_cache;"
        "l: k_page_stride k_cache_head_stride k_row_stride v_page_stride v_cache_head_stride v_row_stride")


class PagedAttentionArgs(C.Structure):
    """lrmoe_paged_attention_args."""

    _fields_ = _fields(
        "i: seqs tokens max_new heads kv_heads dim pages page max_pages fp16; f: scale; i: pad; p: q gate;"
        "l: q_token_stride q_head_stride gate_token_stride gate_head_stride; p: k_cache v_cache;"
        "l: k_page_stride k_head_stride k_row_stride v_page_stride v_head_stride v_row_stride;"
        "p: table starts kv_lengths out; l: out_token_stride out_head_stride")


class DeltaScanArgs(C.Structure):
    """lrmoe_delta_scan_args."""

    _fields_ = _fields(
        "i: seqs tokens max_new heads key_heads dim value_dim fp16 normalize beta_fp32 clear pool; f: scale; i: pad;"
        "p: q k v; l: q_token_stride q_head_stride k_token_stride k_head_stride v_token_stride v_head_stride;"
        "p: g beta; l: g_token_stride beta_token_stride; p: starts slots into fresh initial final out;"
        "l: out_token_stride out_head_stride; p: tape")


class DeltaGradArgs(C.Structure):
    """lrmoe_delta_grad_args."""

    _fields_ = _fields("p: d_out; l: d_out_token_stride d_out_head_stride; p: d_final tape dq dk dv dg dbeta d_initial")


BEAM_MAX = 32            # beams of a group
FORK_TENSORS = 64        # tensors of one lrmoe_fork_rows call
FORK_BYTES = 32768       # its pieces of a row, of which a call has fewer than
FORK_PIECES = 1 << 24
FORK_CACHES = 32         # caches of one lrmoe_page_fork call
PAGE_MAX_ROWS = 4096     # rows (sequences) of a page pool
PAGE_MAX_POSITIONS = 1 << 30  # max_pages * page at most
PAGE_STATUS_TOKENS = 1   # a negative count, or more new positions than the plan has room for
PAGE_STATUS_ROW = 2      # a row past its pages, or corrupt
PAGE_STATUS_POOL = 4     # not enough free pages
PAGE_STATUS_STALE = 8    # a plan committed after another plan, commit or release

STAGE_ROUTE = 1
STAGE_GATE_UP = 2
STAGE_DOWN = 4
STAGE_COMBINE = 8
STAGE_GATHER = 16
STAGE_LAYER = 32
STAGE_DELTA_MIXER = 64
STAGE_DELTA_RULE = 128
DELTA_WS_STATUS_OFFSET = 0  # int32 status word of a mixer workspace
DELTA_MAX_TOKENS = 16    # tokens per lrmoe_delta_mixer call
STAGE_ATTENTION = 256
ATTN_MAX_TOKENS = 16     # tokens per lrmoe_attn_decode call


class NativeError(RuntimeError):
    """A liblrmoe call returned a non-zero status."""

    def __init__(self, name: str, code: int, text: str):
        super().__init__(f"{name} failed ({code}): {text}")
        self.code = code


@lru_cache(maxsize=1)
def library() -> C.CDLL:
    if not LIBRARY.exists():
        raise RuntimeError(
            f"{LIBRARY} is missing: build it with `python -m lightreason_amd.build` "
            "(hipcc --offload-arch=gfx950); there is no CPU fallback")
    lib = C.CDLL(str(LIBRARY))
    for name, (argtypes, restype) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    return lib


def symbols() -> list[str]:
    return list(_SIGNATURES)


def call(name: str, *args) -> None:
    lib = library()
    code = getattr(lib, name)(*args)
    if code != LRMOE_OK:
        text = lib.lrmoe_error_string(code).decode()
        if code == LRMOE_E_ARG:
            raise ValueError(f"{name}: {text}")
        raise NativeError(name, code, text)


def workspace_bytes(tokens: int) -> int:
    return int(library().lrmoe_workspace_bytes(tokens))


def device_check() -> None:
    code = library().lrmoe_device_check()
    if code != LRMOE_OK:
        raise NativeError("lrmoe_device_check", code, library().lrmoe_error_string(code).decode())


def timing_enable(mask: int, launches: int = 4096) -> None:
    call("lrmoe_timing_enable", int(mask), int(launches))


def timing_collect(stage: int) -> tuple[float, int]:
    """(summed milliseconds, launches) of the timed launches of ``stage``."""
    ms, n = C.c_double(0.0), C.c_int(0)
    call("lrmoe_timing_collect", int(stage), C.byref(ms), C.byref(n))
    return ms.value, n.value


# ---- cheap calls ----------------------------------------------------------------

_HERE = nullcontext()
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_stream(device: torch.device) -> int:
    """The hipStream_t of torch's current stream on `device`."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def on_device(device: torch.device):
    """A context in which `device` is the current one (a launch goes to the
    current device, whatever device its tensors are on)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


_traits = attrgetter("dtype", "shape", "device")
_stride = methodcaller("stride")


def checked(forms: dict, tensors, *rest):
    """(signature, form): what the checks of a call depend on -- types,
    shapes, devices and strides of its tensors (None for one that is left
    out), its other arguments and their types (1, 1.0 and True compare equal)
    -- and the form kept for it, if any; (None, None) where an argument is not
    what it should be.  Addresses are not part of it: the library checks their
    alignment in every call."""
    try:
        given = [t for t in tensors if t is not None]
        missing = None if len(given) == len(tensors) else tuple([t is None for t in tensors])
        key = (tuple(map(_traits, given)), tuple(map(_stride, given)), missing, rest, tuple(map(type, rest)))
        return key, forms.get(key)
    except (AttributeError, TypeError, RuntimeError):
        return None, None


def remember(forms: dict, key, form) -> None:
    """Keep the checked form of a signature (a bounded number of them)."""
    if key is not None:
        if len(forms) >= 1024:
            forms.clear()
        forms[key] = form


_WORKSPACES = threading.local()


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch (not cleared) of this thread on torch's current stream of
    `device`, grown as calls need it: two threads' calls on one stream may
    come with their launches mixed, so they share none.  A call under capture
    gets scratch of its own from its graph's memory, so that graphs replayed
    on different streams share none."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    try:
        held = _WORKSPACES.held
    except AttributeError:
        held = _WORKSPACES.held = {}
    key = (device, current_stream(device))
    ws = held.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = held[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws
