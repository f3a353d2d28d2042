"""Operators around a paged key-value cache, on torch tensors: what an autoregressive model needs that is served beside
the synthesiser (a text or prosody model whose tokens, durations or pitch go to `SynthesizerTrn.infer_batches`).

    pages = ops.new_pages(requests=64, width=512, pages=20000, page_size=16, device="cuda")  # table, ring, cursor, lengths
    k_cache, v_cache = (torch.empty(20000, kv_heads, 16, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))   # a layer
    freq = ops.rotary_frequencies(dim, device="cuda")
    ...
    plan = ops.page_plan(lengths, grow, table, ring, cursor, 16, rows=R)        # once a step: which rows, pages and slots
    q = ops.rotary_store(q, k, v, k_cache, v_cache, plan.position, plan.slot, freq)                # every layer
    o = ops.paged_attention(q, k_cache, v_cache, table, plan.request, plan.position)
    lengths, cursor = plan.lengths, plan.cursor

The kernels are in libvits_amd.so (vits_op_page_plan, vits_op_rotary_store, vits_op_paged_attention; include/vits_amd.h has
the formulas and the layouts); there is no fallback.  Everything runs on the current stream of the tensors' device, nothing
waits for the GPU, and with the outputs given (`out=`, `lse=`) a call can be captured into a graph.  Wrong shapes and types
raise ValueError, a library error VitsError; ids on the device that are out of range are left out and OR 1 into `err_flag`
(an int32 tensor of one element), where one is given.  The reference has no counterpart (its attention, attentions.py:179-332, takes
whole rows)."""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Sequence

import torch

from . import _native as N

_TYPES = {torch.float32: N.TYPE_F32, torch.float16: N.TYPE_F16, torch.bfloat16: N.TYPE_BF16}


class PagePlan(NamedTuple):
    """What `page_plan` gives, in the order of its `out`."""
    lengths: torch.Tensor    # int32 [requests]      tokens in the cache after the step
    cursor: torch.Tensor     # int64 [2]             head and tail of the ring after the step
    start: torch.Tensor      # int32 [requests + 1]  where each request's rows begin, and how many there are
    request: torch.Tensor    # int32 [rows]          -1 behind the last
    position: torch.Tensor   # int32 [rows]
    slot: torch.Tensor       # int64 [rows]
    status: torch.Tensor     # int32 [1]             0, or the OR of _native.PLAN_*: nothing was taken


class Pages(NamedTuple):
    """An empty cache's bookkeeping."""
    lengths: torch.Tensor    # int32 [requests]
    table: torch.Tensor      # int32 [requests, width]
    ring: torch.Tensor       # int32 [pages]
    cursor: torch.Tensor     # int64 [2]


def new_pages(requests: int, width: int, pages: int, device="cuda") -> Pages:
    """No request holds a token, and every page is free; a request can hold `width` pages."""
    i32 = dict(dtype=torch.int32, device=device)
    return Pages(torch.zeros(requests, **i32), torch.full((requests, width), -1, **i32), torch.arange(pages, **i32),
                 torch.tensor([0, pages], dtype=torch.int64, device=device))


def _refuse(what: str, name: str, t: torch.Tensor, dtype, shape) -> None:
    raise ValueError(f"{what}: {name} must be contiguous {dtype} [{shape}], got {t.dtype} {list(t.shape)}, strides {list(t.stride())}")


def _rows(what: str, name: str, t: torch.Tensor, shape, dtype) -> tuple:
    """Strides of a tensor of rows [rows, heads, dim] whose channels are contiguous."""
    strides = t.stride()
    if t.dtype is not dtype or t.shape != shape or (strides[2] != 1 and shape[2] > 1):
        raise ValueError(f"{what}: {name} must be {dtype} {list(shape)} with contiguous channels, got {t.dtype} {list(t.shape)}, strides "
                         f"{list(strides)}")
    return strides


def _caches(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor):
    """Shape and page stride of the two caches."""
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or k_cache.dtype not in _TYPES or v_cache.dtype != k_cache.dtype or v_cache.shape != shape or v_cache.stride() != strides \
            or strides[3] != 1 or strides[2] != shape[3] or strides[1] != shape[2] * shape[3]:
        raise ValueError(f"{what}: k_cache and v_cache must be alike, fp32, fp16 or bf16 [pages, kv_heads, page_size, dim], and contiguous within a "
                         f"page, got {k_cache.dtype} {list(shape)} and {v_cache.dtype} {list(v_cache.shape)}, strides {list(strides)} and "
                         f"{list(v_cache.stride())}")
    return shape, strides[0]


def _device(what: str, first: torch.Tensor, *more) -> int:
    """The GPU that every tensor given has to be on."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"{what}: tensors must be on a GPU (vits_amd has no CPU path)")
    for t in more:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: all tensors must be on one GPU, got {t.device} and {first.device}")
    return index


def _call(what: str, index: int, fn, *args) -> None:
    """fn(*args, stream) on the current stream of GPU `index`.  (The two private functions are what torch.cuda.current_device and
    current_stream come down to; those take 2 us a call, as much as a third of the rest of a call.)"""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        N.check(rc, what)


def page_plan(lengths: torch.Tensor, grow: torch.Tensor, table: torch.Tensor, ring: torch.Tensor, cursor: torch.Tensor, page_size: int,
              rows: Optional[int] = None, out: Optional[Sequence[torch.Tensor]] = None) -> PagePlan:
    """One step of a serving loop, planned on the GPU: request s gets grow[s] new tokens (or ends: -1), `table` its new
    pages from `ring`, and every new token a row with its request, position and slot; -1 in rows behind the last.
    `rows` is how many there may be (default: as `out` holds).  table and ring are changed in place; the new lengths and
    cursor are returned beside the old ones, so the caller decides when the step counts.  Where the step does not fit,
    `status` says why and nothing is changed."""
    what = "page_plan"
    i32, i64 = torch.int32, torch.int64
    n = lengths.numel()
    if out is None:
        if rows is None:
            raise ValueError("page_plan: give rows or out")
        d32, d64 = dict(dtype=i32, device=lengths.device), dict(dtype=i64, device=lengths.device)
        out = (torch.empty(n, **d32), torch.empty(2, **d64), torch.empty(n + 1, **d32), torch.empty(rows, **d32),
               torch.empty(rows, **d32), torch.empty(rows, **d64), torch.empty(1, **d32))
    elif len(out) != 7:
        raise ValueError("page_plan: out must hold a PagePlan's seven tensors")
    lengths_out, cursor_out, start, request, position, slot, status = out
    if rows is None:
        rows = request.numel()
    index = _device(what, lengths, grow, table, ring, cursor, *out)
    requests, width = table.shape if table.dim() == 2 else (-1, 0)
    if not (lengths.dtype is i32 and lengths.is_contiguous() and grow.dtype is i32 and grow.numel() == n and grow.is_contiguous()
            and ring.dtype is i32 and ring.is_contiguous() and cursor.dtype is i64 and cursor.numel() == 2 and cursor.is_contiguous()
            and table.dtype is i32 and requests == n and (table.stride(1) == 1 or width == 1)
            and lengths_out.dtype is i32 and lengths_out.numel() == n and lengths_out.is_contiguous()
            and cursor_out.dtype is i64 and cursor_out.numel() == 2 and cursor_out.is_contiguous()
            and start.dtype is i32 and start.numel() == n + 1 and start.is_contiguous()
            and request.dtype is i32 and request.numel() == rows and request.is_contiguous()
            and position.dtype is i32 and position.numel() == rows and position.is_contiguous()
            and slot.dtype is i64 and slot.numel() == rows and slot.is_contiguous() and status.dtype is i32 and status.numel() == 1):
        raise ValueError(f"page_plan: needs contiguous int32 lengths [requests], grow [requests], table [requests, width] (rows contiguous), ring "
                         f"[pages], int64 cursor [2], and as outputs a PagePlan's tensors with {rows} rows, got "
                         + ", ".join(f"{t.dtype} {list(t.shape)}" for t in (lengths, grow, table, ring, cursor, *out)))
    _call(what, index, N.lib.vits_op_page_plan, lengths.data_ptr(), grow.data_ptr(), n, table.data_ptr(), table.stride(0), width,
          ring.data_ptr(), ring.numel(), cursor.data_ptr(), page_size, lengths_out.data_ptr(), cursor_out.data_ptr(), start.data_ptr(),
          request.data_ptr(), position.data_ptr(), slot.data_ptr(), rows, status.data_ptr())
    return out if type(out) is PagePlan else PagePlan(*out)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original_length: int = 4096,
                       fast: float = 32.0, slow: float = 1.0, device="cuda") -> torch.Tensor:
    """Radians a position for each of the rotary_dim / 2 pairs, in 64 bits: base^(-2i / rotary_dim), for contexts `factor`
    times as long as the trained ones as they are ("none"), divided by the factor ("linear": positions are interpolated),
    with the base raised so that the slowest pair is divided by the factor and the fastest kept ("base"), or ("ramp")
    divided by it for pairs that turn less than `slow` times within original_length, kept for those that turn more than
    `fast` times, and blended linearly in the number of turns between (`rotary_store`'s `scale` takes the factor on the
    vectors that goes with it)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim must be even and positive")
    if not factor >= 1.0 or not base > 1.0:
        raise ValueError("rotary_frequencies: factor must be at least 1 and base above 1")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        if not fast > slow:
            raise ValueError("rotary_frequencies: fast must be above slow")
        keep = ((original_length * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        freq = freq / factor * (1 - keep) + freq * keep
    elif scaling not in ("none", "base"):
        raise ValueError("rotary_frequencies: scaling must be 'none', 'linear', 'base' or 'ramp'")
    return freq.to(device)


def rotary_store(q: Optional[torch.Tensor], k: Optional[torch.Tensor], v: Optional[torch.Tensor], k_cache: Optional[torch.Tensor],
                 v_cache: Optional[torch.Tensor], position: torch.Tensor, slot: Optional[torch.Tensor], freq: torch.Tensor,
                 interleaved: bool = False, scale: float = 1.0, out: Optional[torch.Tensor] = None,
                 err_flag: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Turns q [rows, heads, dim] by its rows' positions into `out` (new, given, or q itself), and k [rows, kv_heads, dim]
    into k_cache at the rows' slots, where v goes too, unturned.  The first 2 * freq.numel() channels of a head turn.
    Rows of slot < 0 are left as they were.  q may be None (nothing is returned), or k, v and the caches (then slot may be
    too).  With q alone and -freq it is its own gradient.  The slots of one call have to differ."""
    what = "rotary_store"
    if q is None and k is None:
        raise ValueError("rotary_store: neither queries nor keys")
    first = q if q is not None else k
    dtype = first.dtype
    if first.dim() != 3 or dtype not in _TYPES:
        raise ValueError(f"rotary_store: rows must be fp32, fp16 or bf16 [rows, heads, dim], got {dtype} {list(first.shape)}")
    rows, _, dim = first.shape
    index = _device(what, first, k, v, k_cache, v_cache, position, slot, freq, out, err_flag)
    if position.dtype is not torch.int32 or position.numel() != rows or not position.is_contiguous():
        _refuse(what, "position", position, torch.int32, rows)
    if freq.dtype is not torch.float64 or not freq.is_contiguous():
        _refuse(what, "freq", freq, torch.float64, "pairs")
    if slot is not None and (slot.dtype is not torch.int64 or slot.numel() != rows or not slot.is_contiguous()):
        _refuse(what, "slot", slot, torch.int64, rows)
    q_at = q_row = q_head = out_at = out_row = out_head = heads = 0
    if q is not None:
        shape = q.shape
        heads = shape[1]
        if out is None:
            # rows that are no rows are left as they were: not as the allocator found them
            out = (torch.empty if slot is None else torch.zeros)(shape, dtype=dtype, device=q.device)
        q_at, (q_row, q_head, _) = q.data_ptr(), _rows(what, "q", q, shape, dtype)
        out_at, (out_row, out_head, _) = out.data_ptr(), _rows(what, "out", out, shape, dtype)
    elif out is not None:
        raise ValueError("rotary_store: out without q")
    k_at = k_row = k_head = v_at = v_row = v_head = kc = vc = page_stride = pages = page_size = kv_heads = 0
    if k is not None:
        if v is None or k_cache is None or v_cache is None or slot is None:
            raise ValueError("rotary_store: keys need values, both caches and slots")
        (pages, kv_heads, page_size, channels), page_stride = _caches(what, k_cache, v_cache)
        if k_cache.dtype is not dtype or channels != dim:
            raise ValueError(f"rotary_store: caches of {k_cache.dtype} with {channels} channels for rows of {dtype} with {dim}")
        shape = (rows, kv_heads, dim)
        k_at, (k_row, k_head, _) = k.data_ptr(), _rows(what, "k", k, shape, dtype)
        v_at, (v_row, v_head, _) = v.data_ptr(), _rows(what, "v", v, shape, dtype)
        kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
    elif v is not None or k_cache is not None or v_cache is not None:
        raise ValueError("rotary_store: values or caches without keys")
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        _refuse(what, "err_flag", err_flag, torch.int32, 1)
    _call(what, index, N.lib.vits_op_rotary_store, q_at, q_row, q_head, out_at, out_row, out_head, heads, k_at, k_row, k_head, v_at, v_row, v_head,
          kc, vc, page_stride, pages, page_size, kv_heads, dim, _TYPES[dtype], position.data_ptr(), N.ptr(slot), rows, freq.data_ptr(),
          freq.numel(), scale, interleaved, N.ptr(err_flag))
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, heads: int, kv_heads: int, dim: int, dtype: int, max_keys: int) -> int:
    n = N.lib.vits_op_paged_attention_workspace_bytes(rows, heads, kv_heads, dim, dtype, max_keys)
    if n < 0:
        N.check(-1, "paged_attention")
    return n


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, request: torch.Tensor,
                    position: torch.Tensor, scale: Optional[float] = None, window: int = 0, max_keys: Optional[int] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every row of q [rows, heads, dim] attends to its request's tokens up to and with its own position (the last `window` of
    them, where that is not 0); heads / kv_heads query heads share a key-value head.  scale: 1 / sqrt(dim) by default.  A row
    that sees nothing gives 0, a row of request < 0 is left as it was (0 in an `out` made here).  lse (fp32 [rows, heads],
    optional) receives the log of the sum of the exponentials.  max_keys: the most tokens a row can see as far as the host
    knows, which guides how the work is split; the result does not depend on it beyond rounding."""
    what = "paged_attention"
    if q.dim() != 3:
        raise ValueError(f"paged_attention: q must be [rows, heads, dim], got {list(q.shape)}")
    rows, heads, dim = q.shape
    index = _device(what, q, k_cache, v_cache, table, request, position, out, lse, err_flag)
    (pages, kv_heads, page_size, channels), page_stride = _caches(what, k_cache, v_cache)
    shape = (rows, heads, channels)
    q_row, q_head, _ = _rows(what, "q", q, shape, k_cache.dtype)
    if request.dtype is not torch.int32 or request.numel() != rows or not request.is_contiguous():
        _refuse(what, "request", request, torch.int32, rows)
    if position.dtype is not torch.int32 or position.numel() != rows or not position.is_contiguous():
        _refuse(what, "position", position, torch.int32, rows)
    if table.dtype is not torch.int32 or table.dim() != 2 or (table.stride(1) != 1 and table.shape[1] > 1):
        _refuse(what, "table", table, torch.int32, "requests, width")
    if out is None:
        out = torch.zeros(shape, dtype=q.dtype, device=q.device)
    out_row, out_head, _ = _rows(what, "out", out, shape, q.dtype)
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous()):
        _refuse(what, "lse", lse, torch.float32, f"{rows}, {heads}")
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        _refuse(what, "err_flag", err_flag, torch.int32, 1)
    if (q.data_ptr() | q_row * q.element_size() | q_head * q.element_size()) & 15:
        q = q.clone(memory_format=torch.contiguous_format)      # the library reads heads on 16-byte addresses
        q_row, q_head, _ = q.stride()
    requests, width = table.shape
    keys = width * page_size if max_keys is None else max_keys
    if 0 < window < keys:
        keys = window
    dtype = _TYPES[q.dtype]
    nbytes = _workspace_bytes(rows, heads, kv_heads, dim, dtype, keys)
    # a workspace of this call's own: calls on different streams, and graphs that run side by side, share none
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _call(what, index, N.lib.vits_op_paged_attention, q.data_ptr(), q_row, q_head, k_cache.data_ptr(), v_cache.data_ptr(), page_stride, pages,
          page_size, table.data_ptr(), table.stride(0), width, requests, request.data_ptr(), position.data_ptr(), rows, heads, kv_heads, dim,
          dtype, 1.0 / math.sqrt(dim) if scale is None else scale, window, keys, out.data_ptr(), out_row, out_head, N.ptr(lse),
          N.ptr(err_flag), N.ptr(ws), nbytes)
    return out
