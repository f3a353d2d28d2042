"""Operators around a paged key-value cache, on torch tensors: what an autoregressive model needs that is served beside
the synthesiser (a text or prosody model whose tokens, durations or pitch go to `SynthesizerTrn.infer_batches`).

    lengths, table, ring, cursor = ops.new_pages(requests=64, width=512, pages=20000, device="cuda")       # no request holds anything
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
(an int32 tensor of one element), where one is given.  No call records a gradient or carries a tangent along: tensors that ask
for a gradient are refused unless under torch.no_grad(), and dual tensors of forward-mode differentiation always.  The
reference has no counterpart (its attention, attentions.py:179-332, takes whole rows).

Between these functions and the C ABI stands a binding of host code (csrc/ops_binding.cpp, lib/_vits_ops.so): a step makes two
of these calls a layer, and a call of thirty arguments through ctypes costs as much as the kernel behind it."""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import math
import os
from typing import NamedTuple, Optional, Sequence

import torch

from . import _native as N


def _load():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_vits_ops.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m vits_amd.build`. vits_amd has no CPU or PyTorch fallback path.")
    loader = importlib.machinery.ExtensionFileLoader("_vits_ops", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_vits_ops", path, loader=loader))
    loader.exec_module(module)
    module.bind(*(C.cast(getattr(N.lib, f), C.c_void_p).value for f in (
        "vits_op_page_plan", "vits_op_rotary_store", "vits_op_paged_attention_workspace_bytes", "vits_op_paged_attention", "vits_last_error")), N.VitsError)
    return module


_bound = _load()


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


def _need_tensor(x, what: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise ValueError(what + " must be a tensor")


def _call(first: torch.Tensor, fn, *args) -> None:
    """fn(*args, stream) on the current stream of the first tensor's GPU.  (The two private functions are what torch.cuda.current_device and
    current_stream come down to; those take 2 us a call, as much as the rest of it.)"""
    index = first.get_device()
    if index < 0:
        fn(*args, 0)                           # refused, with the first reason found
    elif torch._C._cuda_getDevice() == index:
        fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            fn(*args, torch._C._cuda_getCurrentRawStream(index))


def page_plan(lengths: torch.Tensor, grow: torch.Tensor, table: torch.Tensor, ring: torch.Tensor, cursor: torch.Tensor, page_size: int,
              rows: Optional[int] = None, out: Optional[Sequence[torch.Tensor]] = None) -> PagePlan:
    """One step of a serving loop, planned on the GPU: request s gets grow[s] new tokens (or ends: -1), `table` its new
    pages from `ring`, and every new token a row with its request, position and slot; -1 in rows behind the last.
    `rows` is how many there may be (default: as `out` holds).  table and ring are changed in place; the new lengths and
    cursor are returned beside the old ones, so the caller decides when the step counts.  Where the step does not fit,
    `status` says why and nothing is changed."""
    _need_tensor(lengths, "page_plan: lengths")
    if out is None:
        if rows is None:
            raise ValueError("page_plan: give rows or out")
        n, d32 = lengths.numel(), dict(dtype=torch.int32, device=lengths.device)
        d64 = dict(dtype=torch.int64, device=lengths.device)
        out = PagePlan(torch.empty(n, **d32), torch.empty(2, **d64), torch.empty(n + 1, **d32), torch.empty(rows, **d32),
                       torch.empty(rows, **d32), torch.empty(rows, **d64), torch.empty(1, **d32))
    elif type(out) is not PagePlan:
        if len(out) != 7:
            raise ValueError("page_plan: out must hold a PagePlan's seven tensors")
        out = PagePlan._make(out)
    if rows is None:
        _need_tensor(out.request, "page_plan: out.request")
        rows = out.request.numel()
    _call(lengths, _bound.page_plan, lengths, grow, table, ring, cursor, page_size, rows, out)
    return out


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
    too).  With q alone and -freq it is its own gradient.  The slots of one call have to differ, and the caches share no cell; q turned
    in place may have k and v between its rows and heads.  An `out` made here with slots is filled with zeros first, by a launch of its own."""
    if q is not None:
        _need_tensor(q, "rotary_store: q")
    elif k is not None:
        _need_tensor(k, "rotary_store: k")
    if q is not None and out is None:
        # rows that are no rows are left as they were: not as the allocator found them
        out = (torch.empty if slot is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    first = k if q is None else q
    if first is None:
        raise ValueError("rotary_store: neither queries nor keys")
    _call(first, _bound.rotary_store, q, k, v, k_cache, v_cache, position, slot, freq, interleaved, scale, out, err_flag)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, request: torch.Tensor,
                    position: torch.Tensor, scale: Optional[float] = None, window: int = 0, max_keys: Optional[int] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every row of q [rows, heads, dim] attends to its request's tokens up to and with its own position (the last `window` of
    them, where that is not 0); heads / kv_heads query heads share a key-value head.  scale: 1 / sqrt(dim) by default.  A row
    that sees nothing gives 0, a row of request < 0 is left as it was (0 in an `out` made here, by a launch of its own).  lse (fp32 [rows, heads],
    optional) receives the log of the sum of the exponentials.  max_keys: the most tokens a row can see as far as the host
    knows, which guides how the work is split; the result does not depend on it beyond rounding."""
    _need_tensor(q, "paged_attention: q")
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if scale is None:
        if q.dim() != 3 or q.shape[-1] == 0:
            raise ValueError(f"paged_attention: q must be [rows, heads, dim], got {tuple(q.shape)}")
        scale = 1.0 / math.sqrt(q.shape[-1])
    _call(q, _bound.paged_attention, q, k_cache, v_cache, table, request, position, scale, window, 0 if max_keys is None else max_keys, out, lse, err_flag)
    return out
