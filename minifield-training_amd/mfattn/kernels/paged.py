"""Serving over a paged key/value cache: plan, append and causal attention.

The cached attention of ``kernels/attention.py:264-282, :591-610`` and the
cache write of ``layers/attention.py:309-317`` for a batch of ragged
sequences, each with any number of new tokens (one: decode; several: drafted
tokens; many: a chunk of a prompt), whose keys and values live in pages of a
pool that all sequences share::

    step = paged.plan(query_starts, context_lengths, page_table, key_pages,
                      tokens=n, query_heads=hq)              # once a step
    q = paged.append(k, v, key_pages, value_pages, step, query=q, rotary=rot,
                     query_gain=qg, key_gain=kg, eps=1e-5)    # every layer
    out = paged.attention(q, key_pages, value_pages, step)

Pools are ``[pages, page_size, Hkv, 64]`` tensors or views of one (heads before
slots, keys and values in one tensor, a contiguous cache through
:func:`cache_pages`): only the last dimension has to be dense.  New tokens are
``[tokens, heads, 64]``, sequence after sequence.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from ..ops import (_ptr, _raw_stream, carries_tangent, dtype_code, launch, require_device,
                   token_rows)
from .rotary import Rotary


class Plan:
    """One step's new tokens and work items on the device, for every layer of the step."""

    __slots__ = ("buf", "page_table", "sequences", "tokens", "query_heads", "kv_heads", "pages",
                 "page_size", "pool", "code", "nbytes", "q_shape", "k_shape", "table_stride", "width",
                 "stream", "workspace")

    def __init__(self, buf, page_table, sequences, tokens, query_heads, pool, code, stream=0):
        self.buf, self.page_table = buf, page_table
        self.sequences, self.tokens, self.query_heads = sequences, tokens, query_heads
        self.pages, self.page_size, self.kv_heads, d = pool
        self.pool, self.code, self.nbytes = pool, code, buf.numel()
        self.q_shape, self.k_shape = (tokens, query_heads, d), (tokens, self.kv_heads, d)
        self.width = page_table.shape[1]
        self.table_stride = page_table.stride(0) if sequences > 1 else self.width
        self.stream = stream
        self.workspace = _sizes(sequences, tokens, query_heads, self.kv_heads, code)[1]

    def used_on(self, stream: int, device: torch.device) -> None:
        """A launch on ``stream`` reads the plan: its memory is not given out anew before."""
        if stream != self.stream:
            current = torch.cuda.current_stream(device)
            self.buf.record_stream(current)
            self.page_table.record_stream(current)

    def token_records(self) -> torch.Tensor:
        """``[tokens, 4]`` int32: position, page (negative: none), slot and sequence of each."""
        return self.buf[512:512 + 16 * self.tokens].view(torch.int32).view(-1, 4)


@functools.lru_cache(maxsize=256)
def _strides_of(strides: tuple[int, ...], shape: tuple[int, ...]):
    """The C ABI's (page, slot, head) strides; a dimension of one is never stepped over."""
    if strides[3] != 1 and shape[3] > 1:
        raise ValueError("the pages' last dimension must be dense")
    return (ctypes.c_longlong * 3)(*(s if n > 1 else 0 for s, n in zip(strides[:3], shape)))


def _pool_strides(key_pages: torch.Tensor, value_pages: torch.Tensor, pool: tuple[int, ...]):
    """Both pools' strides, which mostly are the same."""
    k, v = key_pages.stride(), value_pages.stride()
    strides = _strides_of(k, pool)
    return strides, strides if k == v else _strides_of(v, pool)


@functools.lru_cache(maxsize=256)
def _sizes(sequences: int, tokens: int, query_heads: int, kv_heads: int, code: int):
    """Bytes of a plan and of an attention's workspace."""
    lib = _lib.LIB
    return (lib.mf_paged_plan_bytes(sequences, tokens, query_heads, kv_heads, code),
            lib.mf_paged_attn_workspace_bytes(sequences, tokens, query_heads, kv_heads, code))


def _check_pool(key_pages: torch.Tensor, value_pages: torch.Tensor, plan: Plan) -> None:
    if key_pages.shape != plan.pool or value_pages.shape != plan.pool:
        raise ValueError(f"the plan is for pages {list(plan.pool)}, the call has "
                         f"{list(key_pages.shape)} and {list(value_pages.shape)}")


def _records_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _gain(gain: torch.Tensor | None, dtype: torch.dtype, d: int) -> torch.Tensor | None:
    if gain is None:
        return None
    if gain.shape != (d,):
        raise ValueError(f"gains must be [{d}], got {list(gain.shape)}")
    return gain if gain.dtype is dtype and gain.is_contiguous() else gain.to(dtype).contiguous()


def _int32(x: torch.Tensor, shape: tuple[int, ...], what: str) -> torch.Tensor:
    if x.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}, got {list(x.shape)}")
    if x.dtype is not torch.int32:
        if x.is_floating_point() or x.is_complex() or x.dtype is torch.bool:
            raise ValueError(f"{what} must hold integers, got {x.dtype}")
        if x.dtype is torch.int64:  # (a number that int32 does not hold names no other one)
            x = x.clamp(-2 ** 31, 2 ** 31 - 1)
        x = x.to(torch.int32)
    return x.contiguous()


def plan(query_starts: torch.Tensor, context_lengths: torch.Tensor, page_table: torch.Tensor,
         key_pages: torch.Tensor, *, tokens: int, query_heads: int) -> Plan:
    """Plan one step of ``R`` sequences over the pool ``key_pages`` (values have its shape).

    ``query_starts [R + 1]`` (ascending) delimits the sequences' new tokens in a
    batch of ``tokens``; those before the first and past the last belong to nobody.
    ``context_lengths [R]`` counts each sequence's tokens, the new ones
    included.  Token position ``p`` of sequence ``r`` is slot ``p % page_size``
    of page ``page_table[r, p // page_size]``; entries outside the pool (-1, say,
    behind a context or for a page that was given up) hold no keys, nor do
    positions beyond the table.  Nothing is read back to the host.  The table
    must stay as it is while the plan is used.  Another stream may use the plan
    once it waits for the plan's; a captured graph that reads a plan made outside
    of it needs the plan kept.
    """
    if key_pages.dim() != 4:
        raise ValueError("pages must be [pages, page_size, heads, head_dim]")
    if page_table.dim() != 2:
        raise ValueError("page_table must be [sequences, pages]")
    code = dtype_code(key_pages)
    pool = key_pages.shape
    pages, page_size, kv_heads, d = pool
    if d != _lib.HEAD_DIM:
        raise ValueError(f"paged attention serves head_dim {_lib.HEAD_DIM} (got {d})")
    r, width = page_table.shape
    starts = _int32(query_starts, (r + 1,), "query_starts")
    contexts = _int32(context_lengths, (r,), "context_lengths")
    table = page_table
    if table.dtype is not torch.int32 or (width > 1 and table.stride(1) != 1) or (
            r > 1 and table.stride(0) < width):
        table = _int32(table, (r, width), "page_table")
    device = require_device(key_pages, starts, contexts, table)
    nbytes, _ = _sizes(r, tokens, query_heads, kv_heads, code)
    buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
    stream = _raw_stream(device.index)
    launch(device, _lib.LIB.mf_paged_plan, starts.data_ptr(), contexts.data_ptr(), table.data_ptr(),
           table.stride(0) if r > 1 else width, r, tokens, width, page_size, pages, query_heads,
           kv_heads, code, buf.data_ptr(), nbytes, stream)
    return Plan(buf, table, r, tokens, query_heads, pool, code, stream)


def append(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
           value_pages: torch.Tensor, plan: Plan, *, query: torch.Tensor | None = None,
           rotary: Rotary | None = None, query_gain: torch.Tensor | None = None,
           key_gain: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor | None:
    """Write the step's keys and values into their pages, in place; returns the query.

    Keys and the query (where given) are RMS-normalised over each head with
    their gain, if they have one, then rotated at their token's position, if
    ``rotary`` is given; values are copied.  Tokens without a page are left out
    (their query is still returned).  Gains are taken in the pages' dtype, as the
    training prologue (``prologue.qk_norm_rope``) takes them in its tensors': a
    float32 gain of a bfloat16 model is rounded first.  float32 arithmetic from
    there, one rounding.  Pages that several sequences share must not be
    appended to.  Forward only.
    """
    dtype = key_pages.dtype
    for t in (key, value, value_pages) if query is None else (query, key, value, value_pages):
        if t.dtype is not dtype:
            raise ValueError(f"queries, keys, values and pages must share one dtype (got {dtype} "
                             f"and {t.dtype})")
    code = dtype_code(key_pages)
    if code != plan.code:
        raise ValueError("the plan is for pages of another dtype")
    if torch.is_grad_enabled() and _records_grad(key, value, key_pages, value_pages, query,
                                                 query_gain, key_gain):
        raise ValueError("paged.append has no backward; call it under torch.no_grad()")
    if carries_tangent(key, value, key_pages, value_pages, query, query_gain, key_gain):
        raise ValueError("paged.append has no derivative; an operand carries a tangent")
    _check_pool(key_pages, value_pages, plan)
    if key.shape != plan.k_shape or value.shape != plan.k_shape:
        raise ValueError(f"keys and values must be {list(plan.k_shape)}, got "
                         f"{list(key.shape)} and {list(value.shape)}")
    if query is None:
        if query_gain is not None:
            raise ValueError("query_gain needs a query")
    elif query.shape != plan.q_shape:
        raise ValueError(f"the query must be {list(plan.q_shape)}, got {list(query.shape)}")
    n, _, d = plan.k_shape
    qg, kg = _gain(query_gain, dtype, d), _gain(key_gain, dtype, d)
    if rotary is None:
        turn = (None, 0, 0, 1.0)
    elif not isinstance(rotary, Rotary) or rotary.head_dim != d:
        raise ValueError(f"rotary must be a Rotary of heads of {d}")
    else:
        turn = rotary._args
    if key_pages.data_ptr() == value_pages.data_ptr():
        raise ValueError("keys and values need pages of their own")
    device = require_device(key_pages, plan.buf, key, value, value_pages,
                            *(t for t in (query, qg, kg) if t is not None))
    key, k_step = token_rows(key)
    value, v_step = token_rows(value)
    out, q_step = None, 0
    if query is not None:
        query, q_step = token_rows(query)
        out = torch.empty(plan.q_shape, dtype=dtype, device=device)
    stream = _raw_stream(device.index)
    plan.used_on(stream, device)
    launch(device, _lib.LIB.mf_paged_append, _ptr(query), q_step, key.data_ptr(), k_step,
           value.data_ptr(), v_step, _ptr(qg), _ptr(kg), eps, *turn, code, n, plan.sequences,
           plan.query_heads, plan.kv_heads, d, plan.page_size, plan.pages, plan.buf.data_ptr(),
           plan.nbytes, key_pages.data_ptr(), value_pages.data_ptr(),
           *_pool_strides(key_pages, value_pages, plan.pool), _ptr(out), stream)
    return out


def attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, plan: Plan,
              *, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the step's new tokens over their sequences' pages.

    ``query [tokens, Hq, 64]``: the query at position ``p`` of its sequence sees
    the keys at positions ``0 .. p`` (the step's own keys must be in their pages:
    :func:`append`).  A query that sees no key yields zeros; a NaN or +infinity
    among its scores, or none above -infinity, yields NaN.  ``scale`` defaults
    to ``64 ** -0.5``.  Rows before the first sequence and behind the last are
    zeros, or left as they are in an ``out`` that is given.  Slots behind a
    context may hold anything.
    Forward only; the same inputs give the same bits.
    """
    shape, dtype = plan.q_shape, query.dtype
    if query.shape != shape:
        raise ValueError(f"the query must be {list(shape)}, got {list(query.shape)}")
    if key_pages.dtype is not dtype or value_pages.dtype is not dtype:
        raise ValueError(f"query and pages must share one dtype (got {dtype}, {key_pages.dtype} "
                         f"and {value_pages.dtype})")
    code = dtype_code(query)
    if code != plan.code:
        raise ValueError("the plan is for pages of another dtype")
    _check_pool(key_pages, value_pages, plan)
    if (query.requires_grad or key_pages.requires_grad or value_pages.requires_grad) \
            and torch.is_grad_enabled():
        raise ValueError("paged.attention has no backward; call it under torch.no_grad()")
    if carries_tangent(query, key_pages, value_pages):
        raise ValueError("paged.attention has no derivative; an operand carries a tangent")
    device = require_device(query, key_pages, value_pages, plan.buf)
    query, q_step = token_rows(query)
    if query.data_ptr() % 16:
        query = query.clone()
    zero_rest = out is None
    if zero_rest:
        out = torch.empty(shape, dtype=dtype, device=device)
    elif (out.shape != shape or out.dtype is not dtype or not out.is_contiguous()
          or out.device != device):
        raise ValueError(f"out must be a contiguous {dtype} {list(shape)} on {device}")
    n, hq, d = shape
    ws_bytes = plan.workspace
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    stream = _raw_stream(device.index)
    plan.used_on(stream, device)
    launch(device, _lib.LIB.mf_paged_attn, query.data_ptr(), q_step, key_pages.data_ptr(),
           value_pages.data_ptr(), *_pool_strides(key_pages, value_pages, plan.pool),
           plan.page_table.data_ptr(),
           plan.table_stride, code, n, plan.sequences, plan.width, plan.page_size, plan.pages, hq,
           plan.kv_heads, d, d ** -0.5 if scale is None else scale, plan.buf.data_ptr(), plan.nbytes,
           zero_rest, out.data_ptr(), ws.data_ptr(), ws_bytes, stream)
    return out


def cache_pages(cache: torch.Tensor, page_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A contiguous ``[B, capacity, Hkv, 64]`` cache as pages, without a copy.

    Returns the pages and the page table ``[B, capacity / page_size]`` of its rows.
    """
    if cache.dim() != 4 or not cache.is_contiguous():
        raise ValueError("the cache must be a contiguous [B, capacity, heads, head_dim] tensor")
    b, cap, h, d = cache.shape
    if page_size < 1 or cap % page_size:
        raise ValueError(f"the capacity {cap} must be whole pages of {page_size}")
    per = cap // page_size
    table = torch.arange(b * per, dtype=torch.int32, device=cache.device).view(b, per)
    return cache.view(b * per, page_size, h, d), table
