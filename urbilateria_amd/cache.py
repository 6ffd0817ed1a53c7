"""Paged key-value caches on the GPU (``include/urb_cache.h``).

``PagedCache``: one layer's pages, in BF16 or E4M3, and writing rows into them.  ``Pager``: the pages and
slots of a step's new tokens, and tables that follow the beams of a search (``step.BeamSelector``).
``PagedAttention``: attention of the new tokens of each row over its pages.  They stand between
``step.qk_norm_rope`` and the output projection of a decoder layer.

All compute runs in ``liburb_moe.so``; this module only checks tensors and passes their addresses.  Calls
are stream-ordered; the tensors belong to the context's (the cache's) device.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

from . import native as N
from .moe import torch
from .step import _Context, _stream, _type, _vector

_CACHE_TYPES = {} if torch is None else {torch.bfloat16: N.DTYPES["BF16"],
                                         torch.float8_e4m3fn: N.DTYPES["F8_E4M3"]}


def _cache_type(dtype) -> int:
    return _CACHE_TYPES.get(dtype, 7)


def _call(name: str, device: int, stream, *args) -> None:
    """The library's function, on the device and the stream.  (torch.cuda.current_device() and a context
    manager take a microsecond of a call of six.)"""
    function = getattr(N.moe_lib(), name)
    handle = _stream(stream, device)
    if torch._C._cuda_getDevice() == device:
        st = function(*args, handle)
    else:
        with torch.cuda.device(device):
            st = function(*args, handle)
    if st:
        raise N.UrbError(st, name)


def _address(t, name: str, shape, dtype, device: int) -> int:
    """The address of a contiguous tensor of that shape on the device."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)} tensor on cuda:{device}")
    return t.data_ptr()


def _table(t, name: str, rows: int, device: int):
    """(address, entries from row to row, columns) of a [rows, columns] table."""
    if t.dim() != 2 or t.shape[0] != rows or t.dtype is not torch.int32 or t.get_device() != device or (
            t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be a torch.int32 [{rows}, blocks] tensor of contiguous rows on "
                         f"cuda:{device}")
    columns = t.shape[1]
    return t.data_ptr(), t.stride(0) if rows > 1 else columns, columns


def _strides(t, name: str, shape, dtype, device: int):
    """The strides of all axes but the last, whose values must be contiguous."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name} must be a {dtype} {list(shape)} tensor on cuda:{device}")
    s = t.stride()
    if s[-1] != 1:
        raise ValueError(f"{name}: the values of a head must be contiguous")
    return s[:-1]


class PagedCache:
    """One layer's keys and values (``urb_kv_cache``): ``k`` and ``v`` [pages, heads, page_size, head_dim],
    torch.bfloat16 or torch.float8_e4m3fn, of the same strides (either may be a view of another layout or
    a part of a wider buffer; a head's values are contiguous); for E4M3 ``k_scales`` and ``v_scales``
    [pages, heads, page_size] uint8, contiguous (E8M0).  Its tensors are not to be replaced (AttributeError) or
    resized: another cache takes others."""

    def __init__(self, k, v, k_scales=None, v_scales=None):
        if k.dim() != 4 or k.get_device() < 0:
            raise ValueError("k must be a [pages, heads, page_size, head_dim] tensor on a GPU")
        self.device = k.get_device()
        self.pages, self.heads, self.page_size, self.head_dim = k.shape
        self.dtype = k.dtype
        strides = _strides(k, "k", k.shape, k.dtype, self.device)
        other = _strides(v, "v", k.shape, k.dtype, self.device)
        if any(n > 1 and a != b for n, a, b in zip(k.shape, strides, other)):
            raise ValueError("k and v must have the same strides")
        at = [None if s is None else _address(s, name, k.shape[:3], torch.uint8, self.device)
              for s, name in ((k_scales, "k_scales"), (v_scales, "v_scales"))]
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self._desc = N.KvCache(k.data_ptr(), v.data_ptr(), *at, _cache_type(k.dtype), self.pages,
                               self.heads, self.page_size, self.head_dim, *strides)
        self._ref = ctypes.byref(self._desc)
        self._fixed = frozenset(self.__dict__)

    def __setattr__(self, name, value):
        # calls go by the addresses and sizes that were checked
        if name in self.__dict__.get("_fixed", ()):
            raise AttributeError(f"{name} of a PagedCache cannot be replaced")
        object.__setattr__(self, name, value)

    @classmethod
    def zeros(cls, pages: int, heads: int, page_size: int, head_dim: int, dtype=None, device="cuda"):
        """A cache of its own memory, all zeros; ``dtype`` torch.bfloat16 by default."""
        dtype = torch.bfloat16 if dtype is None else dtype
        shape = (pages, heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype,
                            device=device).view(dtype) for _ in range(2))
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, *(torch.full(shape[:3], 127, dtype=torch.uint8, device=device)
                           for _ in range(2)))

    def append(self, k, v, slots, stream=None) -> None:
        """Writes rows ``k`` and ``v`` [T, heads, head_dim] (torch.bfloat16 or torch.float32; tokens and
        heads may be strided, as in a fused q/k/v row) into the slots ``slots`` [T] int64; slots outside
        the cache, such as -1, skip their token."""
        tokens, dtype, dev = k.shape[0], k.dtype, self.device
        shape = (tokens, self.heads, self.head_dim)
        if k.shape != shape or v.shape != shape or v.dtype is not dtype or k.get_device() != dev or (
                v.get_device() != dev):
            raise ValueError(f"k and v must be {list(shape)} tensors of one type on cuda:{dev}")
        k_token, k_head, k_value = k.stride()
        v_token, v_head, v_value = v.stride()
        if k_value != 1 or v_value != 1:
            raise ValueError("k, v: the values of a head must be contiguous")
        rows = N.KvRows(k.data_ptr(), v.data_ptr(), _type(dtype), k_token, k_head, v_token, v_head)
        _call("urb_kv_append", dev, stream, self._ref, ctypes.byref(rows),
              _vector(slots, "slots", tokens, torch.int64, dev), tokens)


class Plan:
    """What ``Pager.plan_into`` writes: ``lengths`` [rows] int32 after the step, ``starts`` [rows + 1]
    int32, ``rows`` [tokens] int32, ``positions`` and ``slots`` [tokens] int64, ``count`` [1] int32, the
    free pages that are left.  Its tensors may be replaced, but not resized."""

    def __init__(self, lengths, starts, rows, positions, slots, count):
        self.lengths, self.starts, self.rows = lengths, starts, rows
        self.positions, self.slots, self.count = positions, slots, count

    def __setattr__(self, name, value):
        # the checked call is built again when a tensor is replaced
        object.__setattr__(self, name, value)
        object.__setattr__(self, "_checked", None)

    def _call_of(self, rows: int, device: int) -> tuple:
        if self._checked is None or self._checked[:2] != (rows, device):
            i32, i64, tokens = torch.int32, torch.int64, self.slots.numel()
            call = N.PagePlan(rows=rows, tokens=tokens)
            for name, field, n, dtype in (
                    ("lengths", "lengths_out", rows, i32), ("starts", "starts", rows + 1, i32),
                    ("rows", "token_rows", tokens, i32), ("positions", "positions", tokens, i64),
                    ("slots", "slots", tokens, i64), ("count", "free_count_out", 1, i32)):
                setattr(call, field, _vector(getattr(self, name), "plan." + name, n, dtype, device))
            object.__setattr__(self, "_checked", (rows, device, call, ctypes.byref(call)))
        return self._checked


class Pager(_Context):
    """Pages of steps and of beams (``urb_pager``).

    The free pages are a stack of the caller's: ``free`` [pages] int32, of which the first ``count`` [1]
    int32 are free (``new_stack`` makes a full one).  Tables are [rows, blocks] int32 with at least
    ``max_blocks`` columns."""

    _destroy, _sync = "urb_pager_destroy", "urb_pager_sync"

    def __init__(self, pages: int, page_size: int, max_rows: int, max_blocks: int, max_tokens: int = 0):
        self.pages, self.page_size = pages, page_size
        self.max_rows, self.max_blocks, self.max_tokens = max_rows, max_blocks, max_tokens
        desc = N.PagerDesc(pages, page_size, max_rows, max_blocks, max_tokens)
        self._make(N.moe_lib().urb_pager_create, ctypes.byref(desc))

    def new_stack(self):
        """(free, count) with all pages free; page 0 is taken first."""
        free = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=f"cuda:{self.device}")
        return free, torch.full_like(free[:1], self.pages)

    def new_plan(self, rows: int, tokens: int) -> Plan:
        """The tensors of a step of ``rows`` rows and up to ``tokens`` tokens."""
        dev = f"cuda:{self.device}"
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device=dev)
        i64 = lambda n: torch.empty(n, dtype=torch.int64, device=dev)
        return Plan(i32(rows), i32(rows + 1), i32(tokens), i64(tokens), i64(tokens), i32(1))

    def plan_into(self, lengths, added, tables, free, count, plan: Plan, stream=None) -> None:
        """The pages and slots for ``added`` [rows] int32 new tokens (None: one each) behind ``lengths``
        [rows] int32: enters pages in ``tables`` and fills ``plan``.  ``plan.lengths`` may be ``lengths``
        and ``plan.count`` ``count``; ``plan.starts``, ``rows`` and ``positions`` may be None."""
        dev, rows, i32 = self.device, lengths.numel(), torch.int32
        call, ref = plan._call_of(rows, dev)[2:]
        call.tables, call.table_stride, columns = _table(tables, "tables", rows, dev)
        if columns < self.max_blocks:
            raise ValueError(f"tables must have {self.max_blocks} columns")
        call.lengths = _vector(lengths, "lengths", rows, i32, dev)
        call.added = _vector(added, "added", rows, i32, dev)
        call.free_pages = _vector(free, "free", self.pages, i32, dev)
        call.free_count = _vector(count, "count", 1, i32, dev)
        _call("urb_pager_plan", dev, stream, self._ctx, ref)

    def plan(self, lengths, added, tables, free, count, tokens: int) -> Plan:
        """``plan_into`` with new tensors for ``tokens`` tokens; raises UrbError for rows that are not
        served."""
        plan = self.new_plan(lengths.numel(), tokens)
        self.plan_into(lengths, added, tables, free, count, plan)
        self.sync()
        return plan

    def fork_into(self, parents, tables, lengths, free, count, tables_out, lengths_out, count_out,
                  caches: Sequence[PagedCache] = (), stream=None) -> None:
        """Row i of each request becomes its row ``parents`` [requests, width] int32, or ends (negative):
        ``tables`` -> ``tables_out`` (other memory), ``lengths`` -> ``lengths_out`` [requests * width]
        int32, ``count`` -> ``count_out`` [1] int32 (these may be the same tensors), pages that are dropped
        pushed on ``free``.  Pages filled in part that several rows would share are copied in all
        ``caches``."""
        dev, i32 = self.device, torch.int32
        if parents.dim() != 2:
            raise ValueError("parents must be [requests, width]")
        requests, width = parents.shape
        rows = requests * width
        at, stride, columns = _table(tables, "tables", rows, dev)
        out, out_stride, out_columns = _table(tables_out, "tables_out", rows, dev)
        if min(columns, out_columns) < self.max_blocks:
            raise ValueError(f"tables must have {self.max_blocks} columns")
        for c in caches:
            if c.device != dev:
                raise ValueError(f"caches must be on cuda:{dev}")
        layers = (N.KvCache * len(caches))(*(c._desc for c in caches)) if caches else None
        call = N.PageFork(requests, width, stride, out_stride,
                          _vector(parents, "parents", rows, i32, dev), at,
                          _vector(lengths, "lengths", rows, i32, dev), out,
                          _vector(lengths_out, "lengths_out", rows, i32, dev),
                          _vector(free, "free", self.pages, i32, dev),
                          _vector(count, "count", 1, i32, dev),
                          _vector(count_out, "count_out", 1, i32, dev),
                          ctypes.addressof(layers) if caches else None, len(caches))
        _call("urb_pager_fork", dev, stream, self._ctx, ctypes.byref(call))


class PagedAttention(_Context):
    """Attention of the last ``queries`` tokens of each row over its pages (``urb_attention``), for caches of
    the heads, head_dim, page_size and type of ``cache`` (other layers' caches alike).

    ``dtype``: of queries and outputs, torch.bfloat16 (by default) or torch.float32.  ``window``: how many
    tokens a query reaches, itself among them (0: all).  ``scale``: head_dim ** -0.5 by default."""

    _destroy, _sync = "urb_attention_destroy", "urb_attention_sync"

    def __init__(self, q_heads: int, cache: PagedCache, max_rows: int, max_length: int, dtype=None,
                 queries: int = 1, window: int = 0, scale: Optional[float] = None):
        self.q_heads, self.queries, self.head_dim = q_heads, queries, cache.head_dim
        self.max_rows, self.max_length = max_rows, max_length
        self.dtype = torch.bfloat16 if dtype is None else dtype
        desc = N.AttentionDesc(q_heads, cache.heads, cache.head_dim, cache.page_size, _type(self.dtype),
                               _cache_type(cache.dtype), queries, window,
                               cache.head_dim ** -0.5 if scale is None else scale, max_rows, max_length)
        self._blocks = -(-max_length // cache.page_size)
        self._make(N.moe_lib().urb_attention_create, ctypes.byref(desc))

    def attend_into(self, q, cache: PagedCache, tables, lengths, out, lse=None, sinks=None,
                    stream=None) -> None:
        """``q`` [rows, queries, q_heads, head_dim] (rows, tokens and heads may be strided) over the pages
        ``tables`` [rows, blocks] int32 of ``lengths`` [rows] int32 tokens -> ``out``, which may be ``q``.
        ``lse`` [rows, queries, q_heads] f32: the logarithms of the denominators; ``sinks`` [q_heads] f32:
        a score without a value per head."""
        dev, rows = self.device, q.shape[0]
        shape = (rows, self.queries, self.q_heads, self.head_dim)
        q_strides = _strides(q, "q", shape, self.dtype, dev)
        out_strides = _strides(out, "out", shape, self.dtype, dev)
        at, stride, columns = _table(tables, "tables", rows, dev)
        if columns < self._blocks:
            raise ValueError(f"tables must have {self._blocks} columns")
        if cache.device != dev:
            raise ValueError(f"cache must be on cuda:{dev}")
        call = N.AttentionCall(rows, q.data_ptr(), out.data_ptr(), *q_strides, *out_strides, at, stride,
                               _vector(lengths, "lengths", rows, torch.int32, dev),
                               _vector(sinks, "sinks", self.q_heads, torch.float32, dev),
                               None if lse is None else _address(lse, "lse", shape[:3], torch.float32,
                                                                 dev))
        _call("urb_attend", dev, stream, self._ctx, cache._ref, ctypes.byref(call))

    def attend(self, q, cache: PagedCache, tables, lengths, sinks=None):
        """-> out; raises UrbError for lengths or table entries out of range."""
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        self.attend_into(q, cache, tables, lengths, out, sinks=sinks)
        self.sync()
        return out
