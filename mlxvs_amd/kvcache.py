"""A paged key-value cache with retrieval over it, on torch tensors.

A model that answers from a long context searches its own cache: the keys are
the rows, a new token's query the query, blocks of keys the lists.  One step of
a serving loop:

    plan = kv_plan(past, new, table, free_pages, cursor, page_size, tokens)
    cache.append(k, v, plan.slots)
    blocks = cache.select(q, table, plan.requests, plan.positions, 32)
    out = cache.attend(q, table, plan.requests, plan.positions, blocks=blocks)

(or ``attend`` without ``blocks``: over everything).  Tensors are on one GPU;
every call runs on torch's current stream there, returns as soon as its work is
enqueued and can be captured into a graph.  The cache serves: no call has a
gradient.  The work is done by libmlxvs_c.so (``mlxvs_kv_*`` in
include/mlxvs/mlxvs_c.h); without it the calls raise ImportError.  Extensions:
the reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch

from mlxvs_amd import _L, _check

_TYPES = {torch.float16: 0, torch.bfloat16: 1}


class _Cache(ctypes.Structure):
    _fields_ = [("keys", ctypes.c_void_p), ("values", ctypes.c_void_p),
                ("summaries", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("heads", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("dim", ctypes.c_int32), ("type", ctypes.c_int)]


class _Queries(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("tokens", ctypes.c_int64),
                ("q_heads", ctypes.c_int32), ("columns", ctypes.c_int32),
                ("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
                ("requests", ctypes.c_int64), ("token_request", ctypes.c_void_p),
                ("positions", ctypes.c_void_p)]


def _need(ok: bool, op: str, what: str) -> None:
    if not ok:
        raise ValueError(f"[mlxvs::{op}] {what}")


def _ints(x, name: str, op: str, device, dtype=torch.int32, size: Optional[int] = None):
    """The pointer of a contiguous 1-D tensor of whole numbers."""
    if not (isinstance(x, torch.Tensor) and x.dtype == dtype
            and (x.dim() == 1 if size is None else x.shape == (size,))
            and x.is_contiguous() and x.device == device):
        of = "" if size is None else f" of {size}"
        raise ValueError(f"[mlxvs::{op}] {name} must be a contiguous 1-D {dtype} tensor{of} on "
                         f"{device}.")
    return x.data_ptr()


def _table(table, op: str, device):
    _need(isinstance(table, torch.Tensor) and table.dtype == torch.int32 and table.dim() == 2
          and table.device == device
          and (table.shape[1] <= 1 or table.stride(1) == 1 or table.numel() == 0)
          and (table.shape[0] <= 1 or table.stride(0) >= table.shape[1]), op,
          f"table must be an int32 [requests, columns] tensor on {device} with contiguous rows "
          "that do not overlap.")
    return table.data_ptr(), max(table.stride(0), table.shape[1])


# the current stream's handle by device index (a cheaper way to
# torch.cuda.current_stream(i).cuda_stream: 0.1 instead of 2.6 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda i: torch.cuda.current_stream(i).cuda_stream)


class _On:
    """The current stream of a tensor's device, the device made current
    meanwhile."""

    __slots__ = ("index", "guard")

    def __init__(self, device):
        self.index = device.index
        self.guard = None if device.index == torch.cuda.current_device() \
            else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return _raw_stream(self.index) or None

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


class _NoGradient(torch.autograd.Function):
    """Marks results as depending on inputs that want a gradient: asking for it is
    an error then, not a gradient that is silently missing."""

    @staticmethod
    def forward(ctx, op, results, *inputs):
        ctx.op = op
        return results

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"[mlxvs::{ctx.op}] has no gradient.")


class _KvPlan(NamedTuple):
    slots: torch.Tensor      # [tokens] page x page_size + offset, -1: none
    requests: torch.Tensor   # [tokens] the token's request, -1 past the last token
    positions: torch.Tensor  # [tokens] its position in the request, -1: none
    starts: torch.Tensor     # [requests + 1] each request's first token
    lengths: torch.Tensor    # [requests] tokens held after the step
    first: torch.Tensor      # [requests] its first entry of free_pages, -1: not admitted
    cursor: torch.Tensor     # [1] the first unused entry of free_pages


class KvPlan(_KvPlan):
    """A step's bookkeeping (kv_plan): int32 tensors but ``slots`` (int64)."""

    # (what kv_plan made itself it need not check when it is passed back, as long
    # as its memory is where it was)
    made = None


def kv_plan(past, new, table, free_pages, cursor, page_size, tokens, *, out=None) -> KvPlan:
    """Block tables and slot maps of a step, from the requests' lengths.

    ``past`` / ``new`` int32 [requests]: tokens that a request holds and gets.
    ``table`` int32 [requests, columns]: its pages; the pages that new tokens
    need are taken from ``free_pages`` (int32, from entry ``cursor[0]`` on) in
    the requests' order and written into it.  ``tokens``: the batch's size; the
    places past the last token are padding.  A request that the columns or the
    free list cannot hold is not admitted (``first`` -1, its tokens without
    slots), nor is a later one that needs pages when the list has run out.
    ``out``: an earlier plan of the same sizes to write into (none of whose
    tensors may be an input of this call).  Returns KvPlan; the next step's
    ``past`` and ``cursor`` are its ``lengths`` and ``cursor``.
    """
    op = "kv_plan"
    _need(isinstance(past, torch.Tensor) and past.is_cuda, op, "past must be a GPU tensor.")
    device = past.device
    requests, tokens = past.numel(), int(tokens)
    _need(tokens >= 0, op, "tokens must not be negative.")
    pp = _ints(past, "past", op, device)
    pn = _ints(new, "new", op, device, size=requests)
    pf = _ints(free_pages, "free_pages", op, device)
    pc = _ints(cursor, "cursor", op, device, size=1)
    pt, stride = _table(table, op, device)
    _need(table.shape[0] == requests, op, "table must have a row for each request.")
    with _On(device) as stream:
        if out is None:
            i = past.new_empty
            out = KvPlan(past.new_empty(tokens, dtype=torch.int64), i(tokens), i(tokens),
                         i(requests + 1), i(requests), i(requests), i(1))
            ptrs = [x.data_ptr() for x in out]
            out.made = (device, requests, tokens, ptrs)
        else:
            _need(isinstance(out, KvPlan), op, "out must be a KvPlan.")
            ptrs = out.made and [x.data_ptr() for x in out]
            if ptrs is None or out.made != (device, requests, tokens, ptrs):
                sizes = (tokens, tokens, tokens, requests + 1, requests, requests, 1)
                ptrs = [_ints(x, f"out.{name}", op, device, torch.int32 if i else torch.int64, size)
                        for i, (x, name, size) in enumerate(zip(out, out._fields, sizes))]
        _check(_L().mlxvs_kv_plan_device(pp, pn, requests, pt, stride, table.shape[1], pf,
                                         free_pages.numel(), pc, int(page_size), tokens, *ptrs,
                                         stream))
    return out


class PagedKVCache:
    """Attention keys and values in pages, and retrieval over them.

    Args:
        keys: [pages, kv_heads, page_size, dim], float16 or bfloat16.
        values: [pages, kv_heads, dim, page_size] (transposed within a page).
        summaries: int8 [pages, kv_heads, dim], or None: no ``select``.
        scales: float32 [pages, kv_heads], with ``summaries``.

    ``page_size`` is a power of two from 16 to 256, ``dim`` a multiple of 8 up
    to 256.  The tensors are used in place and must be contiguous;
    ``PagedKVCache.empty`` makes them.  They stay the cache's: one that is
    resized or set to other memory is refused by the next call (a larger cache
    is another PagedKVCache).
    """

    def __init__(self, keys, values, summaries=None, scales=None):
        op = "PagedKVCache"
        _need(isinstance(keys, torch.Tensor) and keys.dim() == 4 and keys.dtype in _TYPES
              and keys.is_cuda and keys.is_contiguous(), op,
              "keys must be a contiguous float16 or bfloat16 [pages, kv_heads, page_size, dim] "
              "GPU tensor.")
        pages, heads, page, dim = keys.shape
        _need(isinstance(values, torch.Tensor) and values.shape == (pages, heads, dim, page)
              and values.dtype == keys.dtype and values.device == keys.device
              and values.is_contiguous(), op,
              f"values must be a contiguous {keys.dtype} [pages, kv_heads, dim, page_size] tensor "
              f"on {keys.device}.")
        _need(page in (16, 32, 64, 128, 256), op, "page_size must be 16, 32, 64, 128 or 256.")
        _need(8 <= dim <= 256 and dim % 8 == 0, op, "dim must be a multiple of 8 in [8, 256].")
        _need((summaries is None) == (scales is None), op, "summaries and scales come together.")
        if summaries is not None:
            _need(isinstance(summaries, torch.Tensor) and summaries.shape == (pages, heads, dim)
                  and summaries.dtype == torch.int8 and summaries.device == keys.device
                  and summaries.is_contiguous(), op,
                  f"summaries must be a contiguous int8 [pages, kv_heads, dim] tensor on "
                  f"{keys.device}.")
            _need(isinstance(scales, torch.Tensor) and scales.shape == (pages, heads)
                  and scales.dtype == torch.float32 and scales.device == keys.device
                  and scales.is_contiguous(), op,
                  f"scales must be a contiguous float32 [pages, kv_heads] tensor on "
                  f"{keys.device}.")
        # (read-only from outside: what is checked here is what the kernels get)
        self._keys, self._values, self._summaries, self._scales = keys, values, summaries, scales
        self._held = [x for x in (keys, values, summaries, scales) if x is not None]
        self._at = [x.data_ptr() for x in self._held]
        self._dtype, self._device = keys.dtype, keys.device
        self.page_size, self.dim, self.kv_heads = page, dim, heads
        self._c = _Cache(keys.data_ptr(), values.data_ptr(),
                         None if summaries is None else summaries.data_ptr(),
                         None if scales is None else scales.data_ptr(), pages, heads, page, dim,
                         _TYPES[keys.dtype])
        self._ref = ctypes.byref(self._c)
        self._sizes = {}  # workspace bytes of calls by their sizes

    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    summaries = property(lambda self: self._summaries)
    scales = property(lambda self: self._scales)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, dim, *, dtype=torch.bfloat16, device="cuda",
              summaries=True):
        """A cache of ``pages`` pages that holds nothing yet."""
        def make(*shape, kind=dtype):
            return torch.zeros(shape, dtype=kind, device=device)

        return cls(make(pages, kv_heads, page_size, dim), make(pages, kv_heads, dim, page_size),
                   make(pages, kv_heads, dim, kind=torch.int8) if summaries else None,
                   make(pages, kv_heads, kind=torch.float32) if summaries else None)

    def _cache(self, op: str):
        """The cache as the kernels take it, its memory being where it was."""
        _need([x.data_ptr() for x in self._held] == self._at, op,
              "the cache's tensors have moved: make another PagedKVCache of them.")
        return self._ref

    def _rows(self, x, name: str, op: str, heads: Optional[int] = None):
        """[tokens, heads, dim] rows as the kernels read them, with their address
        and strides: any token and head strides, 16-byte aligned (a copy where
        they are not)."""
        if not (isinstance(x, torch.Tensor) and x.dim() == 3 and x.dtype == self._dtype
                and x.device == self._device and x.shape[2] == self.dim
                and (heads is None or x.shape[1] == heads)):
            raise ValueError(f"[mlxvs::{op}] {name} must be a {self._dtype} [tokens, heads, "
                             f"{self.dim}] tensor on {self._device}.")
        at, st = x.data_ptr(), x.stride()
        if st[2] != 1 or st[0] & 7 or st[1] & 7 or at & 15:
            x = x.clone(memory_format=torch.contiguous_format)
            at, st = x.data_ptr(), x.stride()
        return x, at, st

    def append(self, k, v, slots) -> None:
        """Write the tokens' keys and values [tokens, kv_heads, dim] into their
        ``slots`` (int64 [tokens]; -1 or outside the cache: skipped), and the
        summaries of the pages that this completes.  What is written are values:
        no gradient goes back to ``k`` and ``v``."""
        op = "kv_append"
        cache = self._cache(op)
        k, pk, ks = self._rows(k, "k", op, self.kv_heads)
        v, pv, vs = self._rows(v, "v", op, self.kv_heads)
        tokens = k.shape[0]
        _need(v.shape[0] == tokens, op, "k and v must have the same tokens.")
        ps = _ints(slots, "slots", op, self._device, torch.int64, tokens)
        with _On(self._device) as stream:
            _check(_L().mlxvs_kv_append_device(cache, pk, ks[0], ks[1], pv, vs[0], vs[1], ps,
                                               tokens, stream))

    def _queries(self, q, table, requests, positions, op: str):
        q, pq, st = self._rows(q, "q", op)
        tokens, heads, _ = q.shape
        if heads < self.kv_heads or heads % self.kv_heads:
            raise ValueError(f"[mlxvs::{op}] q must have a multiple of {self.kv_heads} heads.")
        pt, stride = _table(table, op, self._device)
        rows, columns = table.shape
        return q, _Queries(pq, st[0], st[1], tokens, heads, columns, pt, stride, rows,
                           _ints(requests, "requests", op, self._device, size=tokens),
                           _ints(positions, "positions", op, self._device, size=tokens))

    def _workspace(self, size, q, qs, *args):
        """(tensor, bytes) of scratch memory on the current stream."""
        key = (size, q.shape, qs.columns, qs.requests, args)
        need = self._sizes.get(key)
        if need is None:
            need = getattr(_L(), size)(self._ref, ctypes.byref(qs), *args)
            if need < 0:
                raise ValueError(_L().mlxvs_last_error().decode())
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            self._sizes[key] = need
        return (q.new_empty(need, dtype=torch.uint8) if need else None), need

    def select(self, q, table, requests, positions, n, *, first=1, last=1):
        """The ``n`` best blocks of each token and kv head: int32 [tokens,
        kv_heads, n], ascending, -1 after the last.

        ``q`` [tokens, q_heads, dim]; ``table`` int32 [requests, columns];
        ``requests`` / ``positions`` int32 [tokens] (KvPlan's).  Candidates are
        the blocks up to the token's own.  The ``first`` first ones and the
        ``last`` latest (its own among them, last >= 1) are always taken, the
        others by the product of their summary with the query, the lowest
        block among equal ones.  Scores are whole-number products, so the list
        is the same from every implementation."""
        op = "kv_select"
        n = int(n)
        cache = self._cache(op)
        _need(self._summaries is not None, op, "the cache keeps no summaries.")
        q, qs = self._queries(q, table, requests, positions, op)
        with _On(self._device) as stream:
            work, size = self._workspace("mlxvs_kv_select_workspace", q, qs, n)
            out = q.new_empty((q.shape[0], self.kv_heads, n), dtype=torch.int32)
            _check(_L().mlxvs_kv_select_device(
                cache, ctypes.byref(qs), n, int(first), int(last), out.data_ptr(),
                None if work is None else work.data_ptr(), size, stream))
        return out

    def attend(self, q, table, requests, positions, *, blocks=None, scale=None, longest=0,
               lse=False, out=None):
        """Attention of the tokens over the cache, [tokens, q_heads, dim].

        A token sees its request's keys 0 .. position, its own among them;
        ``blocks`` int32 [tokens, kv_heads, n] (n <= 256) limits it to the
        listed ones.  A token that sees nothing gets zeros.  ``scale``: of the
        scores, 1 / sqrt(dim) by default.  ``longest``: tokens of the longest
        request, if the caller knows it (it guides how work is split, never
        what is computed).  With ``lse`` returns (out, float32 [tokens,
        q_heads] logarithms of the sums of exponentials).

        Neighbouring tokens of one request (kv_plan's order) are done together.
        A single token with a very long history is best given in a call of its
        own (slices of the same tensors) when the others are prompts.

        It has no gradient: the result of inputs that want one can be used, but
        not differentiated, and not written into ``out``."""
        op = "kv_attend"
        cache = self._cache(op)
        q, qs = self._queries(q, table, requests, positions, op)
        keys, values = self._keys, self._values
        wanted = (q.requires_grad or keys.requires_grad or values.requires_grad) \
            and torch.is_grad_enabled()
        tokens, heads, dim = q.shape
        n, pb = 0, None
        if blocks is not None:
            if not (isinstance(blocks, torch.Tensor) and blocks.dim() == 3
                    and blocks.dtype == torch.int32 and blocks.is_contiguous()
                    and blocks.device == q.device and blocks.shape[:2] == (tokens, self.kv_heads)
                    and blocks.shape[2] >= 1):
                raise ValueError(f"[mlxvs::{op}] blocks must be a contiguous int32 [tokens, "
                                 f"kv_heads, n] tensor on {q.device}.")
            n, pb = blocks.shape[2], blocks.data_ptr()
        if scale is None:
            scale = 1.0 / math.sqrt(dim)
        longest = int(longest)
        with _On(self._device) as stream:
            work, size = self._workspace("mlxvs_kv_attend_workspace", q, qs, n, longest)
            if out is None:
                out = q.new_empty((tokens, heads, dim))
            else:
                _need(not wanted, op, "out takes no result that wants a gradient.")
                _need(isinstance(out, torch.Tensor) and out.shape == q.shape
                      and out.dtype == q.dtype and out.device == q.device
                      and out.is_contiguous(), op,
                      f"out must be a contiguous {q.dtype} [tokens, q_heads, dim] tensor on "
                      f"{q.device}.")
            sums = q.new_empty((tokens, heads), dtype=torch.float32) if lse else None
            if tokens:
                _check(_L().mlxvs_kv_attend_device(
                    cache, ctypes.byref(qs), pb, n, float(scale), longest, out.data_ptr(),
                    None if sums is None else sums.data_ptr(),
                    None if work is None else work.data_ptr(), size, stream))
        if wanted:
            results = _NoGradient.apply(op, (out, sums) if lse else (out,), q, keys, values)
            return results if lse else results[0]
        return (out, sums) if lse else out
