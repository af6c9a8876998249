"""A paged key-value cache with retrieval over it, on torch tensors.

A model that answers from a long context searches its own cache: the keys are
the rows, a new token's query the query, blocks of keys the lists.  One step of
a serving loop:

    plan = kv_plan(past, new, table, free_pages, cursor, page_size, tokens)
    cache.append(k, v, plan.slots)
    blocks = cache.select(q, table, plan.requests, plan.positions, 32)
    out = cache.attend(q, table, plan.requests, plan.positions, blocks=blocks)

(or ``attend`` without ``blocks``: over everything).  Queries and keys get their
positions, and a norm of each head if the model has one, before that:

    q, k = rotary.rotate(q, k, plan.positions, requests=plan.requests, evicted=evicted)

and a cache that may hold only so much is cut now and then to the tokens that got
most attention, the pages of the others going back into the free list:

    out, lse = cache.attend(q, table, plan.requests, plan.positions, lse=True)
    cache.weigh(q, table, plan.starts, plan.positions, lse, mass)
    kept = cache.keep(mass, plan.lengths, budget, first=4, recent=128)
    lengths, cursor = cache.compact(table, plan.lengths, kept, free_pages, plan.cursor, mass=mass)
    evicted += plan.lengths - lengths

Tensors are on one GPU; every call runs on torch's current stream there, returns as
soon as its work is enqueued and can be captured into a graph.  The cache serves:
no call has a gradient.  The work is done by libmlxvs_c.so (``mlxvs_kv_*`` in
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


class _Rotary(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("dim", ctypes.c_int32), ("rotated", ctypes.c_int32),
                ("layout", ctypes.c_int), ("magnitude", ctypes.c_float), ("type", ctypes.c_int)]


class _Heads(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("heads", ctypes.c_int32),
                ("norm", ctypes.c_void_p), ("norm_type", ctypes.c_int), ("out", ctypes.c_void_p),
                ("out_token_stride", ctypes.c_int64), ("out_head_stride", ctypes.c_int64)]


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
    if not (isinstance(table, torch.Tensor) and table.dtype == torch.int32 and table.dim() == 2
            and table.device == device
            and (table.shape[1] <= 1 or table.stride(1) == 1 or table.numel() == 0)
            and (table.shape[0] <= 1 or table.stride(0) >= table.shape[1])):
        raise ValueError(f"[mlxvs::{op}] table must be an int32 [requests, columns] tensor on "
                         f"{device} with contiguous rows that do not overlap.")
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


# What the kernels have written is told to autograd, as by any operation in place: a
# backward pass that saved what was there before is an error then, not wrong.  (Tensors;
# a cheaper way to torch.autograd.graph.increment_version: 0.1 instead of 0.3 us)
_written = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


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
    _written((table, *out))
    return out


def _aligned(x) -> bool:
    """Whether the kernels read [tokens, heads, dim] rows as they are."""
    st = x.stride()
    return st[2] == 1 and not (st[0] & 7 or st[1] & 7 or x.data_ptr() & 15)


class Rotary:
    """Positions as rotations of queries and keys, with a norm of each head before
    it where the model has one.

    Args:
        dim: values a head, a multiple of 8 up to 256.
        rotated: how many of them are turned, the first ones (even; all of them
            by default); the others pass.
        layout: "halves": value i is turned with value i + rotated / 2; "pairs":
            value 2 i with value 2 i + 1.
        base: pair i turns by base^(-2 i / rotated) radians a position.
        scaling: None, or how that is changed for texts ``factor`` times as long
            as those of ``context`` tokens that the model learnt on: "linear" (all
            of them divided by factor), "base" (a larger base), "ramp" (those that
            make less than one turn over the context divided by factor, those that
            make 32 or more kept, a straight line between them; rotated values
            times 0.1 ln(factor) + 1).
        frequencies, magnitude: radians a position of each pair and the factor
            of rotated values, instead of all that: models whose ramp has other
            bounds, runs over the pairs instead of their turns or has no factor
            come with these.

    A position times a frequency (64 bits, of a turn) is exact modulo a turn, at
    every position; the angle is then rounded to 2^-26 of a turn.  ``frequencies``
    and ``magnitude`` can be read back.
    """

    _LAYOUTS = {"halves": 0, "pairs": 1}
    _SCALINGS = {None: 0, "linear": 1, "base": 2, "ramp": 3}

    def __init__(self, dim, *, rotated=None, layout="halves", base=10000.0, scaling=None,
                 factor=1.0, context=1, frequencies=None, magnitude=None, device="cuda"):
        op = "Rotary"
        dim = int(dim)
        rotated = dim if rotated is None else int(rotated)
        _need(8 <= dim <= 256 and dim % 8 == 0, op, "dim must be a multiple of 8 in [8, 256].")
        _need(0 <= rotated <= dim and rotated % 2 == 0, op, "rotated must be even, in [0, dim].")
        _need(layout in self._LAYOUTS, op, "layout must be 'halves' or 'pairs'.")
        _need(scaling in self._SCALINGS, op,
              "scaling must be None, 'linear', 'base' or 'ramp'.")
        pairs = rotated // 2
        radians, gain = (ctypes.c_double * pairs)(), ctypes.c_float(1.0)
        if frequencies is None:
            _check(_L().mlxvs_kv_rotary_frequencies(rotated, float(base), self._SCALINGS[scaling],
                                                    float(factor), float(context), radians,
                                                    ctypes.byref(gain)))
        else:
            _need(scaling is None, op, "frequencies are not scaled.")
            given = [float(f) for f in frequencies]
            _need(len(given) == pairs, op, f"frequencies must be {pairs} numbers.")
            radians[:] = given
        gain = gain.value if magnitude is None else float(magnitude)
        _need(math.isfinite(gain), op, "magnitude must be finite.")
        turns = (ctypes.c_uint64 * pairs)()
        _check(_L().mlxvs_kv_rotary_turns(radians, pairs, turns))
        self.dim, self.rotated, self.layout = dim, rotated, layout
        self.frequencies, self.magnitude = list(radians), gain
        device = torch.device(device)
        _need(device.type == "cuda", op, "device must be a GPU.")
        signed = [x - (1 << 64) if x >> 63 else x for x in turns]
        self._turns = torch.tensor(signed or [0], dtype=torch.int64, device=device)
        self._c = {dtype: _Rotary(self._turns.data_ptr(), dim, rotated, self._LAYOUTS[layout],
                                  gain, kind) for dtype, kind in _TYPES.items()}

    def _heads(self, x, name, norm, out, like):
        """(rows, where their results go, both as the kernels take them)"""
        op = "kv_rotate"
        device = self._turns.device
        if not (isinstance(x, torch.Tensor) and x.dim() == 3 and x.dtype in _TYPES
                and x.device == device and x.shape[2] == self.dim
                and (like is None or (x.shape[0] == like.shape[0] and x.dtype == like.dtype))):
            raise ValueError(f"[mlxvs::{op}] {name} must be a float16 or bfloat16 [tokens, heads, "
                             f"{self.dim}] tensor on {device}, as many tokens and of one type.")
        if norm is not None:
            if not (isinstance(norm, torch.Tensor) and norm.shape == (self.dim,)
                    and norm.dtype in (x.dtype, torch.float32) and norm.device == device
                    and norm.is_contiguous()):
                raise ValueError(f"[mlxvs::{op}] {name}_norm must be a contiguous {x.dtype} or "
                                 f"float32 [{self.dim}] tensor on {device}.")
            if norm.data_ptr() & 15:
                norm = norm.clone()
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            if not (isinstance(out, torch.Tensor) and out.shape == x.shape
                    and out.dtype == x.dtype and out.device == device and _aligned(out)):
                raise ValueError(f"[mlxvs::{op}] out of {name} must be a {x.dtype} "
                                 f"{list(x.shape)} tensor on {device}, 16-byte aligned with "
                                 "contiguous heads.")
        if not _aligned(x):
            x = x.clone(memory_format=torch.contiguous_format)
        st, so = x.stride(), out.stride()
        return x, norm, out, _Heads(x.data_ptr(), st[0], st[1], x.shape[1],
                                    None if norm is None else norm.data_ptr(),
                                    norm is not None and norm.dtype == torch.float32,
                                    out.data_ptr(), so[0], so[1])

    def rotate(self, q, k, positions, *, q_norm=None, k_norm=None, eps=1e-6, requests=None,
               evicted=None, out=None):
        """Queries [tokens, q_heads, dim] and keys [tokens, kv_heads, dim] (any
        token and head strides; k may be None), normed and turned.

        ``positions`` int32 [tokens] (KvPlan's); a token without one (-1) is
        turned by nothing, as at position 0.  ``evicted`` int32 [requests]: how many
        tokens a request's cache has lost, added to its tokens' positions;
        ``requests`` int32 [tokens] (KvPlan's) says whose they are.  ``q_norm`` / ``k_norm`` [dim]: weights of a norm of
        each head before that, x / sqrt(mean(x^2) + eps) x weight, over the whole
        head.  ``out``: (q, k) tensors to write into, which may be q and k
        themselves.  Returns (q, k).

        It has no gradient: the result of inputs that want one can be used, but not
        differentiated, and not written into ``out``."""
        op = "kv_rotate"
        _need(out is None or (isinstance(out, (tuple, list)) and len(out) == 2), op,
              "out must be (q, k).")
        _need(k is not None or k_norm is None, op, "k_norm needs k.")
        to_q, to_k = (None, None) if out is None else out
        given = q, k, q_norm, k_norm
        # (what is copied for the kernel has to live until the call is made)
        q, q_norm, q_out, hq = self._heads(q, "q", q_norm, to_q, None)
        k_out, hk = None, None
        if k is not None:
            k, k_norm, k_out, hk = self._heads(k, "k", k_norm, to_k, q)
        # (copies want a gradient where what they are copies of does)
        wanted = (q.requires_grad or (k is not None and k.requires_grad)
                  or (q_norm is not None and q_norm.requires_grad)
                  or (k_norm is not None and k_norm.requires_grad)) and torch.is_grad_enabled()
        _need(out is None or not wanted, op, "out takes no result that wants a gradient.")
        device, tokens = q.device, q.shape[0]
        pp = _ints(positions, "positions", op, device, size=tokens)
        pr = pe = None
        if evicted is not None:
            _need(requests is not None, op, "evicted needs requests.")
            pe = _ints(evicted, "evicted", op, device)
            pr = _ints(requests, "requests", op, device, size=tokens)
        with _On(device) as stream:
            _check(_L().mlxvs_kv_rotate_device(
                ctypes.byref(self._c[q.dtype]), ctypes.byref(hq), hk and ctypes.byref(hk), tokens,
                pp, pr, pe, 0 if evicted is None else evicted.numel(), float(eps), stream))
        if out is not None:
            _written((q_out,) if k is None else (q_out, k_out))
        if wanted:
            some = (q_out,) if k is None else (q_out, k_out)
            some = _NoGradient.apply(op, some, *(x for x in given if x is not None))
            return some[0], (None if k is None else some[1])
        return q_out, k_out


class KvCompact(NamedTuple):
    """What PagedKVCache.compact leaves: int32 tensors."""

    lengths: torch.Tensor  # [requests] tokens held now
    cursor: torch.Tensor   # [1] the first unused entry of free_pages


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
        _written(self._held)

    def _queries(self, q, table, requests, positions, op: str):
        q, pq, st = self._rows(q, "q", op)
        tokens, heads, _ = q.shape
        if heads < self.kv_heads or heads % self.kv_heads:
            raise ValueError(f"[mlxvs::{op}] q must have a multiple of {self.kv_heads} heads.")
        pt, stride = _table(table, op, self._device)
        rows, columns = table.shape
        return q, _Queries(pq, st[0], st[1], tokens, heads, columns, pt, stride, rows,
                           None if requests is None
                           else _ints(requests, "requests", op, self._device, size=tokens),
                           _ints(positions, "positions", op, self._device, size=tokens))

    def _workspace(self, size, q, qs, *args):
        """(tensor, bytes) of scratch memory on the current stream."""
        return self._memory((size, q.shape, qs.columns, qs.requests, args), q, size, self._ref,
                            ctypes.byref(qs), *args)

    def _scratch(self, size, like, *args):
        """The same for calls whose sizes are the numbers among args."""
        return self._memory((size, args), like, size, *args)

    def _memory(self, key, like, size, *args):
        need = self._sizes.get(key)
        if need is None:
            need = getattr(_L(), size)(*args)
            if need < 0:
                raise ValueError(_L().mlxvs_last_error().decode())
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            self._sizes[key] = need
        return (like.new_empty(need, dtype=torch.uint8) if need else None), need

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
            given = out
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
        if given is not None:
            _written((given,))
        if wanted:
            results = _NoGradient.apply(op, (out, sums) if lse else (out,), q, keys, values)
            return results if lse else results[0]
        return (out, sums) if lse else out

    def _mass(self, mass, op: str, requests: int, slots: int):
        if not (isinstance(mass, torch.Tensor) and mass.dim() == 3 and mass.dtype == torch.float32
                and mass.device == self._device and mass.is_contiguous()
                and mass.shape[0] == requests and mass.shape[1] == self.kv_heads
                and mass.shape[2] >= slots):
            raise ValueError(f"[mlxvs::{op}] mass must be a contiguous float32 [{requests}, "
                             f"{self.kv_heads}, slots] tensor on {self._device}, with at least "
                             f"{slots} slots.")
        return mass.data_ptr()

    def _mass_to_write(self, mass, op: str, requests: int, slots: int):
        at = self._mass(mass, op, requests, slots)
        _need(not (mass.requires_grad and torch.is_grad_enabled()), op,
              "mass is written: it takes no result that wants a gradient.")
        return at

    def weigh(self, q, table, starts, positions, lse, mass, *, scale=None, decay=1.0,
              longest=0) -> None:
        """Add the attention that each key gets from the step's tokens to ``mass``
        (float32 [requests, kv_heads, slots], a slot for each token that the table
        can hold).

        ``q`` and ``lse`` are those of ``attend(..., lse=True)`` over everything,
        with its ``scale``; ``starts`` and ``positions`` KvPlan's.  A key's mass is
        the sum of its probabilities over the tokens that see it and the query heads
        of its kv head.  The step's own keys start from zero, so a row of ``mass``
        needs no clearing before a new request gets it; what the others had is
        multiplied by ``decay`` (0: not read).  Masses past a request's last token,
        and of requests without tokens, stay as they are; so do those of a step that
        is left out, whose keys have what their places held before.  The same bits
        every time.  What is added are values: no gradient goes back to ``q`` and
        ``lse``, and ``mass`` must not want one.
        """
        op = "kv_weigh"
        cache = self._cache(op)
        q, qs = self._queries(q, table, None, positions, op)
        tokens, heads, dim = q.shape
        ps = _ints(starts, "starts", op, self._device, size=qs.requests + 1)
        if not (isinstance(lse, torch.Tensor) and lse.shape == (tokens, heads)
                and lse.dtype == torch.float32 and lse.device == self._device
                and lse.is_contiguous()):
            raise ValueError(f"[mlxvs::{op}] lse must be a contiguous float32 [tokens, q_heads] "
                             f"tensor on {self._device}.")
        pm = self._mass_to_write(mass, op, qs.requests, qs.columns * self.page_size)
        if scale is None:
            scale = 1.0 / math.sqrt(dim)
        longest = int(longest)
        with _On(self._device) as stream:
            work, size = self._workspace("mlxvs_kv_weigh_workspace", q, qs, longest)
            _check(_L().mlxvs_kv_weigh_device(
                cache, ctypes.byref(qs), ps, lse.data_ptr(), float(scale), float(decay), longest,
                pm, mass.shape[2], None if work is None else work.data_ptr(), size, stream))
        _written((mass,))

    def keep(self, mass, lengths, n, *, first=1, recent=1, above=None):
        """The ``n`` tokens of each request and kv head that a budget leaves: int32
        [requests, kv_heads, n], ascending.

        Of a request of more than ``above`` tokens (n by default) the ``first``
        first and the ``recent`` last ones are kept, and of the others those of the
        largest ``mass``, the lowest among equal ones (NaN counts as less than any
        other).  A request of at most ``above`` keeps all: its list is -1
        throughout.  ``lengths`` int32 [requests]."""
        op = "kv_keep"
        n, first, recent = int(n), int(first), int(recent)
        above = n if above is None else min(int(above), (1 << 31) - 1)
        _need(max(n, first, recent) < 1 << 31, op, "n, first and recent must be below 2^31.")
        device = self._device
        pl = _ints(lengths, "lengths", op, device)
        requests = lengths.numel()
        pm = self._mass(mass, op, requests, 0)
        with _On(device) as stream:
            _need(n >= 1, op, "n must be at least 1.")
            kept = mass.new_empty((requests, self.kv_heads, n), dtype=torch.int32)
            work, size = self._scratch("mlxvs_kv_keep_workspace", mass, requests, self.kv_heads,
                                       mass.shape[2])
            _check(_L().mlxvs_kv_keep_device(pm, requests, self.kv_heads, mass.shape[2], pl, n,
                                             first, recent, above, kept.data_ptr(),
                                             None if work is None else work.data_ptr(), size,
                                             stream))
        return kept

    def compact(self, table, lengths, kept, free_pages, cursor, *, mass=None,
                out=None) -> KvCompact:
        """Cut requests to the tokens of their lists, in place.

        ``kept`` int32 [requests, kv_heads, n]: ``keep``'s, or other ascending
        positions below a request's length, as many for every head.  Key, value and
        (with ``mass``) mass of position ``kept[r, h, j]`` move to position j;
        pages of which a token changed get new summaries.  The table stays as it is;
        the pages past a request's new end are written into ``free_pages`` before
        entry ``cursor[0]``, from where ``kv_plan`` takes them again.  A request
        whose list starts with -1 stays as it is, and so does one whose pages
        find no room in ``free_pages``.  Keys were rotated by their tokens'
        positions before they were written, so what they say stays true; new tokens
        are to be rotated by ``evicted`` more than their positions (``Rotary``).

        The pages of a request that is cut must be its own, not shared with another
        row.  ``lengths`` int32 [requests], ``cursor`` int32 [1].  ``out``: an
        earlier result of as many requests to write into (not the tensors that this
        call reads).  Returns KvCompact(lengths, cursor) after it."""
        op = "kv_compact"
        cache = self._cache(op)
        device = self._device
        pt, stride = _table(table, op, device)
        requests, columns = table.shape
        pl = _ints(lengths, "lengths", op, device, size=requests)
        if not (isinstance(kept, torch.Tensor) and kept.dim() == 3 and kept.dtype == torch.int32
                and kept.is_contiguous() and kept.device == device
                and kept.shape[:2] == (requests, self.kv_heads) and kept.shape[2] >= 1):
            raise ValueError(f"[mlxvs::{op}] kept must be a contiguous int32 [requests, kv_heads, "
                             f"n] tensor on {device}.")
        pf = _ints(free_pages, "free_pages", op, device)
        pc = _ints(cursor, "cursor", op, device, size=1)
        slots, pm = columns * self.page_size, None
        if mass is not None:
            pm = self._mass_to_write(mass, op, requests, slots)
            slots = mass.shape[2]
        n = kept.shape[2]
        with _On(device) as stream:
            if out is None:
                out = KvCompact(lengths.new_empty(requests), lengths.new_empty(1))
            else:
                _need(isinstance(out, KvCompact), op, "out must be a KvCompact.")
            po = _ints(out.lengths, "out.lengths", op, device, size=requests)
            pn = _ints(out.cursor, "out.cursor", op, device, size=1)
            work, need = self._scratch("mlxvs_kv_compact_workspace", lengths, cache, columns,
                                       requests, n)
            _check(_L().mlxvs_kv_compact_device(
                cache, pt, stride, columns, requests, pl, kept.data_ptr(), n, pf,
                free_pages.numel(), pc, pm, slots, po, pn,
                None if work is None else work.data_ptr(), need, stream))
        _written((*self._held, free_pages, *out) if mass is None
                 else (*self._held, free_pages, mass, *out))
        return out
