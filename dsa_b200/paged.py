"""Paged key/value cache next to the indexer: append, attention of new tokens over the cache,
and attention over the positions that a top-k selected.

The reference project temporal_dsa stops at the selection of the keys; a decode step goes on
with these: ``PagedAppender.append`` writes the new tokens' keys (rotated) and values into
their pages, ``paged_attention`` lets a chunk of new tokens attend to the cache (a prompt's
chunk, drafted tokens, or one token per sequence), and ``selected_attention`` lets each token
attend to the positions of its indexer's top-k only.

A cache is two page arrays ``[pages, page_size, kv_heads, head_dim]``; a batch names the
sequences of one call by a page table, the row ranges of their new tokens and their lengths.
The new tokens of all sequences are packed: ``[tokens, heads, head_dim]``, sequence ``b`` in
rows ``query_starts[b]`` to ``query_starts[b + 1] - 1``.  All kernels run on the current torch
stream of the current device, which has to be the cache's (``with torch.cuda.device(...)`` for
another); the batch's tensors live on the device, and nothing here waits for it.
"""

from __future__ import annotations

import ctypes as C
import math
import struct
import threading

import torch

from . import _capi as capi
from .indexer import require_cuda, stream_ptr

# torch.cuda.is_current_stream_capturing without its Python frame
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing",
                     torch.cuda.is_current_stream_capturing)

# torch.cuda.current_device without its Python frame (0.1 us of a call of 9)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

_DTYPES = {torch.float16: capi.TDSA_F16, torch.bfloat16: capi.TDSA_BF16}


class PagedKV:
    """The pages of a cache: ``keys`` and ``values`` ``[pages, page_size, kv_heads, head_dim]``,
    bfloat16 or float16, with the same strides (views of one interleaved buffer have them)."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor):
        require_cuda(keys, values)
        if keys.dim() != 4 or keys.shape != values.shape:
            raise ValueError("keys and values must be [pages, page_size, kv_heads, head_dim]")
        if keys.dtype not in _DTYPES or values.dtype != keys.dtype:
            raise ValueError("keys and values must share a dtype, bfloat16 or float16")
        if keys.device != values.device:
            raise ValueError("keys and values must be on one device")
        if keys.stride() != values.stride() or keys.stride(-1) != 1:
            raise ValueError("keys and values must have the same strides, 1 on the last axis")
        self.keys, self.values = keys, values
        self.pages, self.page_size, self.kv_heads, self.head_dim = keys.shape
        self.dtype, self.device, self._index = keys.dtype, keys.device, keys.get_device()
        self._scale = 1.0 / math.sqrt(self.head_dim) if self.head_dim else 1.0
        self._c = capi.TdsaPagedCache(keys.data_ptr(), values.data_ptr(), *keys.stride()[:3],
                                      *keys.shape, _DTYPES[keys.dtype])
        self._ref = C.byref(self._c)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV":
        shape = (pages, page_size, kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))


class PagedBatch:
    """The sequences of a call.  ``page_table`` int32 ``[batch, max_pages]``: position ``p`` of
    sequence ``b`` is row ``p % page_size`` of page ``page_table[b, p // page_size]``.
    ``query_starts`` int32 ``[batch + 1]`` and ``lengths`` int32 ``[batch]`` (positions with the
    new tokens, which are the last ones).  The tensors may be rewritten in place between calls; other
    tensors need a new batch.
    ``max_new``: the most new tokens a sequence has (default: no bound is known); it chooses
    the kernel, which changes results by rounding at most."""

    def __init__(self, page_table: torch.Tensor, query_starts: torch.Tensor,
                 lengths: torch.Tensor, *, max_new: int | None = None):
        require_cuda(page_table, query_starts, lengths)
        if page_table.dim() != 2 or page_table.shape[0] < 1 or page_table.shape[1] < 1:
            raise ValueError("page_table must be [batch, max_pages]")
        batch = page_table.shape[0]
        if query_starts.shape != (batch + 1,) or lengths.shape != (batch,):
            raise ValueError("query_starts must be [batch + 1] and lengths [batch]")
        for t in (page_table, query_starts, lengths):
            if t.dtype != torch.int32:
                raise ValueError("page_table, query_starts and lengths must be int32")
            if t.stride(-1) != 1:
                raise ValueError("page_table, query_starts and lengths need unit last stride")
            if t.device != page_table.device:
                raise ValueError("page_table, query_starts and lengths must be on one device")
        if max_new is not None and max_new < 0:
            raise ValueError("max_new must be >= 0")
        self.page_table, self.query_starts, self.lengths = page_table, query_starts, lengths
        self.batch, self.max_new, self.device = batch, max_new, page_table.device
        self._index = page_table.get_device()
        self._last = (None, None, None)

    def _for(self, tokens: int):
        """The C batch for a call of ``tokens`` rows (kept until the number changes)."""
        known, limit, ref = self._last
        if known != tokens or limit != self.max_new:
            limit, table = self.max_new, self.page_table
            ref = C.byref(capi.TdsaPagedBatch(
                table.data_ptr(), table.stride(0), self.query_starts.data_ptr(),
                self.lengths.data_ptr(), self.batch, table.shape[1], tokens,
                tokens if limit is None else min(limit, tokens)))
            self._last = (tokens, limit, ref)
        return ref


def _refuse_device(cache: PagedKV, batch: PagedBatch) -> None:
    """The library launches on the current device, and its status word is that device's."""
    if batch._index != cache._index:
        raise ValueError("batch and cache must be on one device")
    raise ValueError(f"the cache is on cuda:{cache._index}, which is not the current device: make "
                     "the call under torch.cuda.device(...)")


class _Rows(threading.local):
    """This thread's C row descriptors (four tdsa_token_rows), written anew for every call."""

    def __init__(self):
        self.buffer = (C.c_int64 * 12)()
        self.address = C.addressof(self.buffer)


_ROWS = _Rows()
_PACK6, _PACK12 = struct.Struct("6q").pack_into, struct.Struct("12q").pack_into


def _check_rows(t: torch.Tensor, cache: PagedKV, heads: int | None, tokens: int | None,
                name: str) -> None:
    """Why ``t`` is not [tokens, heads, head_dim] rows of the cache's kind, if it is not; strides
    and alignment are the library's check."""
    require_cuda(t)
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (
            heads is not None and shape[1] != heads) or (
            tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be [{'tokens' if tokens is None else tokens}, "
                         f"{heads or 'heads'}, {cache.head_dim}], got {list(shape)}")
    if t.dtype != cache.dtype:
        raise ValueError(f"{name} must have the cache's dtype")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on the cache's device")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} needs unit stride on the last axis")


_WORKSPACES: dict[tuple[int, int, int], tuple[torch.Tensor, int, int]] = {}


def paged_workspace(device: torch.device, head_dim: int,
                    stream: int | None = None) -> tuple[torch.Tensor, int, int]:
    """Scratch of the attention calls, its counters zeroed -> (buffer, address, bytes).  Outside
    CUDA-graph capture one buffer per (device, stream, head_dim) is kept: calls on one stream run
    in order and each leaves it ready for the next.  During a capture a fresh one is returned,
    which the graph keeps."""
    if stream is None:
        stream = stream_ptr(device)
    # device_status gives a device's buffers up when it reads a TDSA_ERR_TIMEOUT
    key = (device.index, stream, head_dim)
    ws = _WORKSPACES.get(key)
    capturing = _capturing()
    if ws is None or capturing:
        with torch.cuda.device(device):
            nbytes = capi.lib().tdsa_paged_workspace_bytes(head_dim)
        buffer = torch.empty(max(nbytes, 1), device=device, dtype=torch.uint8)
        buffer[:capi.TDSA_PAGED_COUNTER_BYTES].zero_()
        ws = (buffer, buffer.data_ptr(), nbytes)
        if not capturing:
            _WORKSPACES[key] = ws
    return ws


def release_paged_workspaces(index: int | None = None) -> None:
    """Forgets the kept workspaces of device ``index`` (default: of all): 20 to 39 MB for every
    stream and head dimension in use, which the next call there allocates anew."""
    for key in [k for k in _WORKSPACES if index is None or k[0] == index]:
        _WORKSPACES.pop(key, None)


class PagedAppender:
    """Appends new tokens to a paged cache, one launch (tdsa_paged_append): keys are rotated by
    their positions, keys and values go to their pages, and queries are rotated on the way.

    The rotation turns the pairs of the leading ``rope_dim`` features (a multiple of 16; 0 turns
    nothing) by ``position * inv_freq[j]``: features ``j`` and ``j + rope_dim / 2`` (the layout
    of ``apply_noninterleaved_rope``), or ``2 j`` and ``2 j + 1`` when ``interleaved``.
    ``inv_freq`` float32 ``[rope_dim / 2]`` defaults to ``rope_theta ** (-2 j / rope_dim)``.
    """

    def __init__(self, cache: PagedKV, *, rope_dim: int = 64, rope_theta: float = 10_000.0,
                 inv_freq: torch.Tensor | None = None, interleaved: bool = False):
        if rope_dim < 0 or rope_dim % 16 or rope_dim > cache.head_dim:
            raise ValueError("rope_dim must be a multiple of 16 up to the head dimension")
        half = rope_dim // 2
        if inv_freq is None:
            j = torch.arange(half, device=cache.device, dtype=torch.float64)
            inv_freq = (rope_theta ** (-j / max(half, 1))).float()
        require_cuda(inv_freq)
        if (inv_freq.shape != (half,) or inv_freq.dtype != torch.float32
                or inv_freq.device != cache.device):
            raise ValueError("inv_freq must be float32 [rope_dim / 2] on the cache's device")
        self.cache, self.rope_dim, self.interleaved = cache, int(rope_dim), int(bool(interleaved))
        self.inv_freq = inv_freq.contiguous()
        self._freq = self.inv_freq.data_ptr()
        self._fn = capi.lib().tdsa_paged_append

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor,
               q: torch.Tensor | None = None, *, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """k, v ``[tokens, kv_heads, head_dim]`` -> cache; returns the rotated ``q`` (in
        ``q_out``, a new tensor by default, ``q`` itself allowed) or None without ``q``.
        ``positions`` int64 ``[tokens]`` replaces the tokens' positions in the angles."""
        cache = self.cache
        dtype, index, shape = cache.dtype, cache._index, k.shape
        if batch._index != index or _current_device() != index:
            _refuse_device(cache, batch)
        ks, vs = k.stride(), v.stride()
        if not (len(shape) == 3 and shape == v.shape and shape[1] == cache.kv_heads
                and shape[2] == cache.head_dim and k.dtype is dtype and v.dtype is dtype
                and k.get_device() == index and v.get_device() == index and ks[2] == 1
                and vs[2] == 1):
            _check_rows(k, cache, cache.kv_heads, None, "k")
            _check_rows(v, cache, cache.kv_heads, shape[0], "v")
        tokens = shape[0]
        rows = _ROWS.address
        if q is not None:
            qshape = q.shape
            if q_out is None:
                q_out = torch.empty_like(q)
            qs, os = q.stride(), q_out.stride()
            if not (len(qshape) == 3 and qshape[0] == tokens and qshape[2] == cache.head_dim
                    and q_out.shape == qshape and q.dtype is dtype and q_out.dtype is dtype
                    and q.get_device() == index and q_out.get_device() == index
                    and qs[2] == 1 and os[2] == 1):
                _check_rows(q, cache, None, tokens, "q")
                _check_rows(q_out, cache, qshape[1], tokens, "q_out")
            _PACK12(_ROWS.buffer, 0, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                    q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), os[0], os[1])
            q_rows, o_rows, q_heads = rows + 48, rows + 72, qshape[1]
        else:
            if q_out is not None:
                raise ValueError("q_out needs q")
            _PACK6(_ROWS.buffer, 0, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1])
            q_rows = o_rows = None
            q_heads = 0
        pos = None
        if positions is not None:
            if (positions.dtype != torch.int64 or positions.shape != (tokens,)
                    or positions.device != cache.device or not positions.is_contiguous()):
                raise ValueError("positions must be contiguous int64 [tokens] on the cache's "
                                 "device")
            pos = positions.data_ptr()
        rc = self._fn(cache._ref, batch._for(tokens), rows, rows + 24, q_rows, o_rows, q_heads,
                      self._freq, self.rope_dim, self.interleaved, pos,
                      stream_ptr(cache.device))
        if rc:
            capi.check(rc)
        return q_out


def _attention_args(q, cache, batch, out, return_lse):
    """Checks and descriptors shared by the attention calls."""
    shape, dtype, index = q.shape, cache.dtype, cache._index
    if batch._index != index or _current_device() != index:
        _refuse_device(cache, batch)
    if out is None:
        out = torch.empty_like(q)
    qs, os = q.stride(), out.stride()
    if not (len(shape) == 3 and shape[2] == cache.head_dim and out.shape == shape
            and q.dtype is dtype and out.dtype is dtype and q.get_device() == index
            and out.get_device() == index and qs[2] == 1 and os[2] == 1):
        _check_rows(q, cache, None, None, "q")
        _check_rows(out, cache, shape[1], shape[0], "out")
    _PACK6(_ROWS.buffer, 0, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1])
    lse = (torch.empty(shape[:2], dtype=torch.float32, device=q.device) if return_lse else None)
    stream = stream_ptr(cache.device)
    return out, lse, shape, stream, paged_workspace(cache.device, cache.head_dim, stream)


_ALL = 1 << 30  # positions that a page table can have: a window of so many is none


def paged_attention(q: torch.Tensor, cache: PagedKV, batch: PagedBatch, *,
                    scale: float | None = None, window: int | None = None,
                    out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of the new tokens over their sequences' cached positions up to their own.

    q ``[tokens, heads, head_dim]`` (heads a multiple of the cache's kv_heads; head ``h`` reads
    key/value head ``h // (heads // kv_heads)``) -> out of the same shape, and with
    ``return_lse`` the float32 log-sum-exp ``[tokens, heads]``.  ``window``: a token sees only
    the last ``window`` positions up to its own.  ``scale`` defaults to ``head_dim ** -0.5``.
    A token that sees nothing gets zeros and ``-inf``.  The tokens must be in the cache already
    (``PagedAppender.append``).  ``out`` must not share memory with ``q``.
    """
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError("window must be >= 1")
    elif window > _ALL:  # before it is a C int
        window = _ALL
    out, lse, shape, stream, ws = _attention_args(q, cache, batch, out, return_lse)
    rows = _ROWS.address
    rc = capi.lib().tdsa_paged_attention(
        cache._ref, batch._for(shape[0]), rows, shape[1],
        cache._scale if scale is None else scale, window, rows + 24,
        None if lse is None else lse.data_ptr(), ws[1], ws[2], stream)
    if rc:
        capi.check(rc)
    return (out, lse) if return_lse else out


def selected_attention(q: torch.Tensor, cache: PagedKV, batch: PagedBatch,
                       indices: torch.Tensor, *, scale: float | None = None,
                       out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of every new token over the positions it lists: ``indices`` int32 or int64
    ``[tokens, k]``, positions of the token's own sequence in any order, negative entries
    skipped -- what ``topk`` and ``ScoreTopkPlan`` return.  The rest as ``paged_attention``."""
    out, lse, shape, stream, ws = _attention_args(q, cache, batch, out, return_lse)
    ishape, itype = indices.shape, indices.dtype
    if len(ishape) != 2 or ishape[0] != shape[0] or ishape[1] < 1:
        raise ValueError("indices must be [tokens, k]")
    if itype is not torch.int32 and itype is not torch.int64:
        raise ValueError("indices must be int32 or int64")
    if indices.stride(1) != 1 or indices.get_device() != cache._index:
        raise ValueError("indices need unit last stride, on the cache's device")
    rows = _ROWS.address
    rc = capi.lib().tdsa_selected_attention(
        cache._ref, batch._for(shape[0]), rows, shape[1],
        cache._scale if scale is None else scale, indices.data_ptr(), indices.element_size(),
        indices.stride(0), ishape[1], rows + 24, None if lse is None else lse.data_ptr(), ws[1],
        ws[2], stream)
    if rc:
        capi.check(rc)
    return (out, lse) if return_lse else out
