"""Paged 8-bit key / value cache and the attention of new tokens over it.

The cache is four tensors of the caller's: int8 codes ``[pages, kv_heads, page_size, dim]`` and
float32 scales ``[pages, kv_heads, page_size]`` for keys and for values.  Which tokens of which
sequences a call means is device data, so that a step can be captured into a graph and replayed:

``starts``   int32 ``[batch + 1]``: rows ``starts[b] .. starts[b+1]`` of the packed ``[rows, ...]``
             tensors are the new tokens of sequence ``b``
``lengths``  int32 ``[batch]``: cached tokens of every sequence, the new ones included
``table``    int32 ``[batch, width]``: position ``p`` lies in page ``table[b][p // page_size]``

Rows behind ``starts[batch]`` (padding) are left as they are.  Contents that contradict the sizes
(rows out of order, more tokens than the table has room for, a page that does not exist) fault
nothing: the sequence or token is passed over, a status bit is raised and ``Session.sync`` reports it.

The reference has no cache; its attention block is a graph of matmuls over whole sequences.
"""
from __future__ import annotations

import ctypes as C
import operator

import torch

from . import exceptions
from ._lib import EWORKSPACE, check, lib
from .session import launch_context


class _Struct(C.Structure):  # tfccb200_cache of include/tfcc_b200.h
    _fields_ = [("keys", C.c_void_p), ("key_scales", C.c_void_p), ("values", C.c_void_p),
                ("value_scales", C.c_void_p), ("pages", C.c_uint), ("page_size", C.c_uint),
                ("kv_heads", C.c_uint), ("dim", C.c_uint)]


def _fixed(name):
    """An attribute that is read, and set to nothing but what it is (``cache.keys *= 2`` works in place and puts the
    same tensor back)."""
    slot = "_" + name

    def put(self, value):
        if value is None or getattr(self, slot, None) is not value:
            raise AttributeError(f"{name} of a PagedCache is fixed: make another one")

    def drop(self):
        raise AttributeError(f"{name} of a PagedCache is fixed")

    return property(operator.attrgetter(slot), put, drop)


class PagedCache:
    """The pool: ``keys`` / ``values`` int8 ``[pages, kv_heads, page_size, dim]``, ``key_scales`` /
    ``value_scales`` float32 ``[pages, kv_heads, page_size]``, all contiguous on one CUDA device.
    ``dim`` is 64 or 128, ``page_size`` a power of two up to 1024.

    The attributes are fixed: calls go by the addresses taken here, so another tensor needs another
    ``PagedCache`` (the tensors' contents are the caller's to change)."""

    __slots__ = ("_keys", "_key_scales", "_values", "_value_scales", "_pages", "_kv_heads", "_page_size", "_dim",
                 "_device", "_struct", "_ref")
    keys, key_scales, values, value_scales = _fixed("keys"), _fixed("key_scales"), _fixed("values"), _fixed("value_scales")
    pages, kv_heads, page_size, dim = _fixed("pages"), _fixed("kv_heads"), _fixed("page_size"), _fixed("dim")
    device = _fixed("device")

    def __init__(self, keys: torch.Tensor, key_scales: torch.Tensor, values: torch.Tensor,
                 value_scales: torch.Tensor):
        if not isinstance(keys, torch.Tensor) or keys.dim() != 4 or keys.numel() == 0:
            raise exceptions.InvalidArgumentError("keys must be a [pages, kv_heads, page_size, dim] tensor")
        shape, device = keys.shape, keys.device
        for t, name, dtype, want in ((keys, "keys", torch.int8, shape), (values, "values", torch.int8, shape),
                                     (key_scales, "key_scales", torch.float32, shape[:3]),
                                     (value_scales, "value_scales", torch.float32, shape[:3])):
            if not isinstance(t, torch.Tensor) or t.shape != want:
                raise exceptions.InvalidArgumentError(f"{name}: expected shape {tuple(want)}")
            if t.dtype is not dtype:
                raise exceptions.NotImplementedError(f"{name}: implemented for {dtype}, got {t.dtype}")
        for t in (keys, key_scales, values, value_scales):
            if not t.is_cuda or t.get_device() != device.index or not t.is_contiguous():
                raise exceptions.InvalidArgumentError("the cache's tensors must be contiguous CUDA tensors on one device")
        pages, kv_heads, page_size, dim = shape
        if dim not in (64, 128):
            raise exceptions.InvalidArgumentError(f"the cache exists for dim 64 and 128, not {dim}")
        if page_size > 1024 or page_size & (page_size - 1):
            raise exceptions.InvalidArgumentError(f"page_size must be a power of two up to 1024, not {page_size}")
        self._keys, self._key_scales, self._values, self._value_scales = keys, key_scales, values, value_scales
        self._pages, self._kv_heads, self._page_size, self._dim, self._device = pages, kv_heads, page_size, dim, device
        self._struct = _Struct(keys.data_ptr(), key_scales.data_ptr(), values.data_ptr(), value_scales.data_ptr(),
                               pages, page_size, kv_heads, dim)
        self._ref = C.byref(self._struct)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, dim: int, device) -> "PagedCache":
        """A new pool with uninitialised contents."""
        def make(dtype, *shape):
            return torch.empty(shape, dtype=dtype, device=device)
        return cls(make(torch.int8, pages, kv_heads, page_size, dim), make(torch.float32, pages, kv_heads, page_size),
                   make(torch.int8, pages, kv_heads, page_size, dim), make(torch.float32, pages, kv_heads, page_size))


def _sequences(cache, starts, lengths, table):
    """(starts, lengths, table pointers, batch, table width) of a call, checked."""
    if not isinstance(cache, PagedCache):
        raise exceptions.InvalidArgumentError("cache must be a PagedCache")
    index = cache._device.index
    for t, name, rank in ((starts, "starts", 1), (lengths, "lengths", 1), (table, "table", 2)):
        # (a tensor of the CPU has device -1)
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != index or \
                len(t.shape) != rank or 0 in t.shape or not t.is_contiguous():
            raise exceptions.InvalidArgumentError(f"{name}: expected a contiguous int32 tensor of rank {rank} on {cache._device}")
    batch, width = table.shape
    if lengths.shape[0] != batch or starts.shape[0] != batch + 1:
        raise exceptions.InvalidArgumentError("starts, lengths and table don't match")
    return starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), batch, width


def _packed(t, name, rows, width, device):
    """Row pitch of a [rows, width] float32 tensor with contiguous rows (a column slice will do)."""
    shape = t.shape if isinstance(t, torch.Tensor) else ()
    if len(shape) != 2 or shape[1] != width or (rows is not None and shape[0] != rows) or shape[0] == 0:
        raise exceptions.InvalidArgumentError(f"{name}: expected a [{'rows' if rows is None else rows}, {width}] tensor")
    if t.dtype is not torch.float32:
        raise exceptions.NotImplementedError(f"{name}: implemented for float32, got {t.dtype}")
    pitch, step = t.stride()
    if t.get_device() != device.index or step != 1:
        raise exceptions.InvalidArgumentError(f"{name}: rows must be contiguous, on {device}")
    return width if shape[0] == 1 else pitch


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor,
           table: torch.Tensor) -> None:
    """Quantizes the new tokens' ``k`` and ``v`` ``[rows, kv_heads*dim]`` (float32; column slices of
    a packed projection will do) into their pages, one scale per token and head by the rule of
    ``quantization.quantize_tokens``.  No two new tokens may share a slot."""
    ps, pl, pt, batch, width = _sequences(cache, starts, lengths, table)
    cols = cache._kv_heads * cache._dim
    ldk = _packed(k, "k", None, cols, cache._device)
    ldv = _packed(v, "v", k.shape[0], cols, cache._device)
    sess, stream, guard = launch_context(cache._device)
    with guard:
        check(lib.tfccb200_cache_append_f32(stream, cache._ref, k.data_ptr(), ldk, v.data_ptr(), ldv,
                                            ps, pl, pt, batch, width, k.shape[0], sess.status_ptr))


def read(cache: PagedCache, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, rows: int,
         out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """``(k, v)``, float32 ``[rows, kv_heads*dim]``: ``scale * code`` of the tokens that ``append`` with
    the same sequences writes.  With ``starts`` counting whole sequences
    (``starts[b+1] - starts[b] == lengths[b]``) it reads all of them.  Rows behind ``starts[batch]``
    are left as they are in ``out`` (uninitialised when there is none)."""
    ps, pl, pt, batch, width = _sequences(cache, starts, lengths, table)
    cols = cache._kv_heads * cache._dim
    if out is None:
        if rows <= 0:
            raise exceptions.InvalidArgumentError("rows must be positive")
        k, v = cache._key_scales.new_empty((rows, cols)), cache._key_scales.new_empty((rows, cols))
        ldk = ldv = cols
    else:
        k, v = out
        ldk = _packed(k, "out[0]", rows, cols, cache._device)
        ldv = _packed(v, "out[1]", rows, cols, cache._device)
    sess, stream, guard = launch_context(cache._device)
    with guard:
        check(lib.tfccb200_cache_read_f32(stream, cache._ref, k.data_ptr(), ldk, v.data_ptr(), ldv,
                                          ps, pl, pt, batch, width, rows, sess.status_ptr))
    return k, v


def attention(cache: PagedCache, q: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor,
              scale: float | None = None, *, causal: bool = True, max_new: int | None = None,
              max_length: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q K^T) V`` of the new tokens' queries ``[rows, heads*dim]`` over the cached
    tokens of their sequences (append the new ones first), query head ``h`` reading kv head
    ``h // (heads // kv_heads)``.  ``causal``: a token sees the positions up to its own, otherwise
    all of its sequence; a row that sees none is 0.  ``scale`` defaults to ``1/sqrt(dim)``.

    ``max_new`` / ``max_length`` bound the new / cached tokens of any one sequence; the launch is
    shaped by them (they default to ``rows`` and the table's capacity, and a decode step wants
    ``max_new=1``).  A sequence beyond them is passed over and reported by ``Session.sync``.
    Rows behind ``starts[batch]`` are left as they are in ``out`` (uninitialised when there is none).
    """
    ps, pl, pt, batch, width = _sequences(cache, starts, lengths, table)
    if not isinstance(q, torch.Tensor) or q.dim() != 2 or q.shape[1] == 0 or q.shape[1] % (cache._kv_heads * cache._dim):
        raise exceptions.InvalidArgumentError("q: expected [rows, heads*dim] with heads a multiple of the cache's kv_heads")
    rows, cols = q.shape
    ldq = _packed(q, "q", None, cols, cache._device)
    if out is None:
        out, ldo = q.new_empty((rows, cols)), cols
    else:
        ldo = _packed(out, "out", rows, cols, cache._device)
    max_new = rows if max_new is None else max_new
    max_length = width * cache._page_size if max_length is None else max_length
    if max_new <= 0 or max_length <= 0:
        raise exceptions.InvalidArgumentError("max_new and max_length must be positive")
    max_new, max_length = min(max_new, rows), min(max_length, width * cache._page_size)
    heads = cols // cache._dim
    if scale is None:
        scale = 1.0 / float(cache._dim) ** 0.5
    sess, stream, guard = launch_context(cache._device)
    with guard:
        args = (stream, cache._ref, q.data_ptr(), ldq, out.data_ptr(), ldo, ps, pl, pt, batch, width, rows, heads,
                max_new, max_length, float(scale), 1 if causal else 0)
        st = lib.tfccb200_cache_attention_f32(*args, *sess.scratch_on(stream), sess.status_ptr)
        if st == EWORKSPACE:  # (refused before any launch)
            need = lib.tfccb200_cache_attention_workspace(cache._ref, batch, rows, heads, max_new, max_length)
            ws_ptr, ws_len, _owner = sess.workspace_on(need)
            st = lib.tfccb200_cache_attention_f32(*args, ws_ptr, ws_len, sess.status_ptr)
        check(st)
    return out
