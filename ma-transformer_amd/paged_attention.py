"""Paged key/value cache: serving one new token at a time on MI355X.

The single-token form of this engine's attention (the reference has no cache:
its layers recompute every position).  A ``PagedCache`` holds the keys and
values of many streams in pages of ``page_size`` tokens; a stream is a row of a
page table.  One step of a model's attention layer is

    q = paged_append(cache, k, v, table, start, rotation=rot, query=q)   # new tokens into the cache
    o = paged_decode(q[:, 0], cache, table, start + 1)                   # attention of the newest token

``paged_decode`` reads all of a stream's keys, the causal window
[len-1-left, len-1] with the first ``num_global`` tokens (``sliding_forward``
with right=0, ``longformer_forward``'s local rows), or the pages that
``paged_select`` lists for it: the single-token form of ``select_blocks`` and
``selected_forward`` with blocks of one page.

All tensors are contiguous device tensors on one device, float32, bfloat16 or
float16 (tables, starts, lengths and lists int32); anything else raises
RuntimeError and launches nothing.  Calls run asynchronously on the current
stream and can be captured into a graph.  Tables, lengths and lists are read on
the device: entries outside their range are skipped, lengths are clamped to
what the table holds.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

import ma_attn as _ma
import sparse_attention_cuda as _ext

__all__ = ["PagedCache", "Rotation", "paged_append", "paged_decode", "paged_select"]


class _Desc(ctypes.Structure):
    """Mirror of ``ma_paged_desc`` (include/ma_paged.h)."""

    _fields_ = [(n, ctypes.c_int64) for n in (
        "batch", "num_tokens", "num_heads", "num_kv_heads", "head_dim", "num_pages", "page_size", "table_width")]
    _fields_ += [("dtype", ctypes.c_int32), ("interleaved", ctypes.c_int32)]
    _fields_ += [(n, ctypes.c_int64) for n in (
        "rotary_dim", "left", "num_global", "num_selected", "first_pages", "local_pages")]
    _fields_ += [("scale", ctypes.c_float), ("reserved", ctypes.c_int32),
                 ("start_event", ctypes.c_void_p), ("stop_event", ctypes.c_void_p)]


_lib = _ma.LIB
_P = ctypes.POINTER(_Desc)
_V = ctypes.c_void_p
_lib.ma_paged_append.restype = ctypes.c_int
_lib.ma_paged_append.argtypes = [_P] + [_V] * 12
_lib.ma_paged_decode_workspace_size.restype = ctypes.c_size_t
_lib.ma_paged_decode_workspace_size.argtypes = [_P]
_lib.ma_paged_decode.restype = ctypes.c_int
_lib.ma_paged_decode.argtypes = [_P] + [_V] * 9 + [ctypes.c_size_t, _V]
_lib.ma_paged_select.restype = ctypes.c_int
_lib.ma_paged_select.argtypes = [_P] + [_V] * 6


class PagedCache:
    """Keys and values [num_pages, page_size, num_kv_heads, head_dim], and with
    ``key_sums`` the float32 sums [num_pages, num_kv_heads, head_dim] of each
    page's stored keys, which ``paged_append`` keeps and ``paged_select`` reads.

    page_size: a multiple of 16; head_dim: a multiple of 8, at most 128.
    Memory is not cleared: no call reads a token that was not appended.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None, key_sums: bool = False):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        shape = (int(num_pages), int(page_size), int(num_kv_heads), int(head_dim))
        key = torch.empty(shape, dtype=dtype, device=dev)
        sums = torch.empty((shape[0], shape[2], shape[3]), dtype=torch.float32, device=dev) if key_sums else None
        self._set(key, torch.empty_like(key), sums)

    @classmethod
    def from_tensors(cls, key: torch.Tensor, value: torch.Tensor,
                     key_sums: Optional[torch.Tensor] = None) -> "PagedCache":
        """A cache over tensors the caller holds (not copied)."""
        self = cls.__new__(cls)
        self._set(key, value, key_sums)
        return self

    def _set(self, key, value, sums) -> None:
        _tensors("cache key", key, key.dtype if isinstance(key, torch.Tensor) else None, 4)
        if key.dtype not in _ma.DTYPES:
            raise RuntimeError("cache dtype must be float32, bfloat16 or float16")
        _tensors("cache value", value, key.dtype, 4, key.shape, key.device)
        P, ps, Hkv, D = key.shape
        if ps < 16 or ps % 16:
            raise RuntimeError("page_size must be a multiple of 16")
        if Hkv < 1 or D < 8 or D > 128 or D % 8:
            raise RuntimeError("head_dim must be a multiple of 8 from 8 to 128, with at least one head")
        if sums is not None:
            _tensors("key_sums", sums, torch.float32, 3, (P, Hkv, D), key.device)
        self._key, self._value, self._sums = key, value, sums
        self._descs = {}  # descriptors of calls on this cache, by the calls' sizes

    # the tensors stay the checked ones
    @property
    def key(self) -> torch.Tensor:
        return self._key

    @property
    def value(self) -> torch.Tensor:
        return self._value

    @property
    def key_sums(self) -> Optional[torch.Tensor]:
        return self._sums

    @property
    def page_size(self) -> int:
        return int(self._key.shape[1])


class Rotation:
    """The position rotation of queries and keys: pairs (j, j + dim/2), or
    (2j, 2j + 1) with ``interleaved``, of the first ``dim`` head elements turn by
    position * base^(-2j/dim).  ``inv_freq`` gives the dim/2 frequencies instead.
    Angles are computed in float64.  dim: a multiple of 16, at most head_dim."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, inv_freq=None, device=None):
        self.dim = int(dim)
        if self.dim < 16 or self.dim % 16:
            raise RuntimeError("rotation dim must be a multiple of 16")
        if inv_freq is None:
            if not float(base) > 0.0:
                raise RuntimeError("rotation base must be > 0")
            f = float(base) ** (-torch.arange(0, self.dim, 2, dtype=torch.float64) / self.dim)
        else:
            f = torch.as_tensor(inv_freq).detach().to(torch.float64).reshape(-1)
            if f.numel() != self.dim // 2:
                raise RuntimeError(f"inv_freq must hold dim/2 = {self.dim // 2} frequencies")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.inv_freq = f.to(dev).contiguous()
        self.interleaved = bool(interleaved)


def _tensors(name, t, dtype, dim, shape=None, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA (HIP) device tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != dim or (shape is not None and tuple(t.shape) != tuple(shape)):
        want = f"shape {tuple(shape)}" if shape is not None else f"{dim} dimensions"
        raise RuntimeError(f"{name} must have {want}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on another device than the cache")


def _valid(dtype, dev: int, *ts) -> bool:
    """Whether the tensors are contiguous, of one dtype, on device `dev`: with the
    shapes, the common valid call; any failure takes the ordered checks."""
    try:
        for t in ts:
            if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
                return False
        return dev >= 0
    except AttributeError:
        return False


def _int32(name, t, shape, cache) -> None:
    _tensors(name, t, torch.int32, len(shape), shape, cache._key.device)


def _table(page_table, B, cache) -> None:
    _tensors("page_table", page_table, torch.int32, 2, None, cache._key.device)
    if page_table.shape[0] != B:
        raise RuntimeError(f"page_table must have a row per stream ({B}), got {page_table.shape[0]}")


def _desc(cache, key, B, H, width, workspace=None, **kw):
    """(descriptor, workspace bytes) of a call, kept with the cache per `key` (the
    call's sizes); a call with kernel events gets its own."""
    hit = cache._descs.get(key)
    if hit is None:
        P, ps, Hkv, D = cache._key.shape
        if H < 1 or H % Hkv:
            raise RuntimeError(f"query heads ({H}) must be a multiple of the cache's heads ({Hkv})")
        d = _Desc(batch=B, num_heads=H, num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, table_width=width,
                  dtype=_ma.DTYPES[cache._key.dtype], left=-1)
        for k, v in kw.items():
            setattr(d, k, v)
        if len(cache._descs) > 256:
            cache._descs.clear()
        hit = cache._descs[key] = (d, int(workspace(ctypes.byref(d))) if workspace else 0)
    if _ext._events is not None:
        d = _Desc.from_buffer_copy(hit[0])
        d.start_event, d.stop_event = (e or None for e in _ext._events)
        return d, hit[1]
    return hit


def _ptr(t) -> Optional[int]:
    return t.data_ptr() or None if t is not None else None


def _call(fn, dev: int, *args) -> None:
    if _ext._on_device(dev, lambda stream: fn(*args, stream or None)) != 0:
        raise RuntimeError(_ma.last_error())


def _check_cache(cache) -> None:
    if not isinstance(cache, PagedCache):
        raise RuntimeError("cache must be a PagedCache")


def _check_append(cache, key, value, page_table, start, counts, query) -> None:
    dev = cache._key.device
    _tensors("key", key, cache._key.dtype, 4, None, dev)
    B, N = key.shape[:2]
    Hkv, D = cache._key.shape[2:]
    if tuple(key.shape[2:]) != (Hkv, D):
        raise RuntimeError(f"key must be [B, N, {Hkv}, {D}] as the cache, got {tuple(key.shape)}")
    _tensors("value", value, cache._key.dtype, 4, key.shape, dev)
    _table(page_table, B, cache)
    _int32("start", start, (B,), cache)
    if counts is not None:
        _int32("counts", counts, (B,), cache)
    if query is not None:
        _tensors("query", query, cache._key.dtype, 4, None, dev)
        if tuple(query.shape[:2]) != (B, N) or query.shape[3] != D:
            raise RuntimeError(f"query must be [{B}, {N}, H, {D}], got {tuple(query.shape)}")


def paged_append(cache: PagedCache, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor,
                 start: torch.Tensor, counts: Optional[torch.Tensor] = None, rotation: Optional[Rotation] = None,
                 query: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Appends key/value [B, N, Hkv, D] to the streams of page_table [B, width]:
    row (b, i) becomes token start[b] + i of stream b, for i < counts[b] (None:
    all N; rows behind are not stored).  ``rotation`` turns the keys, and the
    rows of query [B, N, H, D] into the returned tensor, by those positions.

    A token whose page lies outside the table or the cache is dropped; a
    negative start counts as 0.  With cache.key_sums, the sums of the pages that
    receive tokens are renewed from their stored keys.  Two streams that share
    a page may read it, not append to it in one call.
    """
    _check_cache(cache)
    ck = cache._key
    dev = ck.get_device()
    q = key if query is None else query
    n = start if counts is None else counts
    if not (_valid(ck.dtype, dev, key, value, q) and _valid(torch.int32, dev, page_table, start, n)
            and key.dim() == 4 and q.dim() == 4 and page_table.dim() == 2 and start.dim() == 1
            and value.shape == key.shape and n.shape == start.shape
            and key.shape[2:] == ck.shape[2:] and (q is key or (q.shape[:2] == key.shape[:2] and q.shape[3] == ck.shape[3]))
            and page_table.shape[0] == start.shape[0] == key.shape[0]):
        _check_append(cache, key, value, page_table, start, counts, query)
    B, N, Hkv, D = key.shape
    H = q.shape[2]
    out = torch.empty_like(query) if query is not None else None
    freq, kw = None, {}
    if rotation is not None:
        if not isinstance(rotation, Rotation):
            raise RuntimeError("rotation must be a Rotation")
        if rotation.dim > D:
            raise RuntimeError(f"rotation dim ({rotation.dim}) exceeds head_dim ({D})")
        if rotation.inv_freq.device != ck.device:
            raise RuntimeError("rotation is on another device than the cache")
        freq, kw = rotation.inv_freq, dict(rotary_dim=rotation.dim, interleaved=int(rotation.interleaved))
    width = page_table.shape[1]
    d, _ = _desc(cache, ("append", B, N, H, width, *kw.values()), B, H, width, num_tokens=N, **kw)
    _call(_lib.ma_paged_append, dev, ctypes.byref(d), key.data_ptr(), value.data_ptr(), _ptr(query),
          _ptr(out), cache._key.data_ptr(), cache._value.data_ptr(), _ptr(cache._sums), page_table.data_ptr(),
          start.data_ptr(), _ptr(counts), _ptr(freq))
    return out


def _query(query, cache, page_table, lengths):
    _check_cache(cache)
    ck = cache._key
    dev = ck.get_device()
    if not (_valid(ck.dtype, dev, query) and _valid(torch.int32, dev, page_table, lengths) and query.dim() == 3
            and page_table.dim() == 2 and lengths.dim() == 1 and query.shape[2] == ck.shape[3]
            and page_table.shape[0] == lengths.shape[0] == query.shape[0]):
        _tensors("query", query, ck.dtype, 3, None, ck.device)
        if query.shape[2] != ck.shape[3]:
            raise RuntimeError(f"query head_dim ({query.shape[2]}) must be the cache's ({ck.shape[3]})")
        _table(page_table, query.shape[0], cache)
        _int32("lengths", lengths, (query.shape[0],), cache)
    return query.shape


def paged_decode(query: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                 left: Optional[int] = None, num_global: int = 0, pages: Optional[torch.Tensor] = None,
                 scale=None, return_lse: bool = False):
    """Attention of one token per stream, query [B, H, D], over the first
    lengths[b] tokens of stream b (its own among them) -> [B, H, D].

    left: only the keys [len-1-left, len-1], and with num_global also the first
    num_global tokens.  pages: int32 [B, Hkv, S], S <= 64, the logical pages each
    key/value head's queries read instead (paged_select; entries that are
    negative or behind the last page are skipped, repeats count once).  A query
    without keys gives zeros.  return_lse: also float32 [B, H], log2 of the sum
    of exp(scaled scores) (-inf without keys).  scale: softmax scale (None:
    1/sqrt(head_dim)).
    """
    B, H, D = _query(query, cache, page_table, lengths)
    S, num_global = 0, int(num_global)
    if left is not None:
        left = int(left)
        if left < 0:
            raise RuntimeError("left must be >= 0")
    if num_global < 0 or (num_global > 0 and left is None):
        raise RuntimeError("num_global must be >= 0 and goes with left")
    if pages is not None:
        if left is not None:
            raise RuntimeError("pages and left exclude each other")
        _tensors("pages", pages, torch.int32, 3, None, cache._key.device)
        S = pages.shape[2]
        if pages.shape[:2] != (B, cache._key.shape[2]) or not 1 <= S <= 64:
            raise RuntimeError(f"pages must be [{B}, {cache._key.shape[2]}, S] with 1 <= S <= 64, "
                               f"got {tuple(pages.shape)}")
    kw = _ext._scale_kw(scale)
    width = page_table.shape[1]
    d, nbytes = _desc(cache, ("decode", B, H, width, left, num_global, S, kw.get("scale")), B, H, width,
                      _lib.ma_paged_decode_workspace_size, left=-1 if left is None else min(left, 1 << 62),
                      num_global=min(num_global, 1 << 62), num_selected=S, **kw)
    out = torch.empty_like(query)
    lse = torch.empty((B, H), dtype=torch.float32, device=query.device) if return_lse else None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device) if nbytes else None
    _call(_lib.ma_paged_decode, query.get_device(), ctypes.byref(d), query.data_ptr(), cache._key.data_ptr(),
          cache._value.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), _ptr(pages), out.data_ptr(), _ptr(lse),
          _ptr(ws), nbytes)
    return (out, lse) if return_lse else out


def paged_select(query: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                 num_selected: int, first_pages: int = 0, local_pages: int = 1) -> torch.Tensor:
    """The num_selected (at most 64) pages whose mean key has the largest dot
    product with the sum of a key/value head's queries -> int32 [B, Hkv,
    num_selected] logical pages, ascending, -1 behind them.

    The first ``first_pages`` and the newest ``local_pages`` (>= 1) pages are
    always listed.  Scores are float64 over cache.key_sums; ties go to the lower
    page and NaN scores rank last.  At most 16384 pages a stream.
    """
    B, H, D = _query(query, cache, page_table, lengths)
    if cache._sums is None:
        raise RuntimeError("paged_select needs a cache with key_sums")
    S, first, local = int(num_selected), int(first_pages), int(local_pages)
    if not 1 <= S <= 64:
        raise RuntimeError("num_selected must be in [1, 64]")
    if first < 0 or local < 1 or first + local > S:
        raise RuntimeError("first_pages >= 0 and local_pages >= 1 must fit in num_selected")
    width = page_table.shape[1]
    d, _ = _desc(cache, ("select", B, H, width, S, first, local), B, H, width, num_selected=S, first_pages=first,
                 local_pages=local)
    out = torch.empty((B, cache._key.shape[2], S), dtype=torch.int32, device=query.device)
    _call(_lib.ma_paged_select, query.get_device(), ctypes.byref(d), query.data_ptr(), cache._sums.data_ptr(),
          page_table.data_ptr(), lengths.data_ptr(), out.data_ptr())
    return out
