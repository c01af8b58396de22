"""Language-model operators over device tensors: rotary positions with several
axes, a paged key/value cache held in 8 bits, and the attention over it
(include/infvino_b200.h, ivc_kv_*), for a decoder behind a `PlanModel`.

Tensors are anything with torch's `data_ptr()`, `shape`, `stride()`, `dim()`,
`is_contiguous()`, `get_device()` and `dtype`, on the handle's device; this module itself needs no torch.
Streams are `cudaStream_t` values as integers (0: the default stream).
"""
from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence

from . import _native
from ._native import NativeError, lib

__all__ = ["KvOps", "KvCache", "Rotary"]

BLOCK = 16  # tokens that share a scale (IVC_KV_BLOCK)
_DTYPES = {"float16": 0, "bfloat16": 1}
_names: dict = {}  # dtype object -> its name


def _name(t) -> str:
    n = _names.get(t.dtype)
    if n is None:
        n = _names[t.dtype] = str(t.dtype).rsplit(".", 1)[-1]
    return n


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(t, name: str, dtype: str, shape, device: int) -> bytes:
    """ivc_rows of a [tokens, heads, head_dim] tensor whose last dimension is dense."""
    st = t.stride()
    if t.shape != shape or _name(t) != dtype or st[2] != 1 or t.get_device() != device:
        _need(t.get_device() == device, f"{name}: expected a tensor on CUDA device {device}")
        _need(len(t.shape) == 3, f"{name}: expected [tokens, heads, head_dim], got shape {tuple(t.shape)}")
        _need(_name(t) == dtype, f"{name}: expected {dtype}, got {t.dtype}")
        _need(tuple(t.shape) == tuple(shape), f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
        raise ValueError(f"{name}: the last dimension must be dense")
    return _native.ROWS.pack(t.data_ptr(), st[0], st[1])


def _kind(t, name: str) -> str:
    """The dtype of a call, by its first tensor [tokens, heads, head_dim]."""
    n = _name(t)
    if n not in _DTYPES or t.dim() != 3:
        raise ValueError(f"{name}: expected float16 or bfloat16 [tokens, heads, head_dim], got {t.dtype} {tuple(t.shape)}")
    return n


def _dense(t, name: str, dtype: str, rank: int, device=None) -> int:
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name}: expected a tensor on CUDA device {device}")
    if (_names.get(t.dtype) or _name(t)) != dtype or t.dim() != rank or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of rank {rank}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


class Rotary:
    """How heads are turned: `table` [positions, pairs, 2] float32 (cosine and
    sine of each position's angle for each pair) and the axis of each pair."""

    def __init__(self, table, axis_of: Optional[Sequence[int]] = None, interleaved: bool = False):
        self._table = _dense(table, "table", "float32", 3)
        self.positions, self.pairs, two = table.shape
        if two != 2 or (axis_of is not None and len(axis_of) != self.pairs):
            raise ValueError("table: expected [positions, pairs, 2], axis_of: one axis for each pair")
        self.interleaved = int(interleaved)
        self.table, self.device = table, table.get_device()
        self.axes, self._axis_ptr = 1, 0
        if axis_of is not None:
            self._axis_of = array("B", axis_of)
            self._axis_ptr = self._axis_of.buffer_info()[0]
            self.axes = max(self._axis_of) + 1

    def at(self, pos, tokens: int, device: int) -> bytes:
        """ivc_rotary for positions [axes, tokens] (or [tokens] for one axis)."""
        if self.device != device or pos.get_device() != device:
            raise ValueError(f"rotary table and pos: expected tensors on CUDA device {device}")
        sh, st = pos.shape, pos.stride()
        two = len(sh) == 2
        if not 1 <= len(sh) <= 2 or sh[-1] != tokens or _name(pos) != "int32" or (st[-1] != 1 and tokens > 1):
            raise ValueError(f"pos: expected int32 [axes, {tokens}] with dense tokens, got {pos.dtype} {tuple(sh)}")
        axes = sh[0] if two else 1
        if axes < self.axes:
            raise ValueError(f"pos: {axes} axes, but axis_of names {self.axes}")
        return _native.ROTARY.pack(self._table, self.positions, self.pairs, axes, self.interleaved, pos.data_ptr(), st[0] if two else 0,
                                   self._axis_ptr)


class KvCache:
    """One layer's cache over the caller's tensors: k, v int8 [pages, kv_heads,
    page_size, head_dim], k_scale, v_scale float32 [pages, kv_heads,
    page_size / 16]; a value is code * scale."""

    def __init__(self, k, v, k_scale, v_scale):
        ptrs = (_dense(k, "k", "int8", 4), _dense(v, "v", "int8", 4), _dense(k_scale, "k_scale", "float32", 3),
                _dense(v_scale, "v_scale", "float32", 3))
        self.pages, self.kv_heads, self.page_size, self.head_dim = shape = k.shape
        _need(v.shape == shape, "v: expected k's shape")
        want = (self.pages, self.kv_heads, self.page_size // BLOCK)
        _need(k_scale.shape == want and v_scale.shape == want, f"scales: expected shape {want}")
        self.device = k.get_device()
        if not self.device == v.get_device() == k_scale.get_device() == v_scale.get_device():
            raise ValueError("the cache's tensors are on different devices")
        self._keep = (k, v, k_scale, v_scale)
        self._c = _native.KV_CACHE.pack(*ptrs, self.pages, self.page_size, self.kv_heads, self.head_dim)


class KvOps:
    """A handle of the operators on one CUDA device."""

    def __init__(self, device: int = 0):
        L = lib()
        h = ctypes.c_void_p()
        st = L.ivc_kv_create(int(device), ctypes.byref(h))
        if st != 0:
            raise NativeError(st, (L.ivc_kv_last_error(None) or b"").decode())
        self._h, self._L = h, L
        self._rope, self._append, self._read, self._attend = L.ivc_kv_rope, L.ivc_kv_append, L.ivc_kv_read, L.ivc_kv_attend
        self.device = device

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            self._L.ivc_kv_destroy(h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _fail(self, status: int) -> None:
        if not self._h:
            raise ValueError("the handle is closed")
        raise NativeError(status, (self._L.ivc_kv_last_error(self._h) or b"").decode())

    def _check(self, status: int) -> None:
        if status != 0:
            self._fail(status)

    def synchronize(self, stream: int = 0) -> None:
        """Waits for the stream; raises NativeError (KERNEL) if a kernel met
        page numbers, lengths or positions that do not fit."""
        self._check(self._L.ivc_kv_synchronize(self._h, stream))

    def reserve(self, stream: int = 0) -> None:
        """Allocates the stream's attention workspace, as its first `attend` would (needed before a graph capture)."""
        self._check(self._L.ivc_kv_reserve(self._h, stream))

    def release(self, stream: int = 0) -> None:
        """Waits for the stream and frees its attention workspace (some 40 MB), before the stream is destroyed or
        when it is not used any more; graphs captured on it must not be replayed afterwards."""
        self._check(self._L.ivc_kv_release(self._h, stream))

    def rope_table(self, inv_freq: Sequence[float], table, stream: int = 0) -> None:
        """Fills `table` [positions, pairs, 2] with the angles position * inv_freq[pair]."""
        ptr = _dense(table, "table", "float32", 3, self.device)
        pairs = table.shape[1]
        _need(len(inv_freq) == pairs and table.shape[2] == 2, "table: expected [positions, len(inv_freq), 2]")
        f = (ctypes.c_double * pairs)(*inv_freq)
        self._check(self._L.ivc_kv_rope_table(self._h, f, pairs, table.shape[0], ptr, stream))

    def rope(self, x, out, rotary: Rotary, pos, stream: int = 0) -> None:
        """out [tokens, heads, head_dim] = x turned; out may be x."""
        name, sh, d = _kind(x, "x"), x.shape, self.device
        st = self._rope(self._h, _DTYPES[name], *sh, _rows(x, "x", name, sh, d), _rows(out, "out", name, sh, d), rotary.at(pos, sh[0], d),
                        stream)
        if st:
            self._fail(st)

    def _seqs(self, tokens: int, cache: KvCache, offsets, at, pages) -> bytes:
        d = self.device
        if cache.device != d:
            raise ValueError(f"cache: expected tensors on CUDA device {d}")
        o, a = _dense(offsets, "offsets", "int32", 1, d), _dense(at, "starts / lens", "int32", 1, d)
        p = _dense(pages, "pages", "int32", 2, d)
        batch, width = pages.shape
        if offsets.shape[0] != batch + 1 or at.shape[0] != batch:
            raise ValueError("offsets: batch + 1 entries, starts / lens: batch, pages: batch rows")
        return _native.KV_SEQS.pack(batch, tokens, o, a, p, width)

    def append(self, cache: KvCache, k, v, offsets, starts, pages, rotary: Optional[Rotary] = None, pos=None, q=None, q_out=None,
               stream: int = 0) -> None:
        """Appends k (turned by `rotary` at `pos`) and v [tokens, kv_heads,
        head_dim]: sequence b's tokens offsets[b] .. offsets[b + 1] - 1 go to
        cache positions starts[b] and on.  With q, q_out [tokens, q_heads,
        head_dim] turned in the same launch."""
        name, tokens, d = _kind(k, "k"), k.shape[0], self.device
        sh = (tokens, cache.kv_heads, cache.head_dim)
        _need((rotary is None) == (pos is None), "rotary and pos go together")
        _need((q is None) == (q_out is None), "q and q_out go together")
        rot = rotary.at(pos, tokens, d) if rotary is not None else None
        heads, qr, qo = 0, None, None
        if q is not None:
            _need(q.dim() == 3, "q: expected [tokens, heads, head_dim]")
            heads = q.shape[1]
            qsh = (tokens, heads, cache.head_dim)
            qr, qo = _rows(q, "q", name, qsh, d), _rows(q_out, "q_out", name, qsh, d)
        st = self._append(self._h, cache._c, self._seqs(tokens, cache, offsets, starts, pages), _DTYPES[name], _rows(k, "k", name, sh, d),
                          _rows(v, "v", name, sh, d), rot, heads, qr, qo, stream)
        if st:
            self._fail(st)

    def read(self, cache: KvCache, k, v, offsets, starts, pages, stream: int = 0) -> None:
        """The cache's values of positions starts[b] and on into k and v (either may be None)."""
        some = k if k is not None else v
        _need(some is not None, "read: k or v")
        name, tokens, d = _kind(some, "k or v"), some.shape[0], self.device
        sh = (tokens, cache.kv_heads, cache.head_dim)
        kr = _rows(k, "k", name, sh, d) if k is not None else None
        vr = _rows(v, "v", name, sh, d) if v is not None else None
        st = self._read(self._h, cache._c, self._seqs(tokens, cache, offsets, starts, pages), _DTYPES[name], kr, vr, stream)
        if st:
            self._fail(st)

    def attend(self, cache: KvCache, q, out, offsets, lens, pages, max_new: int, scale: Optional[float] = None, window: int = 0,
               sinks: int = 0, stream: int = 0) -> None:
        """out [tokens, q_heads, head_dim] = causal attention of q over the
        cache: lens[b] tokens in it, the call's own (the last ones) included.
        window > 0: a query sees its last `window` keys and the first `sinks`."""
        name, sh, d = _kind(q, "q"), q.shape, self.device
        tokens, heads, dim = sh
        if dim != cache.head_dim:
            raise ValueError(f"q: expected head_dim {cache.head_dim}, got {dim}")
        st = self._attend(self._h, cache._c, self._seqs(tokens, cache, offsets, lens, pages), _DTYPES[name], heads, max_new,
                          _rows(q, "q", name, sh, d), _rows(out, "out", name, sh, d), dim ** -0.5 if scale is None else scale, window, sinks,
                          stream)
        if st:
            self._fail(st)
