"""Language-model operators over device tensors: rotary positions with several
axes, a paged key/value cache held in 8 bits, and the attention over it
(include/infvino_b200.h, ivc_kv_*), for a decoder behind a `PlanModel`.

Tensors are anything with `data_ptr()`, `shape`, `stride()` and `dtype` in
torch's sense, on the handle's device; this module itself needs no torch.
Streams are `cudaStream_t` values as integers (0: the default stream).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

from . import _native
from ._native import NativeError, lib

__all__ = ["KvOps", "KvCache", "Rotary"]

BLOCK = 16  # tokens that share a scale (IVC_KV_BLOCK)
_DTYPES = {"float16": 0, "bfloat16": 1}


def _dtype_name(t) -> str:
    return str(t.dtype).rsplit(".", 1)[-1]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(t, name: str, dtype: str, shape=None) -> _native.Rows:
    """A [tokens, heads, head_dim] tensor whose last dimension is dense."""
    sh, st = t.shape, t.stride()
    if len(sh) != 3 or (st[2] != 1 and sh[2] != 1) or _dtype_name(t) != dtype or (shape is not None and tuple(sh) != shape):
        _need(len(sh) == 3, f"{name}: expected [tokens, heads, head_dim], got shape {tuple(sh)}")
        _need(_dtype_name(t) == dtype, f"{name}: expected {dtype}, got {t.dtype}")
        _need(shape is None or tuple(sh) == shape, f"{name}: expected shape {shape}, got {tuple(sh)}")
        raise ValueError(f"{name}: the last dimension must be dense")
    return _native.Rows(t.data_ptr(), st[0], st[1])


def _dense(t, name: str, dtype: str, rank: int):
    if _dtype_name(t) != dtype or len(t.shape) != rank or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of rank {rank}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


class Rotary:
    """How heads are turned: `table` [positions, pairs, 2] float32 (cosine and
    sine of each position's angle for each pair) and the axis of each pair."""

    def __init__(self, table, axis_of: Optional[Sequence[int]] = None, interleaved: bool = False):
        ptr = _dense(table, "table", "float32", 3)
        positions, self.pairs, two = table.shape
        _need(two == 2, "table: expected [positions, pairs, 2]")
        _need(axis_of is None or len(axis_of) == self.pairs, "axis_of: expected one axis for each pair")
        self.axes = 1 if axis_of is None else max(axis_of) + 1
        self._axis_of = bytes(axis_of) if axis_of is not None else None
        self.table = table  # keeps the memory alive
        self._c = _native.Rotary(ptr, positions, self.pairs, 0, int(interleaved), None, 0, self._axis_of)

    def at(self, pos, tokens: int) -> _native.Rotary:
        """The C struct for positions [axes, tokens] (or [tokens] for one axis)."""
        sh, st = pos.shape, pos.stride()
        two = len(sh) == 2
        if _dtype_name(pos) != "int32" or len(sh) not in (1, 2) or sh[-1] != tokens or (st[-1] != 1 and tokens > 1):
            raise ValueError(f"pos: expected int32 [axes, {tokens}] with dense tokens, got {pos.dtype} {tuple(sh)}")
        axes = sh[0] if two else 1
        _need(axes >= self.axes, f"pos: {axes} axes, but axis_of names {self.axes}")
        c = self._c
        return _native.Rotary(c.table, c.positions, c.pairs, axes, c.interleaved, pos.data_ptr(), st[0] if two else 0, self._axis_of)


class KvCache:
    """One layer's cache over the caller's tensors: k, v int8 [pages, kv_heads,
    page_size, head_dim], k_scale, v_scale float32 [pages, kv_heads,
    page_size / 16]; a value is code * scale."""

    def __init__(self, k, v, k_scale, v_scale):
        kp, vp = _dense(k, "k", "int8", 4), _dense(v, "v", "int8", 4)
        ks, vs = _dense(k_scale, "k_scale", "float32", 3), _dense(v_scale, "v_scale", "float32", 3)
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        _need(tuple(v.shape) == tuple(k.shape), "v: expected k's shape")
        want = (self.pages, self.kv_heads, self.page_size // BLOCK)
        _need(tuple(k_scale.shape) == want and tuple(v_scale.shape) == want, f"scales: expected shape {want}")
        self._keep = (k, v, k_scale, v_scale)
        self._c = _native.KvCache(kp, vp, ks, vs, self.pages, self.page_size, self.kv_heads, self.head_dim)


class KvOps:
    """A handle of the operators on one CUDA device."""

    def __init__(self, device: int = 0):
        L = lib()
        h = ctypes.c_void_p()
        st = L.ivc_kv_create(int(device), ctypes.byref(h))
        if st != 0:
            raise NativeError(st, (L.ivc_kv_last_error(None) or b"").decode())
        self._h, self._L = h, L
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

    def _check(self, status: int) -> None:
        if status != 0:
            raise NativeError(status, (self._L.ivc_kv_last_error(self._h) or b"").decode())

    def synchronize(self, stream: int = 0) -> None:
        """Waits for the stream; raises NativeError (KERNEL) if a kernel met
        page numbers, lengths or positions that do not fit."""
        self._check(self._L.ivc_kv_synchronize(self._h, stream))

    def reserve(self, stream: int = 0) -> None:
        """Allocates the stream's attention workspace, as its first `attend` would (needed before a graph capture)."""
        self._check(self._L.ivc_kv_reserve(self._h, stream))

    def rope_table(self, inv_freq: Sequence[float], table, stream: int = 0) -> None:
        """Fills `table` [positions, pairs, 2] with the angles position * inv_freq[pair]."""
        ptr = _dense(table, "table", "float32", 3)
        pairs = table.shape[1]
        _need(len(inv_freq) == pairs and table.shape[2] == 2, "table: expected [positions, len(inv_freq), 2]")
        f = (ctypes.c_double * pairs)(*inv_freq)
        self._check(self._L.ivc_kv_rope_table(self._h, f, pairs, table.shape[0], ptr, stream))

    def rope(self, x, out, rotary: Rotary, pos, stream: int = 0) -> None:
        """out [tokens, heads, head_dim] = x turned; out may be x."""
        name, sh = _dtype_name(x), tuple(x.shape)
        _need(name in _DTYPES, f"x: expected float16 or bfloat16, got {x.dtype}")
        xr, yr = _rows(x, "x", name), _rows(out, "out", name, sh)
        rot = rotary.at(pos, sh[0])
        self._check(self._L.ivc_kv_rope(self._h, _DTYPES[name], *sh, ctypes.byref(xr), ctypes.byref(yr), ctypes.byref(rot), stream))

    def _seqs(self, tokens: int, offsets, at, pages) -> _native.KvSeqs:
        o, a, p = _dense(offsets, "offsets", "int32", 1), _dense(at, "starts / lens", "int32", 1), _dense(pages, "pages", "int32", 2)
        batch, sh = at.shape[0], pages.shape
        _need(offsets.shape[0] == batch + 1 and sh[0] == batch, "offsets: batch + 1 entries, pages: batch rows")
        return _native.KvSeqs(batch, tokens, o, a, p, sh[1])

    def append(self, cache: KvCache, k, v, offsets, starts, pages, rotary: Optional[Rotary] = None, pos=None, q=None, q_out=None,
               stream: int = 0) -> None:
        """Appends k (turned by `rotary` at `pos`) and v [tokens, kv_heads,
        head_dim]: sequence b's tokens offsets[b] .. offsets[b + 1] - 1 go to
        cache positions starts[b] and on.  With q, q_out [tokens, q_heads,
        head_dim] turned in the same launch."""
        name, tokens = _dtype_name(k), k.shape[0]
        _need(name in _DTYPES, f"k: expected float16 or bfloat16, got {k.dtype}")
        sh = (tokens, cache.kv_heads, cache.head_dim)
        kr, vr, s = _rows(k, "k", name, sh), _rows(v, "v", name, sh), self._seqs(tokens, offsets, starts, pages)
        _need((rotary is None) == (pos is None), "rotary and pos go together")
        rot = ctypes.byref(rotary.at(pos, tokens)) if rotary is not None else None
        heads, qr, qo = 0, None, None
        if q is not None:
            heads = q.shape[1]
            sh = (tokens, heads, cache.head_dim)
            qr, qo = ctypes.byref(_rows(q, "q", name, sh)), ctypes.byref(_rows(q_out, "q_out", name, sh))
        self._check(self._L.ivc_kv_append(self._h, ctypes.byref(cache._c), ctypes.byref(s), _DTYPES[name], ctypes.byref(kr), ctypes.byref(vr),
                                          rot, heads, qr, qo, stream))

    def read(self, cache: KvCache, k, v, offsets, starts, pages, stream: int = 0) -> None:
        """The cache's values of positions starts[b] and on into k and v (either may be None)."""
        some = k if k is not None else v
        _need(some is not None, "read: k or v")
        name, tokens = _dtype_name(some), some.shape[0]
        _need(name in _DTYPES, f"expected float16 or bfloat16, got {some.dtype}")
        sh = (tokens, cache.kv_heads, cache.head_dim)
        kr = ctypes.byref(_rows(k, "k", name, sh)) if k is not None else None
        vr = ctypes.byref(_rows(v, "v", name, sh)) if v is not None else None
        s = self._seqs(tokens, offsets, starts, pages)
        self._check(self._L.ivc_kv_read(self._h, ctypes.byref(cache._c), ctypes.byref(s), _DTYPES[name], kr, vr, stream))

    def attend(self, cache: KvCache, q, out, offsets, lens, pages, max_new: int, scale: Optional[float] = None, window: int = 0,
               sinks: int = 0, stream: int = 0) -> None:
        """out [tokens, q_heads, head_dim] = causal attention of q over the
        cache: lens[b] tokens in it, the call's own (the last ones) included.
        window > 0: a query sees its last `window` keys and the first `sinks`."""
        name, sh = _dtype_name(q), tuple(q.shape)
        _need(name in _DTYPES, f"q: expected float16 or bfloat16, got {q.dtype}")
        qr, yr = _rows(q, "q", name), _rows(out, "out", name, sh)
        _need(sh[2] == cache.head_dim, f"q: expected head_dim {cache.head_dim}, got {sh[2]}")
        s = self._seqs(sh[0], offsets, lens, pages)
        self._check(self._L.ivc_kv_attend(self._h, ctypes.byref(cache._c), ctypes.byref(s), _DTYPES[name], sh[1], max_new, ctypes.byref(qr),
                                          ctypes.byref(yr), sh[2] ** -0.5 if scale is None else scale, window, sinks, stream))
