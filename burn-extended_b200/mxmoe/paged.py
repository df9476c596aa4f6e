"""A paged key-value cache over the C ABI (`mxmqa_paged_*`, `mxmqa_rotary*` in
include/mxmoe.h): many sequences share one pool of pages.

    rotary = RotaryTable.of(RotaryConfig(64, scaling="yarn", scaling_factor=32.0), 131072)
    cache = PagedKvCache(n_pages=4096, page_size=16, n_heads=64, kv_heads=8, head_dim=64, track=True)
    q = cache.append(q, k, v, tables, index, rotary)     # new tokens: rotate, write K and V
    out = cache.decode(q, tables, lens, track=True)      # one new token per row attends
    lens = cache.evict(tables, lens, seen, budget=2048)  # least weight leaves

`tables` [rows, max_pages] int32 names each row's pages; cache index n is slot
n % page_size of tables[row, n // page_size].  Which pages are free is the
caller's book-keeping.  PyTorch provides device memory and streams only; every
call runs on the current stream of the cache's device, and a cache serves one
stream at a time.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from ._lib import (E4M3, BF16, F32, MxMoeError, PagedAppendArgs, PagedBuffers, PagedConfig, PagedDecodeArgs,
                   PagedEvictArgs, RotaryArgs, RotaryTableConfig, check, lib)

_ACT = {torch.float32: F32, torch.bfloat16: BF16}
_CACHE = {torch.float32: F32, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3}
_MOST = (1 << 32) - 1  # of a count in the C structs: ctypes would wrap a larger one around
_SCALING = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3, "streaming": 4}


def _bad(msg: str):
    raise MxMoeError(1, msg)


def _act(name: str, t) -> int:
    code = _ACT.get(t.dtype)
    if code is None:
        _bad(f"{name}: unsupported dtype {t.dtype} (float32 or bfloat16)")
    return code


def _heads(name: str, t, shape, device):
    """A tensor of `shape` [n, heads, head_dim] with contiguous columns -> strides of the first two dimensions."""
    if t.shape != shape or t.device != device:
        _bad(f"{name}: expected a tensor {list(shape)} on {device}, got {tuple(t.shape)} on {t.device}")
    a, b, c = t.stride()
    if c != 1 and shape[2] > 1:
        _bad(f"{name}: the columns of a head must be contiguous")
    return a, b


def _ints(name: str, t, n: int, device) -> int:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device or (n > 1 and t.stride(0) != 1):
        _bad(f"{name}: expected {n} contiguous int32 on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


@dataclass
class RotaryConfig:
    """Frequencies theta^(-2i / rot_dim) of the leading rot_dim columns of a head.

    scaling: "plain"; "linear" (divided by scaling_factor); "ntk" (base x
    scaling_factor^(rot_dim / (rot_dim - 2))); "yarn" (pairs of less than
    ntk_alpha turns within initial_context are divided, those of more than
    ntk_beta kept, a ramp between; cos and sin x (0.1 ln scaling_factor + 1));
    "streaming" (as StreamingMultiQueryAttention.set_rope scales,
    src/rope/mod.rs:11-50)."""
    rot_dim: int
    theta: float = 150000.0
    scaling: str = "plain"
    scaling_factor: float = 1.0
    initial_context: float = 4096.0
    ntk_alpha: float = 1.0
    ntk_beta: float = 32.0


class RotaryTable:
    """cos and sin by position, float32 [n_positions, rot_dim / 2] on the device.

    interleaved: pairs (2i, 2i + 1) rotate together instead of (i, i + rot_dim / 2)."""

    def __init__(self, cos, sin, interleaved: bool = False):
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or not t.is_cuda or t.shape != cos.shape \
                    or t.device != cos.device:
                _bad(f"{name}: expected contiguous float32 [n_positions, rot_dim / 2] on the device")
        self.cos, self.sin, self.interleaved = cos, sin, bool(interleaved)
        self.n_positions, self.rot_dim, self.device = cos.shape[0], 2 * cos.shape[1], cos.device
        self._ptrs = cos.data_ptr(), sin.data_ptr(), self.rot_dim, self.n_positions, int(self.interleaved)

    @staticmethod
    def of(cfg: RotaryConfig, n_positions: int, interleaved: bool = False, device: int = 0) -> "RotaryTable":
        if cfg.scaling not in _SCALING:
            _bad(f"scaling {cfg.scaling!r}: expected one of {sorted(_SCALING)}")
        if not 0 < cfg.rot_dim <= _MOST or not 0 < n_positions <= _MOST:
            _bad("rot_dim and n_positions must be positive and below 2^32")
        dev = torch.device("cuda", device)
        cos, sin = (torch.empty(n_positions, cfg.rot_dim // 2, device=dev) for _ in range(2))
        c = RotaryTableConfig(cfg.rot_dim, _SCALING[cfg.scaling], cfg.theta, cfg.scaling_factor, cfg.initial_context,
                              cfg.ntk_alpha, cfg.ntk_beta)
        check(lib().mxmqa_rotary_table(ctypes.byref(c), 0, n_positions, cos.data_ptr(), sin.data_ptr(), device,
                                       _stream(dev)))
        return RotaryTable(cos, sin, interleaved)

    def apply(self, x, positions, inverse: bool = False, out=None):
        """x [tokens, heads, head_dim] turned to `positions` [tokens] int32; `inverse` turns back, and is the
        gradient towards x.  out may be x."""
        if x.dim() != 3:
            _bad(f"x: expected [tokens, heads, head_dim], got {tuple(x.shape)}")
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
        if out.dtype != x.dtype or out.shape != x.shape:
            _bad("out: expected x's shape and dtype")
        n, heads, hd = x.shape
        xs, os = _heads("x", x, x.shape, self.device), _heads("out", out, x.shape, self.device)
        a = RotaryArgs(x.data_ptr(), *xs, out.data_ptr(), *os, _act("x", x), n, heads, hd,
                       _ints("positions", positions, n, self.device), *self._ptrs, int(inverse), self.device.index)
        check(lib().mxmqa_rotary(ctypes.byref(a), _stream(self.device)))
        return out


class PagedKvCache:
    """Keys and values [n_pages, kv_heads, page_size, head_dim] of many sequences.

    dtype: torch.float32, torch.bfloat16 or torch.float8_e4m3fn; an 8-bit key
    stands for its code times k_scale[kv_head], a value for v_scale's.  track:
    the cache also keeps every token's accumulated attention weight and position
    [n_pages, kv_heads, page_size], which `evict` goes by, and a workspace of 32 bytes for every token, key head and
    8 query heads that read it."""

    def __init__(self, n_pages: int, page_size: int, n_heads: int, kv_heads: int, head_dim: int,
                 dtype=torch.bfloat16, track: bool = False, k_scale=None, v_scale=None, device: int = 0):
        dev = torch.device("cuda", device)
        if min(n_pages, page_size, kv_heads, head_dim) <= 0:
            _bad("zero dimension")
        shape = (n_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2))
        weight = torch.zeros(shape[:3], device=dev) if track else None
        position = torch.zeros(shape[:3], dtype=torch.int32, device=dev) if track else None
        self._open(k, v, n_heads, weight, position, k_scale, v_scale)

    @classmethod
    def over(cls, k, v, n_heads: int, weight=None, position=None, k_scale=None, v_scale=None) -> "PagedKvCache":
        """A cache over tensors that the caller has; their contents stay."""
        self = cls.__new__(cls)
        self._open(k, v, n_heads, weight, position, k_scale, v_scale)
        return self

    def _open(self, k, v, n_heads, weight, position, k_scale, v_scale):
        self._h, self._lib = None, lib()
        if k.dtype not in _CACHE:
            _bad(f"unsupported cache dtype {k.dtype} (float32, bfloat16 or float8_e4m3fn)")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
            _bad("k and v: expected [n_pages, kv_heads, page_size, head_dim] of one dtype")
        n_pages, kv_heads, page_size, head_dim = k.shape
        for name, t, dt, shape in (("k", k, k.dtype, k.shape), ("v", v, k.dtype, k.shape),
                                   ("weight", weight, torch.float32, k.shape[:3]),
                                   ("position", position, torch.int32, k.shape[:3]),
                                   ("k_scale", k_scale, torch.float32, (kv_heads,)),
                                   ("v_scale", v_scale, torch.float32, (kv_heads,))):
            if t is not None and (t.dtype != dt or tuple(t.shape) != tuple(shape) or not t.is_contiguous()
                                  or not t.is_cuda or t.device != k.device):
                _bad(f"{name}: expected contiguous {dt} {tuple(shape)} on the cache's device")
        if not 0 <= n_heads <= _MOST:
            _bad("n_heads must not be negative nor reach 2^32")
        self.k, self.v, self.weight, self.position = k, v, weight, position
        self.k_scale, self.v_scale = k_scale, v_scale
        self.n_pages, self.page_size, self.n_heads = n_pages, page_size, n_heads
        self.kv_heads, self.head_dim, self.device = kv_heads, head_dim, k.device

        def ptr(t):
            return None if t is None else t.data_ptr()

        cfg = PagedConfig(n_pages, page_size, n_heads, kv_heads, head_dim, _CACHE[k.dtype], k.device.index)
        buf = PagedBuffers(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ptr(weight), ptr(position))
        h = ctypes.c_void_p()
        check(lib().mxmqa_paged_create(ctypes.byref(cfg), ctypes.byref(buf), ctypes.byref(h)))
        self._h = h

    def _tables(self, tables):
        shape = tables.shape
        if tables.dtype != torch.int32 or len(shape) != 2 or tables.device != self.device:
            _bad(f"tables: expected int32 [rows, max_pages] on {self.device}")
        stride, one = tables.stride()
        if one != 1 and shape[1] > 1:
            _bad("tables: a row must be contiguous")
        return tables.data_ptr(), stride, shape[0], shape[1]

    def append(self, q, k, v, tables, index, rotary: Optional[RotaryTable] = None, positions=None, rows=None,
               q_out=None, k_out=None):
        """New tokens enter the cache: q [tokens, n_heads, head_dim] and k are turned to their positions, k and v
        written at cache index `index` [tokens] int32 of table row `rows` [tokens] (None: token t is row t).  A
        negative index is turned but not written.  positions: None for the cache indexes.  Returns the turned
        queries (q_out, which may be q; None where q is None); k_out gets the turned keys too.  A written slot's
        weight becomes 0, its position the token's.  A position outside the rotary table keeps its token out of the
        cache; its outputs are turned as position 0."""
        n, dev, hd, dtype = k.shape[0], self.device, self.head_dim, k.dtype
        q_shape, k_shape = (n, self.n_heads, hd), (n, self.kv_heads, hd)
        ks, vs = _heads("k", k, k_shape, dev), _heads("v", v, k_shape, dev)
        code = _act("k", k)
        qs = os = kos = (0, 0)
        if v.dtype != dtype:
            _bad("v: expected k's dtype")
        if q is not None:
            qs = _heads("q", q, q_shape, dev)
            if q.dtype != dtype:
                _bad("q: expected k's dtype")
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
                os = (self.n_heads * hd, hd)
            else:
                os = _heads("q_out", q_out, q_shape, dev)
                if q_out.dtype != dtype:
                    _bad("q_out: expected q's dtype")
        elif q_out is not None:
            _bad("q_out without q")
        if k_out is not None:
            kos = _heads("k_out", k_out, k_shape, dev)
            if k_out.dtype != dtype:
                _bad("k_out: expected k's dtype")
        t, stride, n_rows, max_pages = self._tables(tables)
        if rotary is not None and rotary.device != dev:
            _bad(f"rotary: expected a table on {dev}, got {rotary.device}")
        a = PagedAppendArgs(
            None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs,
            None if q is None else q_out.data_ptr(), *os, None if k_out is None else k_out.data_ptr(), *kos, code, n,
            t, stride, n_rows, max_pages, None if rows is None else _ints("rows", rows, n, dev),
            _ints("index", index, n, dev), None if positions is None else _ints("positions", positions, n, dev),
            *((None, None, 0, 0, 0) if rotary is None else rotary._ptrs))
        check(self._lib.mxmqa_paged_append(self._h, ctypes.byref(a), _stream(dev)))
        return q_out

    def decode(self, q, tables, lens, scale: Optional[float] = None, window: int = 0, sinks=None, quiet: bool = False,
               bias=None, track: bool = False, out=None, out_dtype=None, lse=None):
        """Attention of q [rows, n_heads, head_dim], one new token per table row, over the row's first lens[row]
        cached tokens (0: zeros), the new one's among them.  window: the last `window` only.  sinks: [n_heads]
        float32 logits that join the normalizer; quiet: a 1 does.  bias: float32 [rows, n_heads or 1, length] added
        to the scores, indexes past it get none.  scale: None for 1 / sqrt(head_dim).  track: every token's share,
        summed over the heads that read its key head, is added to its weight.  lse: float32 [rows, n_heads] gets
        the log of the normalizer.  Rows may share pages, except with track."""
        dev, hd, nH = self.device, self.head_dim, self.n_heads
        n = q.shape[0]
        shape = (n, nH, hd)
        qs = _heads("q", q, shape, dev)
        t, stride, n_rows, max_pages = self._tables(tables)
        if n_rows != n:
            _bad(f"tables: expected {n} rows, got {n_rows}")
        if out is None:
            out = torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
            os = (nH * hd, hd)
        else:
            os = _heads("out", out, shape, dev)
            if out_dtype is not None and out.dtype != out_dtype:
                _bad("out: expected out_dtype")
        if sinks is not None and (sinks.dtype != torch.float32 or sinks.shape != (nH,) or sinks.device != dev
                                  or not sinks.is_contiguous()):
            _bad(f"sinks: expected contiguous float32 [{nH}] on {dev}")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != (n, nH) or lse.device != dev
                                or not lse.is_contiguous()):
            _bad(f"lse: expected contiguous float32 [{n}, {nH}] on {dev}")
        b = (None, 0, 0, 0)
        if bias is not None:
            if bias.dtype != torch.float32 or bias.dim() != 3 or bias.device != dev or bias.shape[0] not in (1, n) or \
                    bias.shape[1] not in (1, nH) or (bias.stride(2) != 1 and bias.shape[2] > 1):
                _bad(f"bias: expected float32 [{n} or 1, {nH} or 1, length] on {dev}")
            b = (bias.data_ptr(), 0 if bias.shape[0] == 1 else bias.stride(0),
                 0 if bias.shape[1] == 1 else bias.stride(1), bias.shape[2])
        if not 0 <= window <= _MOST:
            _bad("window must not be negative nor reach 2^32")
        a = PagedDecodeArgs(q.data_ptr(), *qs, out.data_ptr(), *os, None if lse is None else lse.data_ptr(),
                            _act("q", q), _act("out", out), n, max_pages, t, stride, _ints("lens", lens, n, dev),
                            1.0 / math.sqrt(hd) if scale is None else scale, window,
                            None if sinks is None else sinks.data_ptr(), *b, int(quiet), int(track))
        check(self._lib.mxmqa_paged_decode(self._h, ctypes.byref(a), _stream(dev)))
        return out

    def evict(self, tables, lens, seen, budget: int, sink: int = 4, recent: int = 0, new_lens=None):
        """Of every row with more than `budget` cached tokens the ones of least accumulated weight leave, each key
        head its own; positions below `sink` and from seen[row] - recent on stay (seen: tokens of the sequence so
        far, one above its newest position).  Survivors at cache indexes from the budget on move into the places
        below it; the row's later pages are free after that.  Returns min(lens, budget) (new_lens, which may be
        lens, but not overlap a part of it)."""
        dev = self.device
        t, stride, n, max_pages = self._tables(tables)
        if new_lens is None:
            new_lens = torch.empty_like(lens)
        if not (0 <= budget <= _MOST and 0 <= sink <= _MOST and 0 <= recent <= _MOST):
            _bad("budget, sink and recent must not be negative nor reach 2^32")
        a = PagedEvictArgs(t, stride, n, max_pages, _ints("lens", lens, n, dev), _ints("seen", seen, n, dev),
                           _ints("new_lens", new_lens, n, dev), budget, sink, recent)
        check(self._lib.mxmqa_paged_evict(self._h, ctypes.byref(a), _stream(dev)))
        return new_lens

    def sync_status(self):
        """Waits for the stream; raises if a call since the last check met a page, index, length or position out
        of range (such entries are skipped)."""
        check(lib().mxmqa_paged_status(self._h, _stream(self.device)))

    def close(self):
        if getattr(self, "_h", None):
            lib().mxmqa_paged_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
