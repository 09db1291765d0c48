"""Attention over a paged key/value cache, over libsgq.so (ctypes).

The cache of a layer is a pool of pages; a sequence's keys are in the pages that its row
of a table names, in order.  A call takes some new tokens of each of several
sequences (a prompt's chunk, single tokens, both in one batch), as rows one after the other
(inference only: nothing here has a gradient):

    PagedKV(k, v)                         a layer's pool: two tensors [pages, page, kv_heads, head_dim]
    SequenceBatch(table, lens, starts)    which rows and which pages are whose
    rotary_frequencies(dim, base)         radians a position for each pair of a head
    norm_rope_append(q, k, v, kv, batch)  norms of the heads, position rotation, keys and values into their pages
    paged_attention(q, kv, batch)         attention of the new tokens over the cache
    QuantizedAttentionInt8                norm, q/k/v, the two above and the output projection in 8 bits

Everything is float32, bfloat16 or float16, one type in a call.  The reference's attention
(include/sovereigngrad/nn.hpp:503-553) runs over the whole sequence at full width and
has none of this.  Everything runs on the device and stream of its tensors.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import load_library
from .w8a8 import (ChannelsInt8, _call, _current_device, _dtype, _vector, add_rms_norm_int8_tokens,
                   quantize_int8_channels, quantize_int8_tokens, quantized_matmul_w8a8, rms_norm_int8_tokens)

_i64 = ctypes.c_int64


class _PagedCache(ctypes.Structure):
    """sgq_paged_cache (include/sgq.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("pages", _i64), ("page_size", _i64),
                ("kv_heads", _i64), ("head_dim", _i64), ("page_stride", _i64), ("token_stride", _i64),
                ("head_stride", _i64), ("dtype", ctypes.c_int)]


class _Sequences(ctypes.Structure):
    """sgq_sequences (include/sgq.h)."""
    _fields_ = [("table", ctypes.c_void_p), ("table_ld", _i64), ("table_pages", _i64), ("lens", ctypes.c_void_p),
                ("starts", ctypes.c_void_p), ("B", _i64), ("max_len", _i64), ("max_new", _i64)]


class _Scores(ctypes.Structure):
    """sgq_scores (include/sgq.h)."""
    _fields_ = [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("window", _i64),
                ("alibi_slopes", ctypes.c_void_p), ("prefix", ctypes.c_void_p), ("first_key", ctypes.c_void_p)]


class _Held:
    """An object whose struct holds addresses of its tensors, and so is not changed; a copy of it is made of their copies."""

    __slots__ = ()

    def _hold(self, **values) -> None:
        for name, value in values.items():
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__} keeps addresses of its tensors: make a new one instead of assigning {name}")

    def __delattr__(self, name):
        self.__setattr__(name, None)


class PagedKV(_Held):
    """A layer's pool of pages: k and v [pages, page, kv_heads, head_dim], alike in shape,
    strides and type; page a power of two from 8 on, head_dim a multiple of 16 up to 256, heads next to
    each other in any order of the first three dimensions (views of [pages, kv_heads, page, head_dim] will do).
    The pool is written in place: assigning an attribute is refused."""

    __slots__ = ("k", "v", "dtype", "device", "kv_heads", "head_dim", "_step", "_struct", "_at")

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if not k.is_cuda or k.dim() != 4:
            raise ValueError("k must be [pages, page, kv_heads, head_dim] on the device")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride() != k.stride():
            raise ValueError("k and v must be alike in shape, strides, type and device")
        pages, page, heads, d = k.shape
        if page < 8 or page & (page - 1) or page > 65536:
            raise ValueError("a page's rows must be a power of two from 8 to 65536")
        if d < 16 or d % 16 or d > 256:
            raise ValueError("head_dim must be a multiple of 16, at most 256")
        if heads < 1:
            raise ValueError("a cache needs heads")
        step = 16 // k.element_size()
        # The stride of a dimension of one says nothing.
        strides = [s if n > 1 else -(-d // step) * step for s, n in zip(k.stride()[:3], k.shape[:3])]
        if k.stride(3) != 1 or any(s < d or s % step for s in strides) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("every head of a page must be 16-byte aligned and contiguous")
        if k.numel() and k.data_ptr() == v.data_ptr():
            raise ValueError("k and v must have memory of their own")
        struct = _PagedCache(k.data_ptr(), v.data_ptr(), pages, page, heads, d, *strides, _dtype(k.dtype))
        self._hold(k=k, v=v, dtype=k.dtype, device=k.device, kv_heads=heads, head_dim=d, _step=step, _struct=struct,
                   _at=ctypes.addressof(struct))

    def __reduce__(self):
        return PagedKV, (self.k, self.v)

    @classmethod
    def empty(cls, pages: int, page: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "PagedKV":
        shape = (pages, page, kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def _int32(t: torch.Tensor, n: int, dev: torch.device, name: str) -> torch.Tensor:
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.numel() != n:
        raise ValueError(f"{name} must have {n} elements")
    if t.dtype is not torch.int32:
        if t.is_floating_point() or t.is_complex() or t.dtype in (torch.bool, torch.uint64):
            raise ValueError(f"{name} must be whole numbers of at most 64 bits with a sign")
        if t.dtype in (torch.int64, torch.uint32):  # a limit past 32 bits is one past every key, and does not wrap
            t = t.to(torch.int64).clamp(-(2**31), 2**31 - 1)
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


class SequenceBatch(_Held):
    """The new tokens of B sequences and the pages of all their keys (int32, on the device):

      table [B, pages]  page of key j of sequence b: table[b, j // page]
      lens [B]          keys of a sequence, its new tokens included
      starts [B + 1]    first row of a sequence's new tokens; rows before starts[0] and from
                        starts[B] on are of no sequence and stay as they are

    New token i of n stands at position lens - n + i.  max_len and max_new bound lens and
    n from the host, which does not see them; they size launches and workspaces, so a bound
    near the truth is the better one.  A sequence that breaks a bound, or whose pages are not in the
    pool, has NaN for its outputs.  Sequences may share pages of keys that are not new (where two new
    tokens have one place, it holds either's).  The tensors are read when a call runs: a captured graph takes
    what they hold at its replay.  They are written in place, not exchanged: assigning an attribute is refused."""

    __slots__ = ("table", "lens", "starts", "max_len", "max_new", "device", "_struct", "_at")

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor, max_len: int, max_new: int):
        if not table.is_cuda or table.dim() != 2 or table.dtype is not torch.int32:
            raise ValueError("table must be int32 [B, pages] on the device")
        B, pages = table.shape
        if (pages > 1 and table.stride(1) != 1) or (B > 1 and table.stride(0) < pages):
            raise ValueError("table must have contiguous rows")
        for t, n, name in ((lens, B, "lens"), (starts, B + 1, "starts")):
            if t.dtype is not torch.int32 or t.device != table.device or t.numel() != n or not t.is_contiguous():
                raise ValueError(f"{name} must be {n} contiguous int32 beside table")
        max_len, max_new = int(max_len), int(max_new)
        if not 0 <= max_len <= 2**30 or not 0 <= max_new <= 2**30:
            raise ValueError("max_len and max_new must be from 0 to 2^30")
        struct = _Sequences(table.data_ptr(), table.stride(0) if B > 1 else max(pages, 1), pages, lens.data_ptr(),
                            starts.data_ptr(), B, max_len, max_new)
        self._hold(table=table, lens=lens, starts=starts, max_len=max_len, max_new=max_new, device=table.device,
                   _struct=struct, _at=ctypes.addressof(struct))

    def __reduce__(self):
        return SequenceBatch, (self.table, self.lens, self.starts, self.max_len, self.max_new)


def rotary_frequencies(dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """base^(-2i / dim) for the dim / 2 pairs of the turned part of a head, float64: what
    norm_rope_append takes as freqs, as it is or scaled for longer contexts."""
    if dim < 2 or dim % 2:
        raise ValueError("the turned part of a head must be even")
    return (float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).to(device)


def _heads(x: torch.Tensor, name: str, rows: int, heads: int, kv: PagedKV, copy: bool = True):
    """x [rows, heads, head_dim], its address, its row and its head stride; a copy where heads are not
    16-byte aligned."""
    d = kv.head_dim
    if x.shape != (rows, heads, d):
        raise ValueError(f"{name} must be [{rows}, {heads}, {d}]")
    if x.dtype is not kv.dtype or x.device != kv.device:
        raise ValueError(f"{name} must have the cache's type and device")
    at = x.data_ptr()
    if x.is_contiguous():
        if at % 16 == 0:
            return x, at, heads * d, d
    else:
        row, head, one = x.stride()
        if heads == 1:
            head = d
        if rows == 1:
            row = heads * head
        step = kv._step
        if (one == 1 and row % step == 0 and head % step == 0 and at % 16 == 0 and head >= d and row >= d
                and (row >= (heads - 1) * head + d or head >= (rows - 1) * row + d)):
            return x, at, row, head
    if not copy:
        raise ValueError(f"heads of {name} must be contiguous and 16-byte aligned, and not overlap")
    x = x.clone(memory_format=torch.contiguous_format)
    return x, x.data_ptr(), heads * d, d


def _queries(q: torch.Tensor, kv: PagedKV):
    if q.dim() != 3:
        raise ValueError(f"q must be [rows, heads, {kv.head_dim}]")
    rows, heads, _ = q.shape
    if heads == 0 or heads % kv.kv_heads:
        raise ValueError(f"heads of q must be a multiple of {kv.kv_heads}")
    return rows, heads, _heads(q, "q", rows, heads, kv)


def _same_device(kv: PagedKV, batch: SequenceBatch) -> torch.device:
    dev = kv.device
    if batch.device != dev:
        raise ValueError(f"the batch must be on {dev}")
    return dev


def norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv: PagedKV, batch: SequenceBatch,
                     freqs: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                     k_norm: Optional[torch.Tensor] = None, eps: float = 1e-5, interleaved: bool = False,
                     positions: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The new tokens' q [rows, heads, head_dim], normed and turned; k and v [rows, kv_heads, head_dim]
    go, k normed and turned, to the tokens' rows of the cache.

    q_norm, k_norm [head_dim]: weights of an RMSNorm over each head (None: no norm).
    freqs [pairs], float64: pair i of a head is turned by position * freqs[i]
    radians (None: none is); pairs are elements i and i + pairs of a head, or 2i and 2i + 1 where
    interleaved, the elements behind 2 * pairs stay.  positions [rows]: what the rotation takes
    instead of the tokens' own positions (of 32 bits; what they do not hold is the nearest that they do).
    q, k and v may be parts of one projection's rows; out may be q; none shares memory with the cache."""
    dev = _same_device(kv, batch)
    d, KV = kv.head_dim, kv.kv_heads
    T, H, (q, q_at, q_row, q_head) = _queries(q, kv)
    k, k_at, k_row, k_head = _heads(k, "k", T, KV, kv)
    v, v_at, v_row, v_head = _heads(v, "v", T, KV, kv)
    if out is None:
        out = torch.empty(T, H, d, dtype=kv.dtype, device=dev)
        o_at, o_row, o_head = out.data_ptr(), H * d, d
    else:
        out, o_at, o_row, o_head = _heads(out, "out", T, H, kv, copy=False)
    half = 0
    if freqs is not None:
        half = freqs.numel()
        if freqs.device != dev or freqs.dim() != 1 or 2 * half > d:
            raise ValueError(f"freqs must be at most {d // 2} radians on {dev}")
        if freqs.dtype is not torch.float64 or not freqs.is_contiguous():
            freqs = freqs.to(torch.float64).contiguous()
    g = None if q_norm is None else _vector(q_norm, d, dev, "q_norm")
    gk = None if k_norm is None else _vector(k_norm, d, dev, "k_norm")
    pos = None if positions is None else _int32(positions, T, dev, "positions")
    _call(dev, load_library().sgq_norm_rope_append, q_at, q_row, q_head, k_at, k_row, k_head, v_at, v_row, v_head, o_at,
          o_row, o_head, T, H, kv._at, batch._at,
          None if g is None else g.data_ptr(), None if gk is None else gk.data_ptr(), eps,
          freqs.data_ptr() if half else None, 2 * half, interleaved, None if pos is None else pos.data_ptr())
    return out


def _attention_workspace(kv: PagedKV, batch: SequenceBatch, T: int, H: int, window: int, dev: torch.device):
    """A workspace of its own for each call: what a graph captures stays the graph's."""
    s = kv._struct
    args = (H, s.kv_heads, s.head_dim, s.dtype, batch._struct.B, T, batch.max_len, batch.max_new, window, 0)
    query = load_library().sgq_paged_attention_workspace_bytes
    if dev.index == _current_device():
        need = query(*args)
    else:
        with torch.cuda.device(dev):
            need = query(*args)
    return (torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None), need


def paged_attention(q: torch.Tensor, kv: PagedKV, batch: SequenceBatch, scale: Optional[float] = None,
                    softcap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None, window: int = 0,
                    prefix: Optional[torch.Tensor] = None, first_key: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens q [rows, heads, head_dim] over their sequences' keys and values,
    the new ones included (norm_rope_append has put them there).

    Scores s = scale * q . k (scale: 1 / sqrt(head_dim) by itself); softcap > 0: softcap * tanh(s / softcap)
    (0: none; 1024 at most in 16-bit types);
    alibi_slopes [heads]: then less slope * distance of the positions.  A token at position p sees the
    keys j <= p and those below prefix[b] ([B]; also ahead of it), of them those with j > p - window
    (window > 0) and j >= first_key[row] ([rows], its document's first).  A row that sees
    none is zeros.  A value seen that is not finite makes its column so (NaN, or that infinity), whatever its
    weight.  out may be q, but shares no memory with the cache."""
    dev = _same_device(kv, batch)
    d = kv.head_dim
    T, H, (q, q_at, q_row, q_head) = _queries(q, kv)
    if out is None:
        out = torch.empty(T, H, d, dtype=kv.dtype, device=dev)
        o_at, o_row, o_head = out.data_ptr(), H * d, d
    else:
        out, o_at, o_row, o_head = _heads(out, "out", T, H, kv, copy=False)
    if window < 0:
        raise ValueError("window must not be negative")
    slopes = None if alibi_slopes is None else _vector(alibi_slopes, H, dev, "alibi_slopes")
    prefix = None if prefix is None else _int32(prefix, batch.lens.numel(), dev, "prefix")
    first = None if first_key is None else _int32(first_key, T, dev, "first_key")
    how = _Scores(1.0 / math.sqrt(d) if scale is None else scale, softcap, window,
                  None if slopes is None else slopes.data_ptr(), None if prefix is None else prefix.data_ptr(),
                  None if first is None else first.data_ptr())
    ws, need = _attention_workspace(kv, batch, T, H, window, dev)
    _call(dev, load_library().sgq_paged_attention, q_at, q_row, q_head, o_at, o_row, o_head, T, H, kv._at, batch._at,
          ctypes.addressof(how), None if ws is None else ws.data_ptr(), need)
    return out


class QuantizedAttentionInt8:
    """The attention half of a pre-norm block on 8-bit activations and weights, over a paged cache:

      h    = x + residual
      q, k, v = qkv(rms_norm(h, norm)), normed by head (q_norm, k_norm) and turned (freqs);
      out  = proj(paged_attention(q)) with the new keys and values in the cache

    forward() returns (out, h), as QuantizedMLPInt8 does: the next half adds the two in its own
    norm.  x has the cache's type.  Rows of no sequence hold nothing of use."""

    def __init__(self, qkv: ChannelsInt8, proj: ChannelsInt8, norm: torch.Tensor, heads: int, kv_heads: int,
                 freqs: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-5, interleaved: bool = False,
                 scale: Optional[float] = None, softcap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                 window: int = 0, qkv_bias: Optional[torch.Tensor] = None, proj_bias: Optional[torch.Tensor] = None):
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        if qkv.N % (heads + 2 * kv_heads) or proj.N != qkv.K or proj.K * (heads + 2 * kv_heads) != qkv.N * heads:
            raise ValueError("qkv must be [D, (heads + 2 kv_heads) head_dim], proj [heads head_dim, D]")
        self.qkv, self.proj, self.heads, self.kv_heads, self.eps = qkv, proj, heads, kv_heads, eps
        self.head_dim = qkv.N // (heads + 2 * kv_heads)
        dev = qkv.packed.device
        self.norm = _vector(norm, qkv.K, dev, "norm").reshape(-1)
        self.freqs, self.q_norm, self.k_norm, self.interleaved = freqs, q_norm, k_norm, interleaved
        self.qkv_bias, self.proj_bias = qkv_bias, proj_bias
        self.scores = {"scale": scale, "softcap": softcap, "alibi_slopes": alibi_slopes, "window": window}

    @classmethod
    def from_float(cls, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, proj: torch.Tensor, norm: torch.Tensor,
                   heads: int, kv_heads: int, **how) -> "QuantizedAttentionInt8":
        """From float weights q [D, heads head_dim], k and v [D, kv_heads head_dim], proj [heads head_dim, D]."""
        return cls(quantize_int8_channels(torch.cat([q, k, v], 1)), quantize_int8_channels(proj), norm, heads,
                   kv_heads, **how)

    def forward(self, x: torch.Tensor, kv: PagedKV, batch: SequenceBatch, residual: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None,
                first_key: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        if x.dim() != 2:
            raise ValueError("x must be [rows, D]")
        if residual is None:
            t, h = rms_norm_int8_tokens(x, self.norm, self.eps), x
        else:
            t, h = add_rms_norm_int8_tokens(x, residual, self.norm, self.eps)
        H, KV = self.heads, self.kv_heads
        rows = quantized_matmul_w8a8(t, self.qkv, self.qkv_bias, dtype=x.dtype).view(-1, H + 2 * KV, self.head_dim)
        q = rows[:, :H]
        norm_rope_append(q, rows[:, H : H + KV], rows[:, H + KV :], kv, batch, self.freqs, self.q_norm, self.k_norm,
                         self.eps, self.interleaved, positions, out=q)
        a = paged_attention(q, kv, batch, prefix=prefix, first_key=first_key, **self.scores)
        t = quantize_int8_tokens(a.view(-1, H * self.head_dim), keep_nan=True)
        return quantized_matmul_w8a8(t, self.proj, self.proj_bias, dtype=x.dtype), h


__all__ = ["PagedKV", "SequenceBatch", "rotary_frequencies", "norm_rope_append", "paged_attention",
           "QuantizedAttentionInt8"]
