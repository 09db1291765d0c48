"""8-bit activations on 8-bit weights over libsgq.so (ctypes).

Activations become int8 tokens (a scale per row), weights int8 channels (a scale
per output column of W [K, N]), and products of the two run on the int8 matrix
cores, exact until the scales are applied (inference only: nothing here has a gradient):

    quantize_int8_tokens(x)                        x as tokens (keep_nan: rows that are not finite stay so)
    rms_norm_int8_tokens(x, weight)                rms_norm(x) as tokens
    add_rms_norm_int8_tokens(x, residual, weight)  h = x + residual, and rms_norm(h) as tokens
    dequantize_int8_tokens(t)                      their values
    quantize_int8_channels(w), pack_int8_channels(codes, scales)
    dequantize_int8_channels(qw)
    quantized_matmul_w8a8(t, qw, bias)             t . qw + bias
    quantized_swiglu_w8a8(t, gate, up)             silu(t . gate) * (t . up)
    QuantizedMLPInt8                               add, norm, gated MLP and down projection in 8 bits

Activations and outputs are float32, bfloat16 or float16.  The reference has no
counterpart; the quantizer is its INT8 one (src/quantization.cpp:42-75) over rows
of activations and columns of weights.  Everything runs on the device and stream
of its tensors.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _check, _ptr, _raw_stream, _stream, load_library

# torch.cuda.current_device() without its check that CUDA is initialised, which the
# tensors of a call have shown.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
if _raw_stream is None:

    def _raw_stream(index: int) -> int:
        return _stream(torch.device("cuda", index))


_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # SGQ_F32, SGQ_BF16, SGQ_F16


class TokensInt8:
    """Rows of activations as int8 codes with a scale each.  codes [M, row] holds K
    codes a row, the row a multiple of 16 bytes of at least K rounded up to 128."""

    __slots__ = ("codes", "scales", "K")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, K: int):
        self.codes, self.scales, self.K = codes, scales, K

    @property
    def M(self) -> int:
        return self.codes.shape[0]


@dataclass
class ChannelsInt8:
    """A weight [K, N] as packed int8 codes with a scale per output channel."""

    packed: torch.Tensor
    scales: torch.Tensor
    K: int
    N: int

    def __post_init__(self):
        p, s = self.packed, self.scales
        size = load_library().sgq_channels_packed_bytes(self.K, self.N)
        if size < 0:
            raise ValueError("sgq: a weight of channels has at most 131071 rows")
        if not p.is_cuda or not p.is_contiguous() or p.numel() * p.element_size() < size:
            raise ValueError(f"packed must be {size} contiguous bytes on the device")
        if s.device != p.device or s.dtype is not torch.float32 or not s.is_contiguous() or s.numel() != self.N:
            raise ValueError(f"scales must be {self.N} contiguous float32 beside packed")


def _call(dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) on dev's current stream, with dev the current device."""
    i = dev.index
    if i == _current_device():
        status = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(i))
    if status:
        _check(status)


def _dtype(t: torch.dtype) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise ValueError(f"sgq: {t} is not float32, bfloat16 or float16")
    return code


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """x as a matrix of rows on the device, its own memory wherever rows are contiguous."""
    if not x.is_cuda:
        raise ValueError("sgq: expected a device tensor")
    if x.dim() != 2:
        if x.dim() < 2:
            raise ValueError(f"{name} must have at least 2 dimensions")
        x = x.flatten(0, -2)
    if x.is_contiguous():
        return x
    M, K = x.shape
    if (K > 1 and x.stride(1) != 1) or (M > 1 and x.stride(0) < K):
        x = x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    """Row stride of a matrix of contiguous rows (that of a single row says nothing)."""
    M, K = x.shape
    return x.stride(0) if M > 1 else K or 1


def _vector(t: torch.Tensor, n: int, dev: torch.device, name: str) -> torch.Tensor:
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.numel() != n:
        raise ValueError(f"{name} must have {n} elements")
    if t.dtype is not torch.float32:
        t = t.to(torch.float32)
    return t if t.is_contiguous() else t.contiguous()


def _row_bytes(K: int) -> int:
    """sgq_tokens_row_bytes."""
    if K > 131071:
        raise ValueError("sgq: rows of tokens are at most 131071 long")
    return (K + 127 & -128) or 128


def _new_tokens(M: int, K: int, dev: torch.device) -> TokensInt8:
    return TokensInt8(torch.empty(M, _row_bytes(K), dtype=torch.int8, device=dev),
                      torch.empty(M, dtype=torch.float32, device=dev), K)


def _output(out: Optional[torch.Tensor], M: int, N: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    if out is None:
        return torch.empty(M, N, dtype=dtype, device=dev)
    if out.dtype != dtype or out.device != dev or tuple(out.shape) != (M, N):
        raise ValueError(f"out must be a {dtype} [{M}, {N}] on {dev}")
    if (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
        raise ValueError("out must have contiguous rows")
    return out


def quantize_int8_tokens(x: torch.Tensor, keep_nan: bool = False) -> TokensInt8:
    """The rows of x (all dimensions but the last taken together) as int8 tokens.  By
    itself this is quantize_int8's rule, where a NaN loses the maximum: a row of NaN
    becomes small finite values.  keep_nan: a row with a NaN or an infinity has a scale
    of NaN, as it has behind the norms, and every product of it is NaN; what a model
    computes on the way (an MLP's hidden values) wants this."""
    x = _rows(x, "x")
    M, K = x.shape
    t = _new_tokens(M, K, x.device)
    lib = load_library()
    fn = lib.sgq_quantize_tokens_keep_nan if keep_nan else lib.sgq_quantize_tokens
    _call(x.device, fn, x.data_ptr(), _dtype(x.dtype), _ld(x), M, K,
          t.codes.data_ptr(), _row_bytes(K), t.scales.data_ptr())
    return t


def _norm_tokens(x, residual, weight, eps, out):
    M, K = x.shape
    if M and not K:
        raise ValueError("rms_norm of rows without elements")
    dev = x.device
    g = _vector(weight, K, dev, "weight")
    t = _new_tokens(M, K, dev)
    if residual is None:
        r = h = None
        ldr = ldh = 0
    else:
        r, ldr, h, ldh = residual.data_ptr(), _ld(residual), out.data_ptr(), _ld(out)
    _call(dev, load_library().sgq_rms_norm_tokens, x.data_ptr(), _dtype(x.dtype), _ld(x), r, ldr, h, ldh,
          g.data_ptr(), eps, M, K, t.codes.data_ptr(), _row_bytes(K), t.scales.data_ptr())
    return t


def rms_norm_int8_tokens(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> TokensInt8:
    """rms_norm over the last dimension of x, as int8 tokens."""
    return _norm_tokens(_rows(x, "x"), None, weight, eps, None)


def add_rms_norm_int8_tokens(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                             out: Optional[torch.Tensor] = None) -> Tuple[TokensInt8, torch.Tensor]:
    """h = x + residual, and rms_norm(h) as int8 tokens.  h comes in x's shape, or in
    `out`, which may be x or residual itself but share no other memory with them."""
    shape, dtype, dev = x.shape, x.dtype, x.device
    if residual.shape != shape or residual.dtype != dtype or residual.device != dev:
        raise ValueError("x and residual must be alike in shape, type and device")
    x, r = _rows(x, "x"), _rows(residual, "residual")
    if out is None:
        M, K = x.shape
        y = torch.empty(M, K, dtype=dtype, device=dev)
        h = y if len(shape) == 2 else y.view(shape)
    elif out.shape != shape or out.dtype != dtype or out.device != dev:
        raise ValueError("out must be alike x in shape, type and device")
    else:
        h, y = out, _rows(out, "out")
        if y.data_ptr() != out.data_ptr():
            raise ValueError("out must have contiguous rows")
    return _norm_tokens(x, r, weight, eps, y), h


def dequantize_int8_tokens(t: TokensInt8, dtype: torch.dtype = torch.float32,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values [M, K] that tokens stand for."""
    dev, K = t.codes.device, t.K
    codes, ldc, scales, M = _tokens(t, dev)
    y = _output(out, M, K, dtype, dev)
    _call(dev, load_library().sgq_dequantize_tokens, codes, ldc, scales, M, K, y.data_ptr(), _dtype(dtype),
          K if out is None else _ld(y))
    return y


def _weight2d(w: torch.Tensor) -> torch.Tensor:
    if not w.is_cuda:
        raise ValueError("sgq: expected a device tensor")
    if w.dim() != 2:
        raise ValueError("a weight of channels must be [K, N]")
    if w.is_complex():
        raise ValueError("a weight of channels cannot be complex")
    return w.to(torch.float32).contiguous()


def _new_channels(K: int, N: int, scales: torch.Tensor):
    lib, dev = load_library(), scales.device
    size = lib.sgq_channels_packed_bytes(K, N)
    if size < 0:
        raise ValueError("sgq: a weight of channels has at most 131071 rows")
    ws = torch.empty(lib.sgq_channels_workspace_bytes(K, N), dtype=torch.uint8, device=dev)
    return ChannelsInt8(torch.empty(max(size, 16), dtype=torch.uint8, device=dev), scales, K, N), ws


def quantize_int8_channels(w: torch.Tensor) -> ChannelsInt8:
    """A float weight [K, N] as int8 codes with a scale per output channel."""
    w = _weight2d(w)
    K, N = w.shape
    qw, ws = _new_channels(K, N, torch.empty(N, dtype=torch.float32, device=w.device))
    _call(w.device, load_library().sgq_quantize_channels, w.data_ptr(), K, N, None, qw.scales.data_ptr(),
          qw.packed.data_ptr(), ws.data_ptr(), ws.numel())
    return qw


def pack_int8_channels(codes: torch.Tensor, scales: torch.Tensor) -> ChannelsInt8:
    """From codes [K, N] (whole numbers in [-128, 127], of any real type) and scales [N], as
    a checkpoint holds them.  Waits for the stream, to say whether the codes are such.

    Of a QuantizedTensor q with one scale (quantize_int8, per tensor):
    pack_int8_channels(unpack_codes(q), q.scales.expand(N)).  One per channel cannot come
    along: it has a scale for each row of W [K, N], which would have to multiply the terms
    of a sum that is in integers here; such a weight is quantized again, by
    quantize_int8_channels(dequantize_int8(q))."""
    given, codes = codes, _weight2d(codes)
    if given.dtype is torch.float64:
        # What only fp32 takes for a whole number is none.
        codes = torch.where(codes == given, codes, float("nan")).contiguous()
    K, N = codes.shape
    qw, ws = _new_channels(K, N, _vector(scales, N, codes.device, "scales").reshape(-1).clone())
    _call(codes.device, load_library().sgq_pack_channels, codes.data_ptr(), K, N, qw.packed.data_ptr(), ws.data_ptr(),
          ws.numel())
    return qw


def unpack_int8_channels(qw: ChannelsInt8) -> torch.Tensor:
    """The fp32 codes [K, N]."""
    out = torch.empty((qw.K, qw.N), dtype=torch.float32, device=qw.packed.device)
    _call(out.device, load_library().sgq_unpack_channels, _ptr(qw.packed), qw.K, qw.N, out.data_ptr())
    return out


def dequantize_int8_channels(qw: ChannelsInt8) -> torch.Tensor:
    """The fp32 weight [K, N] that the codes stand for."""
    out = torch.empty((qw.K, qw.N), dtype=torch.float32, device=qw.packed.device)
    _call(out.device, load_library().sgq_dequantize_channels, _ptr(qw.packed), _ptr(qw.scales), qw.K, qw.N,
          out.data_ptr())
    return out


def _tokens(t: TokensInt8, dev: torch.device) -> Tuple[int, int, int, int]:
    """Address, row stride and scales' address of tokens on dev, and how many they are."""
    c, s = t.codes, t.scales
    if not c.is_cuda or c.dtype is not torch.int8 or c.dim() != 2:
        raise ValueError("token codes must be int8 rows on the device")
    if c.device != dev or s.device != dev:
        raise ValueError("tokens and weight must be on one device")
    M, row = c.shape
    ld = row
    if not c.is_contiguous():
        if row > 1 and c.stride(1) != 1:
            raise ValueError("token codes must be int8 rows on the device")
        ld = _ld(c)
        if ld < row:
            raise ValueError("rows of token codes overlap")
    if s.dtype is not torch.float32 or s.numel() != M or not s.is_contiguous():
        raise ValueError("token scales must be fp32, one per row")
    if row < _row_bytes(t.K):
        raise ValueError(f"rows of {t.K} token codes take {_row_bytes(t.K)} bytes")
    return c.data_ptr(), ld, s.data_ptr(), M


def _workspace(query, M: int, K: int, N: int, dev: torch.device):
    """A workspace of its own for each call: what a graph captures stays the graph's."""
    if M <= 16:  # such products have none
        return None, 0
    if dev.index == _current_device():
        need = query(M, K, N, 0)
    else:
        with torch.cuda.device(dev):
            need = query(M, K, N, 0)
    return (torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None), need


def _bias(b: Optional[torch.Tensor], N: int, dev: torch.device) -> Optional[torch.Tensor]:
    return None if b is None else _vector(b, N, dev, "bias")


def quantized_matmul_w8a8(t: TokensInt8, qw: ChannelsInt8, bias: Optional[torch.Tensor] = None,
                          dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """t . qw (+ bias) [M, N] in `dtype`."""
    dev = qw.packed.device
    if t.K != qw.K:
        raise ValueError("Matrix inner dimensions must match for matmul!")
    codes, ldc, scales, M = _tokens(t, dev)
    N, lib = qw.N, load_library()
    b = _bias(bias, N, dev)
    y = _output(out, M, N, dtype, dev)
    ws, need = _workspace(lib.sgq_linear_w8a8_workspace_bytes, M, qw.K, N, dev)
    _call(dev, lib.sgq_linear_w8a8, codes, ldc, scales, M, qw.K, N, qw.packed.data_ptr(),
          qw.scales.data_ptr(), None if b is None else b.data_ptr(), y.data_ptr(), _dtype(dtype),
          N if out is None else _ld(y), None if ws is None else ws.data_ptr(), need)
    return y


def quantized_swiglu_w8a8(t: TokensInt8, w_gate: ChannelsInt8, w_up: ChannelsInt8,
                          bias_gate: Optional[torch.Tensor] = None, bias_up: Optional[torch.Tensor] = None,
                          dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu(t . w_gate + bias_gate) * (t . w_up + bias_up) [M, N] in `dtype`."""
    dev = w_gate.packed.device
    if (w_gate.K, w_gate.N) != (w_up.K, w_up.N) or w_up.packed.device != dev:
        raise ValueError("gate and up weights must have the same shape and device")
    if t.K != w_gate.K:
        raise ValueError("Matrix inner dimensions must match for matmul!")
    codes, ldc, scales, M = _tokens(t, dev)
    K, N, lib = w_gate.K, w_gate.N, load_library()
    bg, bu = _bias(bias_gate, N, dev), _bias(bias_up, N, dev)
    h = _output(out, M, N, dtype, dev)
    ws, need = _workspace(lib.sgq_swiglu_w8a8_workspace_bytes, M, K, N, dev)
    _call(dev, lib.sgq_swiglu_w8a8, codes, ldc, scales, M, K, N, w_gate.packed.data_ptr(),
          w_gate.scales.data_ptr(), None if bg is None else bg.data_ptr(), w_up.packed.data_ptr(),
          w_up.scales.data_ptr(), None if bu is None else bu.data_ptr(), h.data_ptr(), _dtype(dtype),
          N if out is None else _ld(h),
          None if ws is None else ws.data_ptr(), need)
    return h


class QuantizedMLPInt8:
    """The feed-forward half of a pre-norm block on 8-bit activations and weights:

      h   = x + residual
      out = down(silu(gate(n)) * up(n)),  n = rms_norm(h, norm)

    forward() returns (out, h); the next layer adds the two in its own norm.  Where a
    row of h is not finite, its squares pass fp32 or its hidden values pass the type,
    the row of out is NaN."""

    def __init__(self, gate: ChannelsInt8, up: ChannelsInt8, down: ChannelsInt8, norm: torch.Tensor,
                 eps: float = 1e-5):
        if (gate.K, gate.N) != (up.K, up.N) or (down.K, down.N) != (gate.N, gate.K):
            raise ValueError("gate and up must be [D, H], down [H, D]")
        self.gate, self.up, self.down, self.eps = gate, up, down, eps
        self.norm = _vector(norm, gate.K, gate.packed.device, "norm").reshape(-1)

    @classmethod
    def from_float(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, norm: torch.Tensor,
                   eps: float = 1e-5) -> "QuantizedMLPInt8":
        return cls(*(quantize_int8_channels(w) for w in (gate, up, down)), norm, eps)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        if residual is None:
            t, h = rms_norm_int8_tokens(x, self.norm, self.eps), x
        else:
            t, h = add_rms_norm_int8_tokens(x, residual, self.norm, self.eps)
        a = quantized_swiglu_w8a8(t, self.gate, self.up, dtype=x.dtype)
        return quantized_matmul_w8a8(quantize_int8_tokens(a, keep_nan=True), self.down, dtype=x.dtype).reshape(x.shape), h


__all__ = ["TokensInt8", "ChannelsInt8", "quantize_int8_tokens", "rms_norm_int8_tokens", "add_rms_norm_int8_tokens",
           "dequantize_int8_tokens", "quantize_int8_channels", "pack_int8_channels", "unpack_int8_channels",
           "dequantize_int8_channels", "quantized_matmul_w8a8", "quantized_swiglu_w8a8", "QuantizedMLPInt8"]
