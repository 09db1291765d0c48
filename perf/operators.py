"""The 8-bit activation operators as cases to time and to compare.

Tokens (rows of activations) and a weight's output channels (columns) are held as
int8 codes with a fp32 scale each; products of the two run on integers.  The plain
forms below are elementary torch operations; with `own` true the same passes go
through the package's entry points.

Kinds:
  norm    h = x + residual, its RMSNorm as 8-bit tokens, read back as values
  tokens  activations as 8-bit tokens, read back as values
  matmul  y = tokens . weight (+ bias)
  swiglu  silu(tokens . gate) * (tokens . up)
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

PKG_DIR = Path(__file__).resolve().parents[1] / "soverign-grad_amd"
W_STD = 0.02
EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
ROW = 128  # a row of codes is held in a multiple of this many bytes


def w8a8():
    """soverign-grad_amd/ as the package `soverign_grad_amd` (its folder's name is no identifier)."""
    name = "soverign_grad_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, PKG_DIR / "__init__.py",
                                                      submodule_search_locations=[str(PKG_DIR)])
        sys.modules[name] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    import soverign_grad_amd.w8a8 as mod

    return mod


# ---- the cases -------------------------------------------------------------


def norm(name, M, K, dtype, residual=True):
    return {"name": name, "kind": "norm", "M": M, "K": K, "dtype": dtype, "residual": residual}


def tokens(name, M, K, dtype):
    return {"name": name, "kind": "tokens", "M": M, "K": K, "dtype": dtype}


def matmul(name, M, K, N, dtype, bias=False):
    return {"name": name, "kind": "matmul", "M": M, "K": K, "N": N, "dtype": dtype, "bias": bias}


def swiglu(name, M, K, N, dtype, bias=False):
    return {"name": name, "kind": "swiglu", "M": M, "K": K, "N": N, "dtype": dtype, "bias": bias}


def listed():
    return [
        # The norm before a projection in a decode step of eight sequences: launch and latency.
        norm("norm_step", 8, 2048, "fp32"),
        # A prompt's norm with the residual stream in bf16.
        norm("norm_prompt", 2048, 4096, "bf16"),
        # A width of no power of two's multiple, the first norm of a model (nothing to add yet).
        norm("norm_odd", 1023, 5003, "fp16", residual=False),
        # Several long prompts at once, the widest model: the largest norm.
        norm("norm_large", 16384, 8192, "bf16"),
        # An MLP's hidden activations before the down projection.
        tokens("tokens_hidden", 2048, 11008, "fp32"),
        # One token through one projection: the smallest product, the weight's bytes.
        matmul("matmul_row", 1, 4096, 4096, "fp32"),
        # A small layer on a batch, with its bias.
        matmul("matmul_batch", 128, 1024, 1024, "fp32", bias=True),
        # Odd sizes everywhere: an output head over a ragged batch.
        matmul("matmul_odd", 333, 2043, 5001, "fp16", bias=True),
        # A prompt through a square projection.
        matmul("matmul_prompt", 2048, 4096, 4096, "bf16"),
        # Long prompts through the widest projection: the largest call.
        matmul("matmul_large", 8192, 8192, 28672, "bf16"),
        # The gated half of an MLP for a served batch of sixteen.
        swiglu("swiglu_step", 16, 4096, 11008, "bf16"),
        # The same for a prompt.
        swiglu("swiglu_prompt", 2048, 4096, 11008, "fp32"),
    ]


LARGEST = 8192 * 8192 * 28672  # M * K * N of the largest product
LARGEST_NORM = 16384 * 8192


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width from lo to hi: mostly multiples of 128 or 64, odd ones among them."""
    step = rng.choice([128, 128, 64, 8, 1])
    return max(lo, _log_int(rng, lo, hi) // step * step)


def _rows(rng, hi):
    return rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 33, 512), _log_int(rng, 513, hi)])


def draw(rng):
    kind = rng.choice(["norm", "tokens", "matmul", "matmul", "matmul", "swiglu", "swiglu"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    c = {"kind": kind, "M": _rows(rng, 16384 if kind in ("norm", "tokens") else 8192), "dtype": dtype}
    c["K"] = _width(rng, 512, 28672 if kind == "tokens" else 8192)
    if kind in ("norm", "tokens"):
        # no more bytes than the largest norm, which is in 16 bits
        c["M"] = max(1, min(c["M"], LARGEST_NORM * 2 // BYTES[dtype] // c["K"]))
        return dict(c, residual=rng.random() < 0.7) if kind == "norm" else c
    c["N"] = _width(rng, 512, 28672)
    per_row = c["K"] * c["N"] * (2 if kind == "swiglu" else 1)
    c["M"] = max(1, min(c["M"], LARGEST // 4 // per_row))
    return dict(c, bias=rng.random() < 0.4)


# ---- inputs ----------------------------------------------------------------


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda:0", dtype=torch.float32) * std


def _activations(gen, M, K, dtype):
    """N(0, 1), one feature in 256 ten times as large (outlier channels); a batch's last row is padding, zeros."""
    loud = torch.rand(K, generator=gen, device="cuda:0") < 1 / 256
    x = _normal(gen, M, K) * (1 + 9 * loud)
    if M >= 8:
        x[-1] = 0
    return x.to(dtype)


def _held(v, dim):
    """int8 codes and fp32 scales of v, each scale over `dim`: what a checkpoint or an earlier layer left."""
    top = v.abs().amax(dim, keepdim=True).clamp_min(1e-8)
    return torch.round(v / top * 127).to(torch.int8), (top / 127).reshape(-1)


def _weight(gen, K, N, bias):
    codes, scales = _held(_normal(gen, K, N, std=W_STD), 0)
    w = {"codes": codes, "scales": scales, "bias": _normal(gen, N, std=W_STD) if bias else None}
    if own:  # a serving program lays its weights out once
        w["handle"] = w8a8().pack_int8_channels(codes, scales)
    return w


def prepare(case, seed):
    c, dtype = case, TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(int(seed))
    s = {"kind": c["kind"], "dtype": dtype, "K": c["K"]}
    x = _activations(gen, c["M"], c["K"], dtype)
    if c["kind"] in ("norm", "tokens"):
        s["x"] = x
        if c["kind"] == "norm":
            s["g"] = 1 + _normal(gen, c["K"], std=0.1)
            s["r"] = _normal(gen, c["M"], c["K"], std=2.0).to(dtype) if c["residual"] else None
        return s
    codes, s["sx"] = _held(x.float(), 1)
    s["cx"] = torch.zeros(c["M"], -(-c["K"] // ROW) * ROW, dtype=torch.int8, device="cuda:0")
    s["cx"][:, : c["K"]] = codes
    s["w"] = [_weight(gen, c["K"], c["N"], c["bias"]) for _ in range(2 if c["kind"] == "swiglu" else 1)]
    return s


# ---- one pass --------------------------------------------------------------


def _quotient(a, b):
    """a / b rounded once to fp32 (torch's own fp32 division by a number is a multiplication)."""
    return (torch.as_tensor(a, dtype=torch.float64) / b.double()).float()


def _codes(v, inv):
    t = v * inv
    whole = torch.trunc(t)
    return (whole + torch.sign(t) * ((t - whole).abs() >= 0.5)).clamp(-127, 127)  # halves go away from zero


def _plain_norm(s):
    x, dtype = s["x"], s["dtype"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(dtype)
    f = h.float()
    rstd = 1 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)
    u = f * s["g"]  # rstd is a factor of the whole row and changes no code
    m = torch.maximum(u.abs().amax(1, keepdim=True), _quotient(1e-8, rstd))
    scale = m * rstd / 127
    values = (_codes(u, _quotient(127.0, m)) * scale).to(dtype)
    return {"values": values} if s["r"] is None else {"values": values, "h": h}


def _plain_tokens(s):
    x = s["x"].float()
    m = x.abs().amax(1, keepdim=True).clamp_min(1e-8)
    return {"values": (_codes(x, _quotient(127.0, m)) * (m / 127)).to(s["dtype"])}


def _plain_matmul(s, w):
    y = s["cx"][:, : s["K"]].float() @ w["codes"].float()
    y = y * s["sx"][:, None] * w["scales"]
    return y if w["bias"] is None else y + w["bias"]


def run(state):
    s, kind = state, state["kind"]
    if own:
        op = w8a8()
        if kind == "norm":
            if s["r"] is None:
                return {"values": op.dequantize_int8_tokens(op.rms_norm_int8_tokens(s["x"], s["g"], EPS), s["dtype"])}
            t, h = op.add_rms_norm_int8_tokens(s["x"], s["r"], s["g"], EPS)
            return {"values": op.dequantize_int8_tokens(t, s["dtype"]), "h": h}
        if kind == "tokens":
            return {"values": op.dequantize_int8_tokens(op.quantize_int8_tokens(s["x"]), s["dtype"])}
        t, w = op.TokensInt8(s["cx"], s["sx"], s["K"]), s["w"]
        if kind == "matmul":
            return op.quantized_matmul_w8a8(t, w[0]["handle"], w[0]["bias"], dtype=s["dtype"])
        return op.quantized_swiglu_w8a8(t, w[0]["handle"], w[1]["handle"], w[0]["bias"], w[1]["bias"],
                                        dtype=s["dtype"])
    if kind == "norm":
        return _plain_norm(s)
    if kind == "tokens":
        return _plain_tokens(s)
    y = _plain_matmul(s, s["w"][0])
    if kind == "swiglu":
        y = y / (1 + torch.exp(-y)) * _plain_matmul(s, s["w"][1])
    return y.to(s["dtype"])


# ---- what a pass cannot do without -----------------------------------------


def work(case):
    c, e = case, BYTES[case["dtype"]]
    M, K = c["M"], c["K"]
    if c["kind"] == "norm":
        # x (and the residual) in, the values (and h) out, the norm's weights
        return {"bytes": e * M * K * (4 if c["residual"] else 2) + 4 * K, "flops": 8 * M * K}
    if c["kind"] == "tokens":
        return {"bytes": 2 * e * M * K, "flops": 4 * M * K}
    n = 2 if c["kind"] == "swiglu" else 1
    weight = K * c["N"] + 4 * c["N"] * (2 if c["bias"] else 1)
    return {"bytes": M * K + 4 * M + n * weight + e * M * c["N"], "flops": 2 * n * M * K * c["N"]}


# ---- the same in 64 bits ---------------------------------------------------


def _rounded(v):
    """64-bit values as fp32 would hold them: the quantiser's definition rounds its quotient and its product to fp32."""
    return v.to(torch.float32).to(torch.float64)


def _read_back(v, floor):
    """Values of v [M, K] (64 bits, exactly fp32) after a pass through int8, a scale per row over `floor`."""
    top = torch.maximum(v.abs().max(1, keepdim=True).values, floor)
    t = _rounded(v * _rounded(127.0 / top))
    code = torch.floor(t.abs() + 0.5).clamp(max=127.0) * torch.sign(t)
    return code, top / 127.0


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["dtype"]).double()
        rms = torch.sqrt(h.pow(2).sum(1, keepdim=True) / c["K"] + EPS)
        code, scale = _read_back(_rounded(h * s["g"].double()), _rounded(1e-8 * rms))
        out = {"values": code * (scale / rms)}
        return out if s["r"] is None else dict(out, h=h)
    if c["kind"] == "tokens":
        code, scale = _read_back(s["x"].double(), torch.tensor(1e-8, device="cuda:0").double())
        return {"values": code * scale}
    x = s["cx"][:, : c["K"]].double() * s["sx"].double()[:, None]
    y = [x @ (w["codes"].double() * w["scales"].double()) for w in s["w"]]
    y = [v if w["bias"] is None else v + w["bias"].double() for v, w in zip(y, s["w"])]
    return y[0] if len(y) == 1 else y[0] * torch.sigmoid(y[0]) * y[1]
