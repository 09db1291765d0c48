"""The attention half of a block on 8-bit projections in 64 bits, with bounds for what the types' roundings make of it.

Inputs are such that the first quantization is exact: every row of the sum x + residual is +-a, and the norm's weights are
+-c, so that all codes are +-127.  What is left are the roundings to the type, with h half a step of it (0 for fp32)
and U = 2^-24 of fp32, and the codes of the attention's output, of 1 / 254 of a row's largest value.  Bounds are of first
order with 5% for the rest:
  a projection        e <= (h + U) |x| + (K + 8) U M,  M = sum |n| |W| + |bias|
  a head's norm       (e_i + |x_i| rms(e) / rms) |g| / rms + 8 U |u|
  the rotation        e_a + e_b + (h + U) |y| + 32 U (|a| + |b|)
  a score             D = scale (sum |q| e_k + e_q |k| + e_q e_k) + 2 (d + 8) U (scale sum |q| |k| + bias + cap)
  the weighted mean   A (exp(2 D) - 1) + exp(2 D) sum w e_v + (h + U) |o| + (h + (n + 16) U) A,  A = sum w |v|
  the last product    sum |W| (e_o + (max |o| + max e_o) / 254) + (h + U) |y| + (K + 8) U sum |W| |o|
"""
import math

import torch

U = 2.0**-24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _norm(x, e, g, eps):
    rms = torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    u = x * g / rms
    spread = torch.sqrt(e.pow(2).mean(-1, keepdim=True)) / rms
    return u, 1.05 * (e + x.abs() * spread) * g.abs() / rms + 8 * U * u.abs()


def _turn(x, e, freqs, pos, interleaved, h):
    half = 0 if freqs is None else freqs.numel()
    y, ey = x.clone(), e.clone()
    if half:
        first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
        second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
        angle = (pos.double()[:, None] * freqs)[:, None]
        a, b = x[..., first], x[..., second]
        y[..., first] = a * angle.cos() - b * angle.sin()
        y[..., second] = b * angle.cos() + a * angle.sin()
        ey[..., first] = ey[..., second] = e[..., first] + e[..., second] + 32 * U * (a.abs() + b.abs())
    return y, ey + (h + U) * y.abs()


def layer(n, parts, proj, heads, kv_heads, pos, seen, h, freqs=None, q_norm=None, k_norm=None, eps=1e-5, interleaved=False,
          scale=None, softcap=0.0, alibi_slopes=None, qkv_bias=None, proj_bias=None):
    """(out, bound) [T, D] of one sequence: n [T, K] normed rows, parts the q, k and v weights [K, heads d], proj [heads d, D],
    pos [T] for the rotation, seen [T, T] which row sees which key; all in 64 bits."""
    T, K = n.shape
    d = parts[0].shape[1] // heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    at, x = 0, []
    for w in parts:
        b = 0.0 if qkv_bias is None else qkv_bias[at : at + w.shape[1]]
        at += w.shape[1]
        y = n @ w + b
        e = (h + U) * y.abs() + (K + 8) * U * (n.abs() @ w.abs() + (0.0 if qkv_bias is None else b.abs()))
        x.append((y.view(T, -1, d), e.view(T, -1, d)))
    (q, eq), (k, ek), (v, ev) = x
    if q_norm is not None:
        q, eq = _norm(q, eq, q_norm, eps)
    if k_norm is not None:
        k, ek = _norm(k, ek, k_norm, eps)
    q, eq = _turn(q, eq, freqs, pos, interleaved, h)
    k, ek = _turn(k, ek, freqs, pos, interleaved, h)
    o, eo = torch.zeros(T, heads, d, dtype=torch.float64), torch.zeros(T, heads, d, dtype=torch.float64)
    away = (torch.arange(T)[:, None] - torch.arange(T)).abs().double()
    for i in range(heads):
        j = i // (heads // kv_heads)
        s = scale * q[:, i] @ k[:, j].T
        mag = abs(scale) * q[:, i].abs() @ k[:, j].abs().T
        err = abs(scale) * (q[:, i].abs() @ ek[:, j].T + eq[:, i] @ k[:, j].abs().T + eq[:, i] @ ek[:, j].T)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        bias = 0.0 if alibi_slopes is None else away * float(alibi_slopes[i])
        s = (s - bias).masked_fill(~seen, -math.inf)
        D = (err + 2 * (d + 8) * U * (mag + bias + softcap)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        w = torch.softmax(s, -1).nan_to_num(0.0)  # rows that see nothing: zeros
        A = w @ v[:, j].abs()
        o[:, i] = w @ v[:, j]
        grow = torch.exp(2 * D)
        eo[:, i] = A * (grow - 1) + grow * (w @ ev[:, j]) + (h + U) * o[:, i].abs() + (h + (T + 16) * U) * A
    o, eo = 1.0 * o.view(T, -1), 1.05 * eo.view(T, -1)
    y = o @ proj + (0.0 if proj_bias is None else proj_bias)
    code = (o.abs().amax(-1, keepdim=True) + eo.amax(-1, keepdim=True)) / 254
    bound = (eo + code) @ proj.abs() + (h + U) * y.abs() + (o.shape[1] + 8) * U * (o.abs() @ proj.abs())
    return y, 1.05 * bound + 2.0**-24


def inputs(T, K, seed):
    """x, residual [T, K] whose sum is +-a in every row, exactly in every type, and the sum."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-8, 9, (T, K), generator=g).double() / 8
    a = 2.0 ** torch.randint(-1, 2, (T, 1), generator=g).double()
    total = (torch.randint(0, 2, (T, K), generator=g).double() * 2 - 1) * a
    return x, total - x, total


def weights(K, heads, kv_heads, d, seed):
    """q, k, v [K, ..], proj [heads d, K], norm [K] of +-c; with which rows' codes are exact."""
    g = torch.Generator().manual_seed(seed)
    parts = [torch.randn(K, n * d, generator=g) * 1.5 * K**-0.5 for n in (heads, kv_heads, kv_heads)]
    proj = torch.randn(heads * d, K, generator=g) * (heads * d) ** -0.5
    norm = (torch.randint(0, 2, (K,), generator=g).float() * 2 - 1) * 1.25
    return parts, proj, norm


VARIANTS = {
    "plain": dict(),
    "turned": dict(freqs=8),
    "norms": dict(freqs=8, norms=True),
    "biases": dict(freqs=4, biases=True, added=False),
    "interleaved": dict(freqs=6, interleaved=True, positions=True, norms=True),
    "cap and window": dict(freqs=8, softcap=3.0, window=9, biases=True),
    "distance and documents": dict(slopes=True, first_key=True, norms=True),
    "prefix": dict(freqs=8, prefix=True, scale=0.4, norms=True),
    "all": dict(freqs=7, norms=True, biases=True, interleaved=True, positions=True, softcap=5.0, window=20, slopes=True,
                prefix=True, first_key=True, scale=-0.3),
}


def variant(name, K, heads, kv_heads, d, lens, seed=3):
    """What a variant gives the layer when it is made, and each sequence in a call."""
    v, g = VARIANTS[name], torch.Generator().manual_seed(seed)
    made = {key: v[key] for key in ("softcap", "scale", "interleaved") if key in v}
    if "freqs" in v:
        made["freqs"] = 10.0 ** (-torch.arange(v["freqs"], dtype=torch.float64) / v["freqs"])
    if "norms" in v:
        made["q_norm"], made["k_norm"] = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    if "biases" in v:
        made["qkv_bias"] = torch.randn((heads + 2 * kv_heads) * d, generator=g)
        made["proj_bias"] = torch.randn(K, generator=g)
    if "slopes" in v:
        made["alibi_slopes"] = 0.5 ** (1 + torch.arange(heads).float())
    calls = []
    for i, n in enumerate(lens):
        p, j = torch.arange(n)[:, None], torch.arange(n)
        seen, call = j <= p, {}
        if "prefix" in v:
            call["prefix"] = n // 2 + i
            seen = seen | (j < call["prefix"])
        if "window" in v:
            seen = seen & (j > p - v["window"])
        call["first_key"] = torch.clamp(torch.arange(n) // 7 * 7 - 3, min=0) if "first_key" in v else None
        if call["first_key"] is not None:
            seen = seen & (j >= call["first_key"][:, None])
        call["positions"] = torch.randint(-1000, 1000, (n,), generator=g) if "positions" in v else None
        call["seen"] = seen
        calls.append(call)
    return made, v.get("window", 0), calls
