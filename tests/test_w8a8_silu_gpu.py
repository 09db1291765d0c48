"""The gated product's silu on gates that are known exactly (the codes are zero, so that gate and up are their biases),
against 64 bits, over the whole range of fp32 and through every kind of kernel that ends with it."""
import ctypes

import pytest
import torch

from test_w8a8_gpu import HALF, TINY, TYPES, U, _gen, _tokens

pytestmark = pytest.mark.gpu

# Roundings of silu in units of U = 2^-24: the exponential's argument, split exactly into a power of two and a rest of
# at most 1/2 + 2^-23 by two fused operations, is off by 2 * 2^-26 (0.35 after the factor ln 2), the hardware's
# exponential by a step (2), the sum by 1, the hardware's reciprocal by a step (2), the product with the gate by 1, the
# product with up by 1; a power of two changes a normal value not at all and a subnormal one by half its step.
STEPS = 8
SPECIAL = [0.0, -0.0, 1e-38, -1e-38, 1e-45, -1e-45, 1e-20, -1e-20, 0.5, -0.5, 1.0, -1.0, 16.0, -16.0, 20.0, -20.0, 43.0, -43.0,
           60.0, -60.0, 86.0, -86.0, 87.0, -87.0, -87.3, -87.4, -88.0, -88.5, 88.0, -88.7, -88.8, -89.0, -92.0, -95.0, -100.0,
           -103.0, -104.0, -110.0, -111.0, 100.0, 120.0, -150.0, 150.0, -1e3, 1e3, -1e10, 1e10, -3e38, 3e38]


def _silu(g):
    """silu of 64-bit values; the quotient's small factor is taken where it does not overflow."""
    e = torch.exp(-g.abs())
    return torch.where(g >= 0, g, g * e) / (1 + e)


def _gates(dev):
    g = torch.linspace(-115, 115, 4786, device=dev)
    tail = torch.linspace(-89.5, -86.5, 600, device=dev)
    small = torch.randn(400, generator=_gen(dev, 3), device=dev) * 0.1
    return torch.cat([g, tail, small, torch.tensor(SPECIAL, device=dev)])


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


# Tokens and K: no product at all, the forms for few tokens, tiles of each size, K split and joined.
FORMS = [(3, 0), (1, 64), (16, 64), (17, 64), (33, 1000), (33, 2243), (90, 64), (17, 9000), (1300, 64), (160, 64), (500, 64),
         (700, 64)]


def _zero(op, dev, K, N):
    if K == 0:
        return op.ChannelsInt8(torch.empty(16, dtype=torch.uint8, device=dev), torch.ones(N, device=dev), 0, N)
    return op.pack_int8_channels(torch.ones(K, N, dtype=torch.int8, device=dev), torch.ones(N, device=dev))


def _same(got, want, tol, dtype):
    """Within tol and the type's rounding; what rounds past the type is infinite, of the right sign."""
    limit = float(torch.finfo(dtype).max) * (1 + HALF[dtype] / 2)
    tol = tol * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + TINY[dtype]
    g = got.double()
    near = (g - want).abs() <= tol
    past = (want.abs() + tol >= limit) & torch.isinf(g) & (torch.sign(g) == torch.sign(want))
    return bool((near | past).all())


def test_forms(sgq):
    seen = set()
    N = 5835
    for M, K in FORMS:
        f, ks = ctypes.c_int(), ctypes.c_int()
        assert sgq.load_library().sgq_w8a8_plan(1, M, K, N, 256, ctypes.byref(f), ctypes.byref(ks)) == 0
        seen.add((f.value, ks.value > 1))
    assert {f for f, _ in seen} == set(range(10)) and any(split for _, split in seen), sorted(seen)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", FORMS)
def test_silu_of_exact_gates(op, dev, M, K, dtype):
    g = _gates(dev)
    N = g.numel()
    t = _tokens(op, torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev))
    w = _zero(op, dev, K, N)
    for up in (1.0, -2.5, 1e30):
        u = torch.full((N,), up, device=dev)
        h = op.quantized_swiglu_w8a8(t, w, w, g, u, dtype)
        assert torch.equal(h, h[:1].expand(M, N))
        want = _silu(g.double()) * u.double()
        # silu itself may be subnormal: half a step of it, times up.
        assert _same(h[0], want, STEPS * U * want.abs() + abs(up) * 2.0**-150 + 2.0**-149, dtype), up


@pytest.mark.parametrize("M,K", [(1, 64), (33, 1000), (17, 9000), (700, 64)])
def test_silu_of_infinite_gates(op, dev, M, K):
    """silu(inf) is inf; -inf times a factor of zero is no number, as in every other silu here; a NaN stays one."""
    g = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0, 0.0] * 4, device=dev)
    u = torch.ones(20, device=dev)
    t = _tokens(op, torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev))
    w = _zero(op, dev, K, 20)
    h = op.quantized_swiglu_w8a8(t, w, w, g, u).view(M, 4, 5)
    assert (h[..., 0] == float("inf")).all() and torch.isnan(h[..., 1:3]).all()
    assert torch.isfinite(h[..., 3:]).all() and not h[..., 4].any()
    h = op.quantized_swiglu_w8a8(t, w, w, u, g).view(M, 4, 5)
    assert torch.isinf(h[..., :2]).all() and torch.isnan(h[..., 2]).all() and torch.isfinite(h[..., 3:]).all()
