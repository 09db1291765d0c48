"""8-bit products at their limits: the widest rows of codes, outputs past their type, scales that are not finite, and
every kernel for one weight and for two, in every type and split of K."""
import ctypes

import pytest
import torch

from test_w8a8_gpu import HALF, TINY, TYPES, U, _codes, _error, _exact, _gen, _problem, _tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


def _plan(sgq, gated, M, K, N):
    form, ks = ctypes.c_int(), ctypes.c_int()
    assert sgq.load_library().sgq_w8a8_plan(gated, M, K, N, 256, ctypes.byref(form), ctypes.byref(ks)) == 0
    return form.value, ks.value


def _check(got, want, tol, dtype):
    """Within tol and a rounding to the type; what is past the type is infinite, with its sign."""
    assert got.dtype == dtype
    limit = float(torch.finfo(dtype).max) * (1 + HALF[dtype] / 2)  # half a step past the largest value
    g = got.double()
    tol = tol * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + TINY[dtype]
    near = (g - want).abs() <= tol
    past = (want.abs() + tol >= limit) & torch.isinf(g) & (torch.sign(g) == torch.sign(want))
    bad = ~(near | past)
    assert not bad.any(), (int(bad.sum()), g[bad][:3].tolist(), want[bad][:3].tolist())


def _gated(g, pg, u, pu):
    """silu(g) * u and its error: silu's slope at the gate (its second derivative is at most 1/2, so slope + error / 2
    covers the step to a gate that is off by its error), eight roundings of silu, one product."""
    sig = torch.sigmoid(g)
    s = g * sig
    eg, eu = _error(pg, g), _error(pu, u)
    slope = (sig * (1 + g * (1 - sig))).abs() + eg / 2
    es = slope * eg + 8 * U * s.abs()
    return s * u, es * (u.abs() + eu) + s.abs() * eu + U * (s * u).abs() + 2.0**-149


# ---- products -----------------------------------------------------------------

# (gated, M, K, N), one for each kernel and each number of K splits that the plan reaches, ragged throughout.
EVERY = [(0, 1, 64, 20), (0, 16, 4099, 515), (0, 21, 64, 17), (0, 40, 4099, 2050), (0, 18, 1541, 17), (0, 33, 64, 5842), (0, 276, 65, 17),
         (0, 4271, 2474, 17), (0, 287, 1561, 18), (0, 264, 3697, 17), (0, 658, 65, 10809), (0, 1857, 840, 9216), (0, 193, 23056, 17747),
         (0, 67, 26302, 8408), (0, 67, 65, 16753), (0, 72, 11007, 9789), (0, 4099, 5001, 17), (0, 2221, 9023, 18), (0, 129, 69, 22842),
         (0, 5564, 11456, 259), (0, 65, 8657, 8275), (0, 2060, 13896, 131), (0, 264, 65, 23091), (0, 131, 21240, 23638),
         (0, 5491, 20260, 259), (0, 4309, 37706, 137), (0, 244, 26697, 18203), (0, 7403, 44855, 1345),
         (1, 1, 64, 20), (1, 16, 4099, 515), (1, 21, 64, 17), (1, 18, 538, 9876), (1, 64, 1340, 5376), (1, 34, 2243, 5835),
         (1, 58, 2944, 8064), (1, 33, 4019, 576), (1, 276, 65, 17), (1, 4271, 2474, 17), (1, 287, 1561, 18), (1, 17, 3587, 18),
         (1, 6551, 68, 515), (1, 198, 22878, 8310), (1, 74, 38121, 4106), (1, 67, 65, 8612), (1, 68, 11614, 4839), (1, 4138, 5618, 18),
         (1, 2210, 10904, 17), (1, 67, 65, 16753), (1, 131, 12029, 5604), (1, 4114, 9168, 68), (1, 2119, 15180, 66),
         (1, 133, 68, 16884), (1, 134, 21218, 11277), (1, 5547, 20258, 133), (1, 4243, 32403, 70), (1, 1506, 29609, 1613),
         (1, 91, 4454, 7424)]


def test_every_kernel_for_one_weight_and_two(sgq):
    """EVERY runs forms 1..9 for one weight and for two, each, and the tiles with K split as far as the plan does."""
    seen = {(gated, *_plan(sgq, gated, M, K, N)) for gated, M, K, N in EVERY}
    want = {(g, f, 1) for g in (0, 1) for f in range(1, 10)}
    want |= {(g, f, s) for g in (0, 1) for f in (5, 7, 8, 9) for s in (2, 4, 8)} | {(g, 6, s) for g in (0, 1) for s in (4, 8)}
    assert seen >= want, sorted(want - seen)


@pytest.mark.parametrize("gated,M,K,N", EVERY)
def test_every_kernel_in_every_type(op, dev, gated, M, K, N):
    cx, cw, sx, sw, b = _problem(op, dev, M, K, N, M + K + N, True)
    t, qw = _tokens(op, cx, sx), op.pack_int8_channels(cw, sw)
    p, y = _exact(cx, cw, sx, sw, b)
    if not gated:
        for dtype in TYPES:
            _check(op.quantized_matmul_w8a8(t, qw, b, dtype), y, _error(p, y), dtype)
        return
    del cw
    _, cu, _, su, bu = _problem(op, dev, M, K, N, M + K + N + 50, True)
    qu = op.pack_int8_channels(cu, su)
    pu, u = _exact(cx, cu, sx, su, bu)
    del cu
    want, tol = _gated(y, p, u, pu)
    for dtype in TYPES:
        _check(op.quantized_swiglu_w8a8(t, qw, qu, b, bu, dtype), want, tol, dtype)


# One row block, two, four, a tile of each kind, a split K.
KINDS = [(5, 700, 333), (30, 1000, 1003), (100, 2000, 300), (300, 5000, 640), (700, 64, 5835), (2050, 300, 1100), (70, 9000, 4100)]


@pytest.mark.parametrize("M,K,N", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_outputs_past_their_type(op, dev, M, K, N, dtype):
    """Columns whose values pass the type's largest come out infinite, the others as they are."""
    cx, cw, sx, sw, b = _problem(op, dev, M, K, N, M + K, True)
    peak = float(((cx.double() @ cw.double()[:, ::3]) * sx.double()[:, None]).abs().max())
    # half as much again, or as much as fp32 still holds and bfloat16 does not
    sw[::3] = float(torch.finfo(dtype).max) / peak * (1.5 if dtype is torch.float16 else 1.003)
    t, qw = _tokens(op, cx, sx), op.pack_int8_channels(cw, sw)
    p, y = _exact(cx, cw, sx, sw, b)
    got = op.quantized_matmul_w8a8(t, qw, b, dtype)
    _check(got, y, _error(p, y), dtype)
    assert torch.isinf(got).any() and torch.isfinite(got[:, 1::3]).all()
    if dtype is torch.float16:
        h = op.quantized_swiglu_w8a8(t, qw, qw, b, b, dtype)
        want, tol = _gated(y, p, y, p)
        _check(h, want, tol, dtype)
        assert torch.isinf(h).any()


@pytest.mark.parametrize("M,K,N", KINDS)
def test_scales_that_are_not_finite_through_the_gate(op, dev, M, K, N):
    """A scale of NaN or infinity on a token, or on a column of either weight, reaches its row or column only."""
    cx, cg, sx, sg, bg = _problem(op, dev, M, K, N, M + K, True)
    _, cu, _, su, bu = _problem(op, dev, M, K, N, M + K + 50, True)
    wg, wu = op.pack_int8_channels(cg, sg), op.pack_int8_channels(cu, su)
    clean = op.quantized_swiglu_w8a8(_tokens(op, cx, sx), wg, wu, bg, bu)
    assert torch.isfinite(clean).all()
    nan, inf = float("nan"), float("inf")
    sx[M - 1], sx[1] = nan, inf
    sg[0], sg[N - 1], su[3], su[N - 2] = nan, inf, inf, nan
    got = op.quantized_swiglu_w8a8(_tokens(op, cx, sx), op.pack_int8_channels(cg, sg), op.pack_int8_channels(cu, su), bg, bu)
    rows, cols = [m for m in range(M) if m not in (1, M - 1)], [n for n in range(N) if n not in (0, 3, N - 1, N - 2)]
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    assert torch.isnan(got[M - 1]).all() and torch.isnan(got[:, [0, N - 2]]).all()
    assert not torch.isfinite(got[1]).any()
    g = (cx.double() @ cg.double()[:, [N - 1]])[rows, 0]  # sign of the gate's product: inf, or NaN where silu of -inf is none
    last = got[rows, N - 1]
    assert torch.isinf(last[g > 0]).all() and torch.isnan(last[g <= 0]).all()
    assert not torch.isfinite(got[rows, 3]).any()


def test_rows_of_codes_as_far_apart_as_they_may_be(op, sgq, dev):
    """Rows 2^21 bytes apart: the offsets of a 64-row block and of a 256-row tile with it, and a remainder of rows."""
    row = 2**21
    for M, k, N, form in ((33, 300, 40, 2), (59, 2048, 7278, 4), (300, 300, 900, 5), (523, 300, 20000, 9)):
        assert _plan(sgq, 0, M, k, N)[0] == form
        cx, cw = _codes(dev, 1, M, k), _codes(dev, 2, k, N)
        sx = torch.rand(M, generator=_gen(dev, 3), device=dev) + 0.5
        qw = op.pack_int8_channels(cw, torch.ones(N, device=dev))
        held = -(-k // 128) * 128
        far = torch.empty((M - 1) * row + held, dtype=torch.int8, device=dev).as_strided((M, held), (row, 1))
        far.fill_(77)
        far[:, :k] = cx
        want = op.quantized_matmul_w8a8(_tokens(op, cx, sx), qw)
        got = op.quantized_matmul_w8a8(op.TokensInt8(far, sx, k), qw)
        assert torch.equal(got, want)
        p, y = _exact(cx[-1:], cw, sx[-1:], torch.ones(N, device=dev), None)
        _check(got[-1:], y, _error(p, y), torch.float32)
        near, far = _tokens(op, cx, sx), op.TokensInt8(far, sx, k)
        assert torch.equal(op.quantized_swiglu_w8a8(far, qw, qw), op.quantized_swiglu_w8a8(near, qw, qw))
        assert torch.equal(op.dequantize_int8_tokens(far), op.dequantize_int8_tokens(near))
        del far

