"""8-bit tokens, 8-bit channels and their products against 64 bits.

Codes are fixed bits: the quantizer is single fp32 operations on values that do
not depend on the order of a sum, and the products' sums are exact integers.  What
is left are a few fp32 roundings (2^-24 each) and one to the output's type (half
of its eps), which the tolerances count.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _randn(dev, seed, *shape):
    return torch.randn(*shape, generator=_gen(dev, seed), device=dev)


def _codes(dev, seed, *shape):
    return torch.randint(-127, 128, shape, generator=_gen(dev, seed), device=dev, dtype=torch.int8)


def _f32(a):
    return a.to(torch.float32).to(torch.float64)


def _quantized(v, floor):
    """Codes (64 bits) and the maximum of rows of v (64 bits, fp32 values): the quantizer's definition."""
    top = torch.maximum(torch.where(torch.isnan(v), 0.0, v.abs()).amax(1, keepdim=True), floor)
    t = _f32(v * _f32(127.0 / top))
    code = (torch.floor(t.abs() + 0.5) * torch.sign(t)).clamp(-127, 127)
    return torch.where(torch.isnan(t), 127.0, code), top


def _floor(dev):
    return torch.tensor(float(np.float32(1e-8)), dtype=torch.float64, device=dev)


def _tokens(op, codes, scales):
    """Tokens from bare codes: rows padded as the layout wants, the padding not zero."""
    M, K = codes.shape
    buf = torch.full((M, max(128, -(-K // 128) * 128)), 99, dtype=torch.int8, device=codes.device)
    buf[:, :K] = codes
    return op.TokensInt8(buf, scales, K)


# ---- tokens -----------------------------------------------------------------

WIDTHS = [1, 7, 8, 100, 128, 129, 512, 1000, 1024, 1025, 2048, 4099, 8192, 8193, 20000, 32768, 33000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", WIDTHS)
def test_quantize_tokens(op, dev, K, dtype):
    M = 5
    x = (_randn(dev, K, M, K) * 3).to(dtype)
    x[1] = 0
    x[2] *= 2.0**-12
    t = op.quantize_int8_tokens(x)
    code, top = _quantized(x.double(), _floor(dev))
    assert torch.equal(t.codes[:, :K].double(), code)
    assert not t.codes[:, K:].any()
    assert torch.equal(t.scales.double(), _f32(top[:, 0] / 127))
    for out_t in TYPES:
        v = op.dequantize_int8_tokens(t, out_t)
        assert v.dtype == out_t and torch.equal(v, _f32(code * t.scales.double()[:, None]).to(out_t))


def test_quantize_tokens_is_the_weights_quantizer(op, sgq, dev):
    """fp32 rows: sgq_quantize_int8 per channel, bit for bit, ties and a NaN among them."""
    x = _randn(dev, 3, 64, 1000)
    x[0, :5] = torch.tensor([127.0, 0.5, -0.5, 1.5, -126.5], device=dev)
    x[1, 3] = float("nan")
    x[2, 3] = float("inf")
    x[3] = 1e-9
    q = sgq.quantize_int8(x, sgq.PER_CHANNEL)
    t = op.quantize_int8_tokens(x)
    assert torch.equal(t.codes[:, :1000].float(), q.qdata + 0.0) and torch.equal(t.scales, q.scales)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("K", WIDTHS)
def test_norm_tokens(op, dev, K, dtype, residual):
    M, eps = 6, 1e-5
    x, r = (_randn(dev, K, M, K) * 2).to(dtype), _randn(dev, K + 1, M, K).to(dtype)
    x[1] = 0
    r[1] = 0
    x[2] *= 2.0**-13
    r[2] *= 2.0**-14
    g = 1 + 0.2 * _randn(dev, K + 2, K)
    if residual:
        t, h = op.add_rms_norm_int8_tokens(x, r, g, eps)
        assert torch.equal(h, (x.double() + r.double()).to(dtype))
        h = h.double()
    else:
        t, h = op.rms_norm_int8_tokens(x, g, eps), x.double()
    rms = torch.sqrt(h.pow(2).mean(1, keepdim=True) + np.float32(eps).item())
    # The floor needs rstd, known to a few roundings: no row here is near it but the zeros.
    code, top = _quantized(_f32(h * g.double()), _floor(dev) * rms)
    assert torch.equal(t.codes[:, :K].double(), code)
    assert not t.codes[:, K:].any()
    # K terms in any order (half of it after the root; far less in a tree), then a
    # division, a sum, a root, a quotient, a product and a quotient.
    tol = (K / 256 + 16) * U
    assert bool(((t.scales.double() * 127 * rms[:, 0] / top[:, 0] - 1).abs() <= tol).all())


def test_norm_of_small_rows_meets_the_floor(op, dev):
    """max|n| below 1e-8: the scale is that of 1e-8, as the quantizer has it, and the codes are nearly all zero."""
    x = torch.full((2, 256), 1e-14, device=dev)
    t = op.rms_norm_int8_tokens(x, torch.ones(256, device=dev), 1e-5)
    assert bool(((t.scales.double() * 127 / 1e-8 - 1).abs() <= 32 * U).all())
    n = 1e-14 / 1e-5**0.5
    assert int(t.codes[0, 0]) == round(n * 127 / 1e-8)


def test_norm_of_rows_that_are_not_finite(op, dev):
    x = _randn(dev, 5, 4, 300)
    x[1, 7], x[2, 9] = float("nan"), float("-inf")
    t = op.rms_norm_int8_tokens(x, torch.ones(300, device=dev))
    v = op.dequantize_int8_tokens(t)
    assert torch.isnan(t.scales[1:3]).all() and torch.isnan(v[1:3]).all()
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 3, 4, 5, 257, 4097])
def test_norm_tokens_rows(op, dev, M, dtype):
    """Many rows are the rows one by one."""
    K = 640
    x, r, g = _randn(dev, M, M, K).to(dtype), _randn(dev, M + 1, M, K).to(dtype), 1 + 0.2 * _randn(dev, 9, K)
    t, h = op.add_rms_norm_int8_tokens(x, r, g)
    for m in {0, M // 2, M - 1}:
        one, h1 = op.add_rms_norm_int8_tokens(x[m : m + 1], r[m : m + 1], g)
        assert torch.equal(one.codes[0], t.codes[m]) and torch.equal(one.scales[0], t.scales[m])
        assert torch.equal(h1[0], h[m])
    assert torch.equal(h, (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,off", [(512, 1), (513, 0), (1000, 3), (4096, 1), (9001, 5)])
def test_tokens_of_views(op, dev, K, off, dtype):
    """Rows with a stride of their own from an address of the element's alignment only, columns taken apart, three
    dimensions, and h in place of either input."""
    M = 6
    base = _randn(dev, K, M, K + 11).to(dtype)
    x = base[:, off : off + K]
    r = _randn(dev, K + 1, M, 2 * K).to(dtype)[:, ::2]
    g = 1 + 0.2 * _randn(dev, 9, K)
    want, hw = op.add_rms_norm_int8_tokens(x.contiguous(), r.contiguous(), g)
    for a, b in ((x, r), (x.reshape(2, 3, K), r.reshape(2, 3, K))):
        got, h = op.add_rms_norm_int8_tokens(a, b, g)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        assert h.shape == a.shape and torch.equal(h.reshape(M, K), hw)
    q, qv = op.quantize_int8_tokens(x.contiguous()), op.quantize_int8_tokens(x)
    assert torch.equal(q.codes, qv.codes) and torch.equal(q.scales, qv.scales)
    before = base.clone()
    got, h = op.add_rms_norm_int8_tokens(x, r, g, out=x)  # over x, in its view
    assert h is x and torch.equal(x, hw) and torch.equal(got.codes, want.codes)
    base[:, off : off + K] = before[:, off : off + K]
    assert torch.equal(base, before)  # what lies around the view is left alone
    r2 = r.contiguous()
    got, h = op.add_rms_norm_int8_tokens(x, r2, g, out=r2)
    assert torch.equal(r2, hw) and torch.equal(got.codes, want.codes)
    v = torch.full((M, K + 9), 7.0, device=dev).to(dtype)
    op.dequantize_int8_tokens(q, dtype, out=v[:, 4 : 4 + K])
    assert torch.equal(v[:, 4 : 4 + K], op.dequantize_int8_tokens(q, dtype))
    assert bool((v[:, :4] == 7).all()) and bool((v[:, 4 + K :] == 7).all())


@pytest.mark.parametrize("K", [300, 5000, 20000])
def test_norm_of_rows_at_the_ends_of_the_range(op, dev, K):
    """Squares past fp32's largest value give a scale of NaN, not a wrong row; squares below its smallest are eps's."""
    x = _randn(dev, 5, 4, K)
    want = op.rms_norm_int8_tokens(x, torch.ones(K, device=dev))
    x[1] *= 1e25
    x[2] *= 1e-30
    t = op.rms_norm_int8_tokens(x, torch.ones(K, device=dev))
    assert torch.isnan(t.scales[1]) and torch.isnan(op.dequantize_int8_tokens(t)[1]).all()
    assert not t.codes[2].any() and abs(float(t.scales[2]) * 127 / 1e-8 - 1) <= 32 * U
    for i in (0, 3):
        assert torch.equal(t.codes[i], want.codes[i]) and torch.equal(t.scales[i], want.scales[i])


def test_norm_into_the_memory_around_an_input(op, dev):
    """h between the rows of the inputs, behind them and over them is right; across them it is refused."""
    M, K = 7, 200
    g = 1 + 0.2 * _randn(dev, 9, K)
    x, r = _randn(dev, 1, M, K), _randn(dev, 2, M, K)
    want, hw = op.add_rms_norm_int8_tokens(x, r, g)
    buf = torch.empty(2 * M, 3 * K, device=dev)
    a, b = buf[:M, :K], buf[:M, K : 2 * K]
    for out in (buf[:M, 2 * K :], buf[M:, :K], a, b):
        a.copy_(x), b.copy_(r)
        t, h = op.add_rms_norm_int8_tokens(a, b, g, out=out)
        assert torch.equal(h, hw) and torch.equal(t.codes, want.codes) and torch.equal(t.scales, want.scales)
    for out in (buf[1 : M + 1, :K], buf[:M, K - 1 : 2 * K - 1], buf[:M, 1 : K + 1], buf[:M, 2 * K - 1 : 3 * K - 1]):
        with pytest.raises(RuntimeError, match="over an input"):
            op.add_rms_norm_int8_tokens(a, b, g, out=out)
    one, _ = op.add_rms_norm_int8_tokens(x[:1], r[:1], g, out=r[:1])
    assert torch.equal(one.codes[0], want.codes[0])
    with pytest.raises(RuntimeError, match="over an input"):
        op.add_rms_norm_int8_tokens(buf[:1, :K], r[:1], g, out=buf[:1, 1 : K + 1])


def test_tokens_without_rows_or_columns(op, dev):
    t = op.quantize_int8_tokens(torch.empty(0, 64, device=dev))
    assert t.codes.shape == (0, 128) and op.dequantize_int8_tokens(t).shape == (0, 64)
    t = op.quantize_int8_tokens(torch.empty(3, 0, device=dev))
    assert torch.equal(t.scales, torch.full((3,), np.float32(1e-8) / np.float32(127), device=dev))
    with pytest.raises(ValueError):
        op.rms_norm_int8_tokens(torch.empty(3, 0, device=dev), torch.empty(0, device=dev))


# ---- channels ---------------------------------------------------------------

SHAPES = [(1, 1), (1, 64), (15, 17), (64, 16), (127, 63), (128, 64), (129, 65), (300, 1000), (1000, 300), (2048, 130)]


@pytest.mark.parametrize("K,N", SHAPES)
def test_channels(op, dev, K, N):
    w = _randn(dev, K + N, K, N) * 0.02
    if N > 3:
        w[:, 2] = 0
        w[0, 3] = float("nan")
    qw = op.quantize_int8_channels(w)
    code, top = _quantized(w.double().t().contiguous(), _floor(dev))
    assert torch.equal(op.unpack_int8_channels(qw).double(), code.t())
    assert torch.equal(qw.scales.double(), _f32(top[:, 0] / 127))
    assert torch.equal(op.dequantize_int8_channels(qw), _f32(code.t() * qw.scales.double()).float())
    # The layout: chunk (column block, k chunk, column) of sixteen k, zeros past K and N.
    Kp, Nb = -(-K // 128) * 128, -(-N // 16)
    full = torch.zeros(Kp, Nb * 16, dtype=torch.int8, device=dev)
    full[:K, :N] = code.t().to(torch.int8)
    model = full.reshape(Kp // 16, 16, Nb, 16).permute(2, 0, 3, 1).contiguous()
    assert torch.equal(qw.packed.view(torch.int8), model.reshape(-1))
    again = op.pack_int8_channels(op.unpack_int8_channels(qw), qw.scales)
    assert torch.equal(again.packed, qw.packed)
    bad = op.unpack_int8_channels(qw)
    bad[K - 1, N - 1] = 128
    with pytest.raises(RuntimeError, match="code"):
        op.pack_int8_channels(bad, qw.scales)


def test_channels_of_a_very_wide_weight(op, sgq, dev):
    """The widest weight, which has more columns than one launch has threads for: scales and fp32 codes."""
    N = 2**30
    w = torch.ones(1, N, device=dev)
    w[0, -3:] = torch.tensor([2.0, 0.0, -5.0], device=dev)
    lib = sgq.load_library()
    ws = torch.empty(lib.sgq_channels_workspace_bytes(1, N), dtype=torch.uint8, device=dev)
    scales, q = torch.full((N,), -1.0, device=dev), torch.zeros(1, N, device=dev)
    s = torch.cuda.current_stream().cuda_stream
    assert lib.sgq_quantize_channels(w.data_ptr(), 1, N, q.data_ptr(), scales.data_ptr(), None, ws.data_ptr(), ws.numel(), s) == 0
    one = float(np.float32(1) / np.float32(127))
    assert bool((scales[:-3] == one).all()) and bool((q[0, :-3] == 127).all())
    want = (np.array([2, 1e-8, 5], np.float32) / np.float32(127)).tolist()
    assert scales[-3:].tolist() == want and q[0, -3:].tolist() == [127.0, 0.0, -127.0]


# ---- products ---------------------------------------------------------------


def _problem(op, dev, M, K, N, seed, bias):
    cx, cw = _codes(dev, seed, M, K), _codes(dev, seed + 1, K, N)
    sx = torch.rand(M, generator=_gen(dev, seed + 2), device=dev) * 0.02 + 1e-4
    sw = torch.rand(N, generator=_gen(dev, seed + 3), device=dev) * 1e-3 + 1e-6
    b = _randn(dev, seed + 4, N) if bias else None
    return cx, cw, sx, sw, b


def _exact(cx, cw, sx, sw, b):
    """(product, product + bias) in 64 bits; integer sums below 2^53 are exact."""
    p = (cx.double() @ cw.double()) * sx.double()[:, None] * sw.double()
    return p, p if b is None else p + b.double()


def _error(p, y):
    """Roundings of (float)acc, * sx, * sw, + bias."""
    return 4 * U * p.abs() + U * y.abs() + 2.0**-149


def _check(got, want, tol, dtype):
    # fp16 stops at 65504: what rounds past it is infinite.
    assert got.dtype == dtype
    over = want.abs() > torch.finfo(dtype).max
    d = (got.double() - want).abs()
    ok = (d <= tol * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + TINY[dtype]) | over
    assert bool(ok.all()), float((d / (want.abs() + 1e-30))[~ok].max())


PRODUCTS = [(1, 64, 16), (1, 1, 1), (1, 4096, 100), (2, 129, 40), (3, 2048, 2048), (7, 1000, 513), (16, 512, 4096),
            (16, 11008, 48), (17, 256, 1000), (31, 384, 65), (33, 1500, 129), (64, 640, 256), (100, 2000, 300),
            (128, 1024, 1024), (129, 1024, 511), (200, 300, 1000), (256, 4096, 257), (257, 127, 512), (300, 5000, 640),
            (512, 2048, 2048), (513, 1023, 1025), (1000, 130, 4099), (2048, 512, 768), (1111, 2222, 3333), (40, 4099, 2050), (48, 4096, 4096), (60, 1000, 8003),
            (30, 1000, 8003), (600, 1100, 5000), (90, 14000, 1030), (130, 9000, 2000), (1030, 2048, 4096),
            (700, 8200, 4000), (2050, 4096, 4100), (1500, 14336, 1999), (520, 8192, 9000), (300, 11008, 4096),
            (70, 14000, 4100), (141, 24011, 5612), (1542, 268, 2433), (20, 3267, 34), (2240, 2949, 69)]


def test_products_take_every_form(op, sgq):
    """The shapes here run every kernel of the products, with K split and not (one weight and two together)."""
    import ctypes

    seen = set()
    for M, K, N in PRODUCTS:
        for gated in (0, 1):
            form, ks = ctypes.c_int(), ctypes.c_int()
            assert sgq.load_library().sgq_w8a8_plan(gated, M, K, N, 256, ctypes.byref(form), ctypes.byref(ks)) == 0
            seen.add((form.value, ks.value > 1))
    assert seen >= {(f, False) for f in range(1, 10)} | {(f, True) for f in (5, 7, 8, 9)}, sorted(seen)


@pytest.mark.parametrize("M,K,N", PRODUCTS)
@pytest.mark.parametrize("bias", [False, True])
def test_matmul(op, dev, M, K, N, bias):
    cx, cw, sx, sw, b = _problem(op, dev, M, K, N, M + K + N, bias)
    qw, t = op.pack_int8_channels(cw, sw), _tokens(op, cx, sx)
    p, y = _exact(cx, cw, sx, sw, b)
    for dtype in TYPES:
        _check(op.quantized_matmul_w8a8(t, qw, b, dtype), y, _error(p, y), dtype)


@pytest.mark.parametrize("M,K,N", PRODUCTS)
@pytest.mark.parametrize("bias", [False, True])
def test_swiglu(op, dev, M, K, N, bias):
    cx, cg, sx, sg, bg = _problem(op, dev, M, K, N, M + K + N, bias)
    _, cu, _, su, bu = _problem(op, dev, M, K, N, M + K + N + 50, bias)
    wg, wu, t = op.pack_int8_channels(cg, sg), op.pack_int8_channels(cu, su), _tokens(op, cx, sx)
    (pg, g), (pu, u) = _exact(cx, cg, sx, sg, bg), _exact(cx, cu, sx, su, bu)
    s = g * torch.sigmoid(g)
    # silu's slope is at most 1.1; its own exponential, sum and quotient take a few
    # roundings (the exponential's argument is exact), the product one.
    tol = u.abs() * (1.1 * _error(pg, g) + 8 * U * s.abs()) + s.abs() * _error(pu, u) + U * (s * u).abs()
    for dtype in TYPES:
        _check(op.quantized_swiglu_w8a8(t, wg, wu, bg, bu, dtype), s * u, tol, dtype)


# Forms of two column blocks a workgroup, with an odd number of blocks: the last workgroup's second one is past the weight.
ODD_BLOCKS = [(30, 1000, 8003), (60, 1000, 8003), (100, 2000, 300), (48, 1000, 5295), (59, 2048, 7278)]


def test_few_tokens_past_the_last_column_block(op, sgq, dev):
    import ctypes

    seen = set()
    for M, K, N in ODD_BLOCKS:
        cx, cw, sx, sw, b = _problem(op, dev, M, K, N, M + K, True)
        qw, t = op.pack_int8_channels(cw, sw), _tokens(op, cx, sx)
        p, y = _exact(cx, cw, sx, sw, b)
        _check(op.quantized_matmul_w8a8(t, qw, b), y, _error(p, y), torch.float32)
        # The weight's buffer ends with its last block.
        assert qw.packed.numel() == 16 * (-(-N // 16)) * 128 * (-(-K // 128)) and -(-N // 16) % 2 == 1
        for gated in (0, 1):
            form, ks = ctypes.c_int(), ctypes.c_int()
            assert sgq.load_library().sgq_w8a8_plan(gated, M, K, N, 256, ctypes.byref(form), ctypes.byref(ks)) == 0
            seen.add((gated, form.value))
        h = op.quantized_swiglu_w8a8(t, qw, qw, b, b)
        s = y * torch.sigmoid(y)
        _check(h, s * y, y.abs() * (1.1 * _error(p, y) + 8 * U * s.abs()) + s.abs() * _error(p, y) + U * (s * y).abs(),
               torch.float32)
    assert seen >= {(0, 3), (0, 4), (1, 3), (1, 4)}, sorted(seen)


def test_extreme_codes_and_scales(op, dev):
    """Every code -128 over the longest K: the sum comes within 128^2 of int32's end.  Scales of NaN and infinity
    reach their row or column only."""
    K, N, M = 131071, 33, 5
    cx = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    cw = torch.full((K, N), -128, dtype=torch.int8, device=dev)
    cw[:, 1] = 127
    sx, sw = torch.ones(M, device=dev), torch.ones(N, device=dev)
    y = op.quantized_matmul_w8a8(_tokens(op, cx, sx), op.pack_int8_channels(cw, sw))
    want = torch.full((M, N), float(np.float32(K * 16384)), device=dev)
    want[:, 1] = float(np.float32(-K * 128 * 127))
    assert torch.equal(y, want)
    sx[1], sw[2], sw[3] = float("nan"), float("inf"), 0.0
    y = op.quantized_matmul_w8a8(_tokens(op, cx, sx), op.pack_int8_channels(cw, sw))
    assert torch.isnan(y[1]).all() and torch.isinf(y[[0, 2, 3, 4], 2]).all() and not y[[0, 2, 3, 4], 3].any()
    assert torch.isfinite(y[[0, 2, 3, 4]][:, [0, 1, 3, 4]]).all()


@pytest.mark.parametrize("M", [1, 9, 40, 300])
def test_products_into_views(op, dev, M):
    """`out` with a stride of its own: what lies beside it and behind the last row is left alone."""
    K, N = 500, 321
    cx, cw, sx, sw, b = _problem(op, dev, M, K, N, M, True)
    qw, t = op.pack_int8_channels(cw, sw), _tokens(op, cx, sx)
    wide = op.TokensInt8(torch.zeros(M, 1024, dtype=torch.int8, device=dev)[:, 256:768], sx, K)
    wide.codes[:, :K] = cx
    for dtype in TYPES:
        want = op.quantized_matmul_w8a8(t, qw, b, dtype)
        buf = torch.full((M + 2, N + 7), 5.0, device=dev).to(dtype)
        got = op.quantized_matmul_w8a8(wide, qw, b, dtype, out=buf[:M, 3 : 3 + N])
        assert torch.equal(got, want)
        buf[:M, 3 : 3 + N] = 5.0
        assert bool((buf == 5).all())
        h = op.quantized_swiglu_w8a8(t, qw, qw, b, None, dtype)
        got = op.quantized_swiglu_w8a8(wide, qw, qw, b, None, dtype, out=buf[:M, 1 : 1 + N])
        assert torch.equal(got, h)
        buf[:M, 1 : 1 + N] = 5.0
        assert bool((buf == 5).all())


def test_products_without_rows_columns_or_sums(op, dev):
    sx, b = torch.ones(3, device=dev), _randn(dev, 1, 40)
    none = op.ChannelsInt8(torch.empty(16, dtype=torch.uint8, device=dev), torch.ones(40, device=dev), 0, 40)
    t = op.TokensInt8(torch.zeros(3, 128, dtype=torch.int8, device=dev), sx, 0)
    assert torch.equal(op.quantized_matmul_w8a8(t, none, b), b.expand(3, 40))
    assert not op.quantized_matmul_w8a8(t, none).any()
    h = op.quantized_swiglu_w8a8(t, none, none, b, b)
    assert torch.allclose(h, (b * torch.sigmoid(b) * b).expand(3, 40), rtol=1e-5)
    w = op.pack_int8_channels(_codes(dev, 2, 64, 40), torch.ones(40, device=dev))
    t0 = op.TokensInt8(torch.zeros(0, 128, dtype=torch.int8, device=dev), sx[:0], 64)
    assert op.quantized_matmul_w8a8(t0, w).shape == (0, 40)
    w0 = op.pack_int8_channels(_codes(dev, 2, 64, 0), torch.ones(0, device=dev))
    t3 = op.TokensInt8(torch.zeros(3, 128, dtype=torch.int8, device=dev), sx, 64)
    assert op.quantized_matmul_w8a8(t3, w0).shape == (3, 0)


def test_offsets_past_32_bits(op, dev):
    """Token codes, outputs and activations of more than 2^32 bytes."""
    K, N = 256, 24
    row, M = 65536, 70000
    codes = torch.zeros(M, row, dtype=torch.int8, device=dev)
    codes[-3:, :K] = _codes(dev, 1, 3, K)
    cw = _codes(dev, 2, K, N)
    sx, sw = torch.ones(M, device=dev), torch.ones(N, device=dev)
    y = torch.empty(M, 40000, device=dev, dtype=torch.bfloat16)[:, :N]
    op.quantized_matmul_w8a8(op.TokensInt8(codes, sx, K), op.pack_int8_channels(cw, sw), None, torch.bfloat16, out=y)
    want = codes[-3:, :K].double() @ cw.double()
    _check(y[-3:].contiguous(), want, U * want.abs(), torch.bfloat16)
    assert not y[:-3].any()
    x = torch.zeros(M, 40000, device=dev, dtype=torch.bfloat16)
    x[-1, :K] = torch.arange(K, device=dev)
    t = op.quantize_int8_tokens(x[:, :K])
    assert not t.codes[:-1].any()
    one = op.quantize_int8_tokens(x[-1:, :K].contiguous())
    assert torch.equal(one.codes[0], t.codes[-1]) and torch.equal(one.scales[0], t.scales[-1])


# ---- together ----------------------------------------------------------------


def _mlp(op, dev, D, H, dtype, seed=1):
    w = [_randn(dev, seed + i, *s) * 0.02 for i, s in enumerate([(D, H), (D, H), (H, D)])]
    norm = 1 + 0.1 * _randn(dev, seed + 5, D)
    return w, norm, op.QuantizedMLPInt8.from_float(*w, norm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 8, 130, 700])
def test_mlp(op, dev, M, dtype):
    """add, norm, gated MLP and down projection as they are used: the calls one after another, bit for bit, and
    near the float MLP in 64 bits.  Rounding to a step of max/127 has a standard error of at most
    1/sqrt(12) steps, that is 0.0023 of a row's maximum, or about 0.01 of the rms of normal values, whose
    maximum over a row is near 4 times that; two such tensors enter each product, and two products follow
    each other (the gate's and the up's in one), so the whole is off by well under 0.05 of its rms."""
    D, H = 512, 1408
    w, norm, mlp = _mlp(op, dev, D, H, dtype)
    x, r = _randn(dev, 11, M, D).to(dtype), _randn(dev, 12, M, D).to(dtype)
    out, h = mlp.forward(x, r)
    t, h2 = op.add_rms_norm_int8_tokens(x, r, norm)
    a = op.quantized_swiglu_w8a8(t, mlp.gate, mlp.up, dtype=dtype)
    y = op.quantized_matmul_w8a8(op.quantize_int8_tokens(a), mlp.down, dtype=dtype)
    assert torch.equal(h, h2) and torch.equal(out, y)
    f = h.double()
    n = f / torch.sqrt(f.pow(2).mean(1, keepdim=True) + 1e-5) * norm.double()
    g = n @ w[0].double()
    ref = (g * torch.sigmoid(g) * (n @ w[1].double())) @ w[2].double()
    assert float((out.double() - ref).norm() / ref.norm()) < 0.05
    first, h = mlp.forward(x)
    assert h is x and torch.equal(first, mlp.forward(x - x + x, torch.zeros_like(x))[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_mlp_of_sequences(op, dev, dtype):
    """Three dimensions, a padded batch seen through a view, and no tokens at all."""
    D, H = 256, 600
    _, _, mlp = _mlp(op, dev, D, H, dtype)
    x, r = _randn(dev, 11, 3, 9, D).to(dtype), _randn(dev, 12, 3, 9, D).to(dtype)
    out, h = mlp.forward(x[:, :5], r[:, :5])
    flat, fh = mlp.forward(x[:, :5].reshape(15, D), r[:, :5].reshape(15, D))
    assert out.shape == h.shape == (3, 5, D) and torch.equal(out.view(15, D), flat) and torch.equal(h.view(15, D), fh)
    for shape in ((0, D), (2, 0, D)):
        none = torch.empty(shape, dtype=dtype, device=dev)
        out, h = mlp.forward(none, none)
        assert out.shape == h.shape == shape and out.dtype == dtype
        assert mlp.forward(none)[0].shape == shape


def test_more_rows_and_columns_than_a_launch_takes(op, dev):
    """Products in slices: rows past 2^26, columns past 2^24."""
    M = 2**26 + 37
    x = torch.zeros(M, 1, device=dev)
    x[-40:, 0] = torch.arange(40, device=dev) - 20.0
    t = op.quantize_int8_tokens(x)
    w = op.pack_int8_channels(torch.tensor([[3, -2]], device=dev), torch.tensor([0.5, 1.0], device=dev))
    b = torch.tensor([0.0, 1.0], device=dev)
    y = op.quantized_matmul_w8a8(t, w, b, torch.bfloat16)
    want = op.quantized_matmul_w8a8(op.TokensInt8(t.codes[-40:], t.scales[-40:], 1), w, b, torch.bfloat16)
    assert torch.equal(y[-40:], want) and bool((want[:20, 0] < 0).all()) and bool((want[21:, 0] > 0).all())
    assert not y[:-40, 0].any() and bool((y[:-40, 1] == 1).all())
    del x, t, y
    N = 2**24 + 45
    cw = torch.zeros(1, N, dtype=torch.int8, device=dev)
    cw[0, -60:] = torch.arange(60, device=dev) - 30
    sw = torch.ones(N, device=dev)
    wide = op.pack_int8_channels(cw, sw)
    few = op.pack_int8_channels(cw[:, -60:], sw[-60:])
    b = torch.zeros(N, device=dev)
    b[-30:] = 0.25
    for m in (3, 40, 300):
        t = op.quantize_int8_tokens(_randn(dev, m, m, 1))
        y = op.quantized_matmul_w8a8(t, wide, b, torch.float16)
        assert torch.equal(y[:, -60:], op.quantized_matmul_w8a8(t, few, b[-60:], torch.float16)) and not y[:, :-60].any()
        y = op.quantized_swiglu_w8a8(t, wide, wide, b, None, torch.bfloat16)
        h = op.quantized_swiglu_w8a8(t, few, few, b[-60:], None, torch.bfloat16)
        assert torch.equal(y[:, -60:], h) and not y[:, :-60].any()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_graph_replays_match_eager(op, dev, M):
    """Two captured MLPs on one stream, replayed in turn on new inputs, with eager work between the replays."""
    D, H = 640, 1500
    _, _, mlp = _mlp(op, dev, D, H, torch.float32)
    xs = [_randn(dev, 20 + i, M, D) for i in range(4)]
    want = [mlp.forward(x, xs[0])[0] for x in xs]
    s = torch.cuda.Stream(dev)
    graphs = []
    for _ in range(2):
        x, r = xs[0].clone(), xs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y, _ = mlp.forward(x, r)
        graphs.append((g, x, r, y))
    for rep in range(3):
        for i, (g, x, r, y) in enumerate(graphs):
            k = 1 + (rep + i) % 3
            x.copy_(xs[k])
            y.fill_(float("nan"))
            eager = mlp.forward(xs[k], xs[0])[0]
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[k]) and torch.equal(eager, want[k]), (rep, i)


def test_graphs_and_threads_at_the_same_time(op, sgq, dev):
    """Two graphs of products that split K replayed on two streams at once, and eager calls of two host threads: each
    has partial sums of its own."""
    import threading

    M, K, N = 90, 14000, 1030
    assert sgq.load_library().sgq_linear_w8a8_workspace_bytes(M, K, N, 256) > 0
    qw = op.quantize_int8_channels(_randn(dev, 1, K, N))
    ts = [op.quantize_int8_tokens(_randn(dev, 2 + i, M, K)) for i in range(2)]
    want = [op.quantized_matmul_w8a8(t, qw) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    graphs, outs = [], []
    for s, t in zip(streams, ts):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(op.quantized_matmul_w8a8(t, qw))
        graphs.append(g)
    for _ in range(5):
        for y in outs:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(outs, want))
    got = [[], []]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i].append(op.quantized_matmul_w8a8(ts[i], qw))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 10 and all(torch.equal(y, want[i]) for y in got[i])


def test_other_stream(op, dev):
    D, H, M = 512, 1024, 64
    _, _, mlp = _mlp(op, dev, D, H, torch.float32)
    x = _randn(dev, 31, M, D)
    want = mlp.forward(x)[0]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    got = []
    for _ in range(4):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(mlp.forward(x)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals_on_the_device(op, dev):
    x = _randn(dev, 1, 4, 64)
    t = op.quantize_int8_tokens(x)
    w = op.quantize_int8_channels(_randn(dev, 2, 64, 32))
    w2 = op.quantize_int8_channels(_randn(dev, 2, 65, 32))
    with pytest.raises(ValueError):
        op.quantize_int8_tokens(x.double())
    with pytest.raises(ValueError):
        op.quantize_int8_tokens(x[0])
    with pytest.raises(ValueError):
        op.add_rms_norm_int8_tokens(x, x[:3], torch.ones(64, device=dev))
    with pytest.raises(ValueError):
        op.add_rms_norm_int8_tokens(x, x.bfloat16(), torch.ones(64, device=dev))
    with pytest.raises(ValueError):
        op.add_rms_norm_int8_tokens(x, x, torch.ones(64, device=dev), out=x[:, ::2])
    with pytest.raises(ValueError):
        op.rms_norm_int8_tokens(x, torch.ones(63, device=dev))
    with pytest.raises(ValueError):
        op.rms_norm_int8_tokens(x, torch.ones(64))
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w2)
    with pytest.raises(ValueError):
        op.quantized_swiglu_w8a8(t, w, w2)
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w, torch.ones(31, device=dev))
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w, dtype=torch.float64)
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w, out=torch.empty(4, 33, device=dev))
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w, out=torch.empty(4, 32, device=dev, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(t, w, out=torch.empty(32, 4, device=dev).t())
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(op.TokensInt8(t.codes[:, :64], t.scales, 64), w)  # no room for padding
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(op.TokensInt8(t.codes.float(), t.scales, 64), w)
    with pytest.raises(ValueError):
        op.quantized_matmul_w8a8(op.TokensInt8(t.codes, t.scales[:3], 64), w)
    for bad in ((w.packed[:-1], w.scales, 64, 32), (w.packed, w.scales[:31], 64, 32), (w.packed, w.scales.half(), 64, 32),
                (w.packed, w.scales, 129, 32), (w.packed, w.scales.cpu(), 64, 32), (w.packed.cpu(), w.scales, 64, 32),
                (w.packed[::2], w.scales, 64, 16), (w.packed, w.scales, 1 << 20, 32), (w.packed, w.scales, -1, 32)):
        with pytest.raises(ValueError):
            op.ChannelsInt8(*bad)
    odd = torch.zeros(4, 129, dtype=torch.int8, device=dev)
    with pytest.raises(RuntimeError, match="16"):
        op.quantized_matmul_w8a8(op.TokensInt8(odd[:, :128], t.scales, 64), w)  # rows of 129 bytes
