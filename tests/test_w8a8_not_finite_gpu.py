"""Values that are not finite, or not held by fp32, on their way through 8-bit activations: they stay visible in what
comes out, and reach their own rows only."""
import pytest
import torch

from test_w8a8_gpu import TYPES, _mlp, _randn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_mlp_keeps_rows_that_are_not_finite(op, dev, M, dtype):
    """A row with a NaN or an infinity, or one whose squares pass fp32, has a norm of NaN in every value, and so has
    the MLP; the other rows are those of a batch without it."""
    D, H = 512, 1408
    _, _, mlp = _mlp(op, dev, D, H, dtype)
    x, r = _randn(dev, 11, M, D).to(dtype), _randn(dev, 12, M, D).to(dtype)
    clean = mlp.forward(x, r)[0]
    bad = {0: NAN, 1: INF, 3: -INF}
    if dtype is not torch.float16:
        bad[4] = 1e25  # finite; its square is not
    bad = {m: v for m, v in bad.items() if m < M}
    for m, v in bad.items():
        x[m, (37 * m + 5) % D] = v
    for out in (mlp.forward(x, r)[0], mlp.forward(x + r)[0]):
        assert torch.isnan(out[list(bad)]).all()
    rest = [m for m in range(M) if m not in bad]
    assert torch.equal(mlp.forward(x, r)[0][rest], clean[rest]) and torch.isfinite(clean).all()


@pytest.mark.parametrize("M", [2, 40])
def test_mlp_whose_hidden_values_pass_the_type(op, dev, M):
    """gate and up of 512 each: 2^18 is past fp16, and what follows is not a number."""
    D, H = 512, 640
    ones = [torch.ones(s, device=dev) for s in ((D, H), (D, H), (H, D))]
    mlp = op.QuantizedMLPInt8.from_float(*ones, torch.ones(D, device=dev))
    x = torch.ones(M, D, device=dev, dtype=torch.float16)
    x[1] = 0
    out, _ = mlp.forward(x)
    assert torch.isnan(out[0]).all() and not out[1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1, 7, 129, 512, 1025, 2500, 4099, 8193, 20000, 33000])
def test_tokens_that_keep_nan(op, dev, K, dtype):
    """keep_nan: rows with a NaN or an infinity in any place have a scale of NaN, every other row is as without it."""
    M = 7
    x = (_randn(dev, K, M, K) * 3).to(dtype)
    x[1] = 0
    x[2, K - 1], x[3, 0], x[4, K // 2], x[5, (3 * K) // 4] = NAN, INF, -INF, -NAN
    t = op.quantize_int8_tokens(x, keep_nan=True)
    plain = op.quantize_int8_tokens(x)
    good, bad = [0, 1, 6], [2, 3, 4, 5]
    assert torch.isnan(t.scales[bad]).all() and torch.isnan(op.dequantize_int8_tokens(t, dtype)[bad]).all()
    assert torch.equal(t.codes[good], plain.codes[good]) and torch.equal(t.scales[good], plain.scales[good])
    assert not t.codes[:, K:].any()
    none = op.quantize_int8_tokens(x[:, :0], keep_nan=True)
    assert torch.equal(none.scales, op.quantize_int8_tokens(x[:, :0]).scales)
    assert op.quantize_int8_tokens(x[:0], keep_nan=True).codes.shape[0] == 0
