"""8-bit tokens of a norm without eps, whose rows may have no maximum."""
import pytest
import torch

from test_w8a8_gpu import TYPES, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1, 7, 100, 1000, 5003, 20001])
def test_norm_without_eps_of_rows_of_nothing(op, dev, K, dtype):
    """eps = 0 and a row of zeros: the norm is no number, and the scale says so; the codes past K are zero as ever.  Rows
    whose squares vanish have an infinite norm, of the right sign."""
    x = _randn(dev, K, 4, K).to(dtype)
    x[1] = 0
    t = op.rms_norm_int8_tokens(x, torch.ones(K, device=dev), 0.0)
    assert torch.isnan(t.scales[1]) and torch.isnan(op.dequantize_int8_tokens(t)[1]).all()
    assert torch.isfinite(t.scales[[0, 2, 3]]).all() and not t.codes[:, K:].any()
    if dtype is torch.float32:
        x[2] = torch.where(x[2] < 0, -1e-38, 1e-38)
        t = op.rms_norm_int8_tokens(x, torch.ones(K, device=dev), 0.0)
        v = op.dequantize_int8_tokens(t)
        assert torch.isinf(v[2]).all() and torch.equal(torch.sign(v[2]), torch.sign(x[2])) and not t.codes[:, K:].any()
