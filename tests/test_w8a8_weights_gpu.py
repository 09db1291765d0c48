"""8-bit channels from the framework's other INT8 weights."""
import pytest
import torch

from test_w8a8_gpu import _error, _exact, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


def test_channels_of_a_weight_quantized_per_tensor(op, sgq, dev):
    """A QuantizedTensor with one scale: its codes, that scale for each column."""
    w = _randn(dev, 1, 300, 200) * 0.02
    qt = sgq.quantize_int8(w, sgq.PER_TENSOR)
    qw = op.pack_int8_channels(sgq.unpack_codes(qt), qt.scales.expand(200))
    assert torch.equal(op.dequantize_int8_channels(qw), sgq.dequantize_int8(qt))
    x = _randn(dev, 2, 9, 300)
    t = op.quantize_int8_tokens(x)
    p, y = _exact(t.codes[:, :300], qt.qdata, t.scales, qt.scales.expand(200), None)
    assert bool(((op.quantized_matmul_w8a8(t, qw).double() - y).abs() <= _error(p, y)).all())
