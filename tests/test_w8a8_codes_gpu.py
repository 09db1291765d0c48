"""Which codes pack_int8_channels takes for whole numbers in [-128, 127]."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


def test_codes_that_are_whole_only_in_fp32(op, dev):
    """Codes of a wider type are looked at in that type."""
    scales = torch.ones(5, device=dev)
    codes = torch.arange(20, device=dev, dtype=torch.float64).reshape(4, 5) - 10
    want = op.pack_int8_channels(codes.float(), scales)
    for dtype in (torch.float64, torch.int64, torch.int16, torch.int8, torch.bfloat16, torch.float16):
        assert torch.equal(op.pack_int8_channels(codes.to(dtype), scales).packed, want.packed)
    for v in (3.00000001, 127.000001, -128.000001, 1e-40, 1e300, float("inf"), -float("inf"), float("nan")):
        bad = codes.clone()
        bad[2, 3] = v
        with pytest.raises(RuntimeError, match="code"):
            op.pack_int8_channels(bad, scales)
        with pytest.raises(RuntimeError, match="code"):
            op.pack_int8_channels(bad.t().contiguous().t(), scales)
    for v in (2**40, -(2**62), 128, -129):
        bad = codes.long()
        bad[0, 0] = v
        with pytest.raises(RuntimeError, match="code"):
            op.pack_int8_channels(bad, scales)
    with pytest.raises(ValueError, match="complex"):
        op.pack_int8_channels(codes.to(torch.complex64), scales)
    with pytest.raises(ValueError, match="complex"):
        op.quantize_int8_channels(codes.to(torch.complex64))
