"""Per-sequence and per-row numbers of every type of whole numbers."""
import pytest
import torch


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64])
def test_numbers_keep_their_values(op, dtype):
    top = torch.iinfo(dtype).max
    t = torch.tensor([top, 0, 5], dtype=dtype)
    got = op._int32(t, 3, t.device, "first_key")
    assert got.dtype is torch.int32 and got.tolist() == [min(top, 2**31 - 1), 0, 5]


@pytest.mark.parametrize("dtype", [torch.uint64, torch.float32, torch.bool, torch.complex64])
def test_others_are_refused(op, dtype):
    t = torch.zeros(3, dtype=dtype)
    with pytest.raises(ValueError, match="whole numbers"):
        op._int32(t, 3, t.device, "prefix")


def test_most_sequences_and_heads_of_one_call(op, sgq):
    """2^24 workgroups are refused: 2^20 sequences of 16 kv heads."""
    from test_attention_cpu import UNSUPPORTED, _attend

    lib = sgq.load_library()
    call = dict(cache=dict(kv_heads=16, token_stride=1024, page_stride=16384), heads=16, q_row=1024, o_row=1024,
                out=1 << 40)  # behind all rows of q
    assert _attend(op, lib, seqs=dict(B=1 << 20, max_new=1), **call) == UNSUPPORTED
    assert b"too many sequences" in lib.sgq_last_error()
    assert _attend(op, lib, seqs=dict(B=1 << 20, max_new=64), rows=1 << 20, **call) == UNSUPPORTED
