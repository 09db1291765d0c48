"""PagedKV and SequenceBatch as objects of a user's program: not changed, but copied."""
import copy
import pickle

import pytest
import torch

from test_attention_gpu import Batch, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


def test_attributes_are_not_assigned(op, dev):
    """An address kept of a tensor that the assignment frees would be read by the next call."""
    b = Batch(op, dev, [(1, 100)], 16, 2, 64, torch.bfloat16)
    for x, attrs in ((b.kv, ("k", "v", "head_dim")), (b.batch, ("table", "lens", "starts", "max_len", "max_new"))):
        for attr in attrs:
            old = getattr(x, attr)
            with pytest.raises(AttributeError):
                setattr(x, attr, old)
            assert getattr(x, attr) is old


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_copies_stand_for_their_own_tensors(op, dev, how):
    b = Batch(op, dev, [(3, 100), (1, 40)], 16, 2, 64, torch.bfloat16)
    q = _randn(dev, 1, 4, 4, 64).bfloat16()
    want = op.paged_attention(q, b.kv, b.batch)
    kv, batch = how(b.kv), how(b.batch)
    assert kv._struct.k == kv.k.data_ptr() and kv._struct.v == kv.v.data_ptr()
    assert batch._struct.table == batch.table.data_ptr() and batch._struct.lens == batch.lens.data_ptr()
    if how is not copy.copy:
        assert kv.k.data_ptr() != b.k.data_ptr()
        b.k.fill_(0), b.v.fill_(0), b.batch.lens.fill_(1), b.table.fill_(0)
    assert torch.equal(op.paged_attention(q, kv, batch), want)
