"""QuantizedAttentionInt8 as a layer of a program."""
import pytest
import torch

from test_attention_gpu import TYPES, _i32, _layers, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences", [0, 2])
@pytest.mark.parametrize("added", [False, True])
def test_no_tokens(op, dev, dtype, sequences, added):
    """A step without tokens is one like any other."""
    attn, mlp = _layers(op, dev, dtype, n=1)[0]
    kv = op.PagedKV(*(torch.full((4, 16, 2, 64), 3, dtype=dtype, device=dev) for _ in range(2)))
    batch = op.SequenceBatch(torch.zeros(sequences, 2, dtype=torch.int32, device=dev), _i32(dev, [5] * sequences),
                             _i32(dev, [0] * (sequences + 1)), 16, 1)
    x = torch.empty(0, 256, dtype=dtype, device=dev)
    y, h = attn.forward(x, kv, batch, residual=x.clone() if added else None)
    assert y.shape == h.shape == (0, 256) and y.dtype == dtype
    y, h = mlp.forward(y, residual=h)
    assert y.shape == (0, 256)
    assert bool((kv.k == 3).all() and (kv.v == 3).all())
