"""Which rows the norm, rotation and append and the attention over a paged cache write."""
import pytest
import torch

from test_attention_gpu import TYPES, Batch, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [2, 40])
def test_rows_before_the_first_sequence_stay(op, dev, dtype, new):
    """Rows before starts[0] are of no sequence, also where the first breaks a bound."""
    b = Batch(op, dev, [(new, 50), (new, 60)], 16, 2, 64, dtype)
    rows = 3 + 2 * new
    q, k, v = (_randn(dev, i, rows, h, 64).to(dtype) for i, h in enumerate((4, 2, 2)))
    starts = _i32(dev, [3, 3 + new, rows])
    for lens, broken in (((50, 60), False), ((61, 60), True), ((-1, 60), True)):
        batch = op.SequenceBatch(b.table, _i32(dev, lens), starts, 60, new)
        for run in (lambda out: op.norm_rope_append(q, k, v, b.kv, batch, out=out),
                    lambda out: op.paged_attention(q, b.kv, batch, out=out)):
            out = run(torch.full_like(q, 7))
            assert bool((out[:3] == 7).all()), lens
            assert bool(out[3 : 3 + new].isnan().all()) == broken
            assert bool(torch.isfinite(out[3 + new :]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("d, rot", [(64, 0), (64, 32), (128, 96), (80, 20), (16, 2), (256, 64)])
def test_what_is_not_turned_is_of_no_other_element(op, dev, d, rot, interleaved, value, dtype):
    """Elements behind the turned ones come as they are, whatever stands beside them."""
    b = Batch(op, dev, [(4, 30)], 16, 2, d, dtype)
    q, k = (_randn(dev, i, 4, h, d).to(dtype) for i, h in enumerate((4, 2)))
    q[0, 0, rot], q[1, 1, -1], q[2, 2, (rot + d) // 2], k[0, 1, rot] = value, value, value, value
    q[3, 3, -3] = -0.0
    freqs = op.rotary_frequencies(rot, device=dev) if rot else None
    out = op.norm_rope_append(q, k, k, b.kv, b.batch, freqs, interleaved=interleaved)
    pos = torch.arange(26, 30, device=dev)
    kept = b.k[b.table[0, pos // 16].long(), pos % 16]
    bits = torch.int32 if dtype is torch.float32 else torch.int16
    for got, x in ((out, q), (kept, k)):
        assert torch.equal(got[..., rot:].contiguous().view(bits), x[..., rot:].contiguous().view(bits))
        assert bool(torch.isfinite(got[..., :rot]).all())
