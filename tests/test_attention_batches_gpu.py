"""Batches of attention over a paged cache as a server has them: many sequences, chunks beside single tokens, results in q's place."""
import pytest
import torch

from test_attention_gpu import SHAPES, TYPES, Batch, _check, _i32, _randn, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


def _shared_out(op, b, H):
    """Whether the call's keys are shared out over several workgroups."""
    return op._attention_workspace(b.kv, b.batch, b.rows, H, 0, b.dev)[1] > 0


# form: (new tokens of sequence i, longest, heads)
FORMS = {"tiles": (lambda i: (0, 17, 40, 1, 129)[i % 5], 300, 2), "few": (lambda i: (1, 0, 4, 1)[i % 4], 900, 2),
         "lanes": (lambda i: (1, 0, 2)[i % 3], 900, 2)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("count", [64, 65, 130, 257])
def test_many_sequences(op, dev, count, form, dtype):
    """Workgroups find their sequence and tile among more sequences than a wavefront has lanes, some without tokens."""
    new, longest, H = FORMS[form]
    seqs = [(new(i), max(new(i), 1 + 37 * i % longest)) for i in range(count)]
    seqs[-1] = (seqs[1][0] or 1, longest)
    b = Batch(op, dev, seqs, 16, 1, 32, dtype, pad=3)
    q = _randn(dev, 5, b.rows, H, 32).to(dtype)
    out = torch.full_like(q, 7)
    op.paged_attention(q, b.kv, b.batch, out=out)
    if form != "tiles":
        assert _shared_out(op, b, H)
    _check(out, _reference(b, q), b, dtype, f"{count} sequences")
    assert bool((out[-3:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [65, 70])
def test_many_sequences_whose_tiles_share_out_their_keys(op, dev, count, dtype):
    seqs = [(0, 30)] * (count - 3) + [(20, 2000), (0, 0), (33, 1500)]
    b = Batch(op, dev, seqs, 16, 1, 64, dtype)
    q = _randn(dev, 5, b.rows, 2, 64).to(dtype)
    assert _shared_out(op, b, 2)
    _check(op.paged_attention(q, b.kv, b.batch), _reference(b, q), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_chunk_beside_single_tokens(op, dev, dtype):
    seqs = [(1, 1 + 61 * i % 700) for i in range(40)]
    seqs[17] = (333, 1000)
    b = Batch(op, dev, seqs, 16, 2, 128, dtype)
    q = _randn(dev, 5, b.rows, 8, 128).to(dtype)
    _check(op.paged_attention(q, b.kv, b.batch), _reference(b, q), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_results_in_the_place_of_q(op, dev, shape, dtype):
    """out may be q itself, by itself and as a part of a projection's rows, of which the rest stays."""
    seqs, page, H, KV, d = SHAPES[shape]
    b = Batch(op, dev, seqs, page, KV, d, dtype, seed=shape, pad=2)
    T = b.starts[-1]
    q = (_randn(dev, 77, b.rows, H, d) * 2).to(dtype)
    want = op.paged_attention(q, b.kv, b.batch)
    want[T:] = q[T:]  # rows of no sequence
    for _ in range(3):
        y = q.clone()
        assert op.paged_attention(y, b.kv, b.batch, out=y) is y
        assert torch.equal(y, want)
        rows = torch.full((b.rows, H + 2 * KV, d), 5, dtype=dtype, device=dev)
        rows[:, :H] = q
        op.paged_attention(rows[:, :H], b.kv, b.batch, out=rows[:, :H])
        assert torch.equal(rows[:, :H], want) and bool((rows[:, H:] == 5).all())


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint8])
def test_limits_of_other_types(op, dev, dtype):
    b = Batch(op, dev, [(4, 50), (1, 30)], 16, 2, 64, torch.float16)
    q = _randn(dev, 1, 5, 4, 64).half()
    for how in (dict(prefix=[48, 3]), dict(first_key=[0, 20, 47, 200, 9])):
        want = op.paged_attention(q, b.kv, b.batch, **{k: _i32(dev, v) for k, v in how.items()})
        got = op.paged_attention(q, b.kv, b.batch, **{k: _i32(dev, v).to(dtype) for k, v in how.items()})
        assert torch.equal(got, want)
    if dtype is torch.uint32:  # behind every key
        far = torch.full((5,), 2**32 - 1, dtype=torch.int64, device=dev).to(dtype)
        assert bool((op.paged_attention(q, b.kv, b.batch, first_key=far) == 0).all())
