"""Values and scores at the ends of the types' ranges, in every form of attention over a paged cache.

Exact weights are positive, however small: a NaN among the values that a row sees makes that column of
the row NaN, an infinity that infinity, infinities of both signs NaN.  It may not depend on whether fp32
has the weight, or on how a call's keys are shared out.  Tolerances of finite columns are those of
test_attention_gpu.
"""
import math

import pytest
import torch

from test_attention_gpu import TYPES, Batch, _check, _i32, _randn, _reference

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


def _put(b, seq=0):
    """The sequence's values (and keys) into their pages again."""
    n = b.seqs[seq][1]
    j = torch.arange(n, device=b.dev)
    at = b.table[seq, j // b.page].long(), j % b.page
    b.k[at], b.v[at] = b.keys[seq], b.values[seq]


def _expect(b, y, q, bad, dtype, **how):
    """bad: {column: what it is} for every row; the other columns against 64 bits."""
    for col, want in bad.items():
        got = y[..., col].float()
        ok = got.isnan() if math.isnan(want) else got == want
        assert bool(ok.all()), f"column {col}: {got.flatten()[~ok.flatten()][:4].tolist()} for {want}"
    for v in b.values:
        v.copy_(torch.where(torch.isfinite(v), v, 0))
    out, A, ds, n = _reference(b, q, **how)
    hit = torch.zeros(y.shape[-1], dtype=torch.bool, device=y.device)
    hit[list(bad)] = True
    _check(torch.where(hit, out, y.double()), (out, A, ds, n), b, dtype)


# (new, keys): lanes or few rows, few rows in fp32 too, tiles; keys in one piece and shared out.
SEQS = [(1, 90), (1, 4000), (6, 90), (6, 4000), (40, 90), (40, 4000), (150, 700)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seq", SEQS)
@pytest.mark.parametrize("where", ["bias", "low", "early"])
def test_seen_values_that_are_not_finite_whatever_their_weight(op, dev, seq, dtype, where):
    """Keys whose weights are far below fp32's range, by a bias, by their scores, or by a maximum that comes
    later: at the beginning, in the middle, in the last page that all rows see."""
    new, n = seq
    d, last = 64, n - new
    b = Batch(op, dev, [seq], 16, 1, d, dtype)
    q = _randn(dev, 3, new, 2, d).to(dtype)
    b.keys[0][..., 0], q[..., 0] = 0, 8
    keys = {0: (1, INF), last // 2: (2, -INF), max(last - 1, 0): (3, NAN)}
    how = dict(scale=1.0)
    if where == "bias":  # 50 keys from every row, e^-700
        how["alibi_slopes"] = torch.full((2,), 14.0, device=dev)
        keys = {k: c for k, c in keys.items() if k <= n - new - 50}
    else:
        b.keys[0][..., 1:] = 0
        for k in list(keys) + [1]:
            b.keys[0][k, :, 0] = -40 if where == "low" else 0
        if where == "early":
            b.keys[0][last, :, 0] = 40  # all rows see it
    keys[1] = (4, INF)
    b.values[0][1, 0, 5] = INF
    for k, (col, value) in keys.items():
        b.values[0][k, 0, col] = value
    b.values[0][max(k for k in keys if k != 1), 0, 5] = -INF
    _put(b)
    bad = {col: value for col, value in keys.values()}
    bad[5] = NAN
    y = op.paged_attention(q, b.kv, b.batch, **how)
    _expect(b, y, q, bad, dtype, **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 6, 40])
def test_they_do_not_reach_rows_that_do_not_see_them(op, dev, dtype, new):
    """Weights below fp32's range again, and half of the rows begin behind the key."""
    n, d = 4000, 64
    b = Batch(op, dev, [(new, n), (2, 50)], 16, 1, d, dtype)
    q = _randn(dev, 3, b.rows, 4, d).to(dtype)
    how = dict(alibi_slopes=torch.full((4,), 0.25, device=dev))
    b.values[0][500, 0, 7] = INF
    _put(b)
    first = [0 if i % 2 == 0 else 501 for i in range(b.rows)]
    how["first_key"] = _i32(dev, first)
    y = op.paged_attention(q, b.kv, b.batch, **how)
    sees = torch.tensor([f == 0 for f in first], device=dev)
    sees[new:] = False
    assert bool((y[sees][..., 7] == INF).all())
    b.values[0][500, 0, 7] = 0
    out, A, ds, cnt = _reference(b, q, **how)
    hit = sees[:, None, None] & (torch.arange(d, device=dev) == 7)
    _check(torch.where(hit, out, y.double()), (out, A, ds, cnt), b, dtype)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("seq", SEQS + [(1, 131072), (6, 131072)])
def test_large_values_under_a_maximum_that_grows(op, dev, seq, dtype):
    """Values of 2^123 whose weights, of 1 at most, sum to less than 4: the sums stay within fp32, also where the largest
    score comes after one that is 5 (2^7.2) less."""
    new, n = seq
    b = Batch(op, dev, [seq], 16, 1, 64, dtype)
    top = 128 if n > 300 else n - new  # a later tile, of the same wavefront where keys are many
    k = b.keys[0]
    k.zero_()
    k[..., 0] = -20
    k[0, :, 0], k[top, :, 0] = -0.625, 0  # scores of -160, -5, 0
    b.values[0].copy_(b.values[0].sign() * 2.0**123)
    _put(b)
    q = torch.zeros(new, 2, 64, dtype=dtype, device=dev)
    q[..., 0] = 8
    y = op.paged_attention(q, b.kv, b.batch, scale=1.0)
    assert bool(torch.isfinite(y).all())
    _check(y, _reference(b, q, scale=1.0), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seq", SEQS)
@pytest.mark.parametrize("bias", [False, True])
def test_scores_of_many_digits(op, dev, seq, dtype, bias):
    """Scores of up to 2^33 (fp16) and 2^50, whose differences fp32 still has: the largest takes it all, and its value comes out
    as it is."""
    new, n = seq
    big = 2.0**15 if dtype is torch.float16 else 2.0**23
    b = Batch(op, dev, [seq], 16, 1, 64, dtype)
    top = (n - new) // 2
    b.keys[0].copy_(b.keys[0].sign() * big)
    b.keys[0][top] = big
    q = (0.5 + _randn(dev, 3, new, 2, 1).abs().clamp(max=3) / 4) * big  # up to 1.25 of it
    q = q.expand(-1, -1, 64).contiguous().to(dtype)
    _put(b)
    # The next score is at least two of 64 terms below.
    assert int((b.keys[0] > 0).sum(-1).kthvalue(n - 1, 0).values) <= 62
    how = dict(alibi_slopes=torch.full((2,), 0.5, device=dev)) if bias else {}
    y = op.paged_attention(q, b.kv, b.batch, **how)
    assert torch.equal(y, b.values[0][top].expand_as(y))


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("seq", SEQS + [(1, 131072), (6, 131072)])
@pytest.mark.parametrize("bias", [False, True])
def test_means_of_the_largest_values(op, dev, seq, dtype, bias):
    """Values of 2^127 and more, whose mean fp32 holds and whose sum it does not; beside them columns of ordinary ones."""
    new, n = seq
    b = Batch(op, dev, [seq], 16, 1, 64, dtype)
    v = b.values[0]
    big = torch.arange(64, device=dev) % 3 != 1
    v.copy_(torch.where(big, ((1 + v.float().abs().clamp(max=1) / 2) * 2.0**127) * v[0].float().sign(), v.float()))
    _put(b)
    q = (_randn(dev, 3, new, 2, 64) / 4).to(dtype)
    how = dict(alibi_slopes=torch.full((2,), 0.003, device=dev)) if bias else {}
    y = op.paged_attention(q, b.kv, b.batch, **how)
    assert bool(torch.isfinite(y).all())
    _check(y, _reference(b, q, **how), b, dtype)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("new", [1, 6, 40])
def test_large_values_of_one_part_of_the_keys(op, dev, dtype, new):
    """Only one workgroup's keys have sums past fp32, and the others' are joined to them."""
    n = 131072
    b = Batch(op, dev, [(new, n)], 16, 1, 64, dtype)
    b.values[0][40000:44000] = 2.0**127
    b.values[0][40000:44000, :, 3] = 1
    _put(b)
    q = (_randn(dev, 3, new, 2, 64) / 4).to(dtype)
    y = op.paged_attention(q, b.kv, b.batch)
    assert bool(torch.isfinite(y).all())
    _check(y, _reference(b, q), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new, n", [(1, 3), (3, 5), (1, 2000), (7, 60), (60, 64), (300, 900)])
@pytest.mark.parametrize("alike", [False, True])
def test_a_mean_of_the_largest_value_is_no_infinity(op, dev, dtype, new, n, alike):
    """Columns of one value, the type's largest of either sign: rounded weights may sum to more than their sum, by half a step,
    and what comes out is that value or less by as much (and the sums' roundings).  alike: all keys but the first are, so that
    their weights are rounded the same way."""
    b = Batch(op, dev, [(new, n)] * 4, 16, 1, 64, dtype)
    top = torch.finfo(dtype).max
    for i in range(4):
        b.values[i][..., ::2], b.values[i][..., 1::2] = top, -top
        if alike:
            b.keys[i][:], b.keys[i][0] = 0.125, 0.25
        _put(b, i)
    q = _randn(dev, 3, b.rows, 8, 64).abs().to(dtype)
    y = op.paged_attention(q, b.kv, b.batch)
    assert bool(torch.isfinite(y).all()), int((~torch.isfinite(y)).sum())
    sign = 1.0 - 2.0 * (torch.arange(64, device=dev) % 2)
    low = top * (1 - 2 * torch.finfo(dtype).eps - (n + 16) * 2.0**-24)
    assert float((y.double() * sign).min()) >= low
