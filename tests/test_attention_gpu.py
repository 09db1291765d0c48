"""Attention over a paged cache, and the norm, rotation and append before it, against 64 bits.

Tolerances, with U = 2^-24 and h half a step of the type (0 for fp32, where the last
rounding is one of U).  Attention: a score's error is at most
  ds = U ((d + 8) S + 8 (bias + cap)),  S = max over the keys of scale * sum |q| |k|
(a sum of d products in any order, the scaling, the base of the exponential), and moves a weight by
a factor of e^(2 ds); a weight is rounded to the type before its product (h; for fp16 below 2^-21 by
2^-32 at most, n of them, where the largest weight is at least 1), and sums of n terms are off by n U of
sum p |v| = A.  So |out - ref| <= A (h + 2 ds + (n + 16) U) + h |ref| + the smallest step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _randn(dev, seed, *shape):
    return torch.randn(*shape, generator=_gen(dev, seed), device=dev)


def _i32(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Batch:
    """Sequences of (new, keys) in pages of a pool in no order; whatever is of no key is `hole`."""

    def __init__(self, op, dev, seqs, page, kv_heads, d, dtype, seed=0, hole=float("nan"), head_major=False, pad=0,
                 max_len=None, max_new=None, kv=None):
        self.seqs, self.page, self.dev = seqs, page, dev
        used = [-(-n // page) for _, n in seqs]
        pool = sum(used) + 3
        order = torch.randperm(pool, generator=_gen(dev, seed), device=dev).int()
        self.table = torch.full((len(seqs), max(used + [1]) + 1), -7, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at : at + n]
            at += n
        shape = (pool, kv_heads, page, d) if head_major else (pool, page, kv_heads, d)
        self.k, self.v = (torch.full(shape, hole, dtype=dtype, device=dev) for _ in range(2))
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.keys, self.values = [], []
        for b, (_, n) in enumerate(seqs):
            k = kv[0][b] if kv else _randn(dev, 10 * b + seed, n, kv_heads, d).to(dtype)
            v = kv[1][b] if kv else _randn(dev, 10 * b + seed + 1, n, kv_heads, d).to(dtype)
            self.keys.append(k)
            self.values.append(v)
            j = torch.arange(n, device=dev)
            self.k[self.table[b, j // page].long(), j % page] = k
            self.v[self.table[b, j // page].long(), j % page] = v
        self.starts = [0]
        for n, _ in seqs:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + pad
        self.kv = op.PagedKV(self.k, self.v)
        self.batch = op.SequenceBatch(self.table, _i32(dev, [n for _, n in seqs]), _i32(dev, self.starts),
                                      max([n for _, n in seqs] + [1]) if max_len is None else max_len,
                                      max([n for n, _ in seqs] + [1]) if max_new is None else max_new)


def _reference(b, q, scale=None, softcap=0.0, alibi_slopes=None, window=0, prefix=None, first_key=None):
    """(out, A, ds, n) in 64 bits, rows of no sequence left zero."""
    T, H, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(T, H, d, dtype=torch.float64, device=q.device)
    A, ds, cnt = torch.zeros_like(out), torch.zeros(T, H, 1, device=q.device).double(), torch.zeros(T, 1, 1, device=q.device).double()
    for i, (n, length) in enumerate(b.seqs):
        if n == 0:
            continue
        rows = slice(b.starts[i], b.starts[i + 1])
        p = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)
        seen = j <= p
        if prefix is not None:
            seen = seen | (j < int(prefix[i]))
        if window:
            seen = seen & (j > p - window)
        if first_key is not None:
            seen = seen & (j >= first_key[rows, None])
        KV = b.keys[i].shape[1]
        k = b.keys[i].double().repeat_interleave(H // KV, 1)
        v = b.values[i].double().repeat_interleave(H // KV, 1)
        for h in range(H):
            s = q[rows, h].double() @ k[:, h].T * scale
            mag = (q[rows, h].double().abs() @ k[:, h].abs().T * abs(scale)).masked_fill(~seen, 0).nan_to_num(0, 0, 0)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            bias = 0.0
            if alibi_slopes is not None:
                away = (p - j).abs().double() * float(alibi_slopes[h])
                s = s - away
                bias = away.masked_fill(~seen, 0).abs().amax(-1, keepdim=True)
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(top == -math.inf, 0.0, top)).masked_fill(~seen, 0)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total > 0, w / total, w)  # NaN stays
            w = torch.where(total.isnan(), total, w)
            # What a row does not see counts for nothing, whatever it is.
            bad = ~torch.isfinite(v[:, h]).all(-1)
            clean = torch.where(bad[:, None], 0.0, v[:, h])
            out[rows, h] = w @ clean
            for key in bad.nonzero()[:, 0].tolist():
                out[rows, h] += torch.where(seen[:, key, None], w[:, key, None] * v[key, h], 0.0)
            A[rows, h] = w @ clean.abs()
            ds[rows, h] = U * ((d + 8) * mag.amax(-1, keepdim=True) + 8 * (bias + softcap))
        cnt[rows] = seen.sum(-1).double()[:, None, None]
    return out, A, ds, cnt


def _check(y, ref, b, dtype, what=""):
    out, A, ds, n = ref
    T = b.starts[-1]
    y, out, A, ds, n = y[:T].double(), out[:T], A[:T], ds[:T], n[:T]
    h = HALF[dtype]
    tol = A * (h + 2 * ds + (n + 16) * U) + (h + U) * out.abs() + TINY[dtype]
    if dtype is torch.float16:
        vmax = max((float(v.double().abs().nan_to_num(0, 0, 0).max()) for v in b.values if v.numel()), default=0.0)
        tol = tol + n * 2.0**-32 * vmax
    bad = ~((y - out).abs() <= tol) & ~(y.isnan() & out.isnan()) & ~(y == out)
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        worst = ((y - out).abs() / tol).nan_to_num(0, 0, 0).max()
        raise AssertionError(f"{what} at {at}: {float(y[tuple(at)])} for {float(out[tuple(at)])}, {int(bad.sum())} bad, worst {float(worst)}")


# ---- attention -------------------------------------------------------------

SHAPES = [  # sequences (new, keys), page, heads, kv_heads, head_dim
    ([(1, 1)], 16, 1, 1, 64),
    ([(1, 2), (1, 1), (1, 33)], 16, 4, 2, 128),
    ([(1, 1000), (1, 64), (1, 65), (1, 63), (1, 513)], 16, 8, 2, 128),
    ([(1, 300)] * 3, 8, 16, 16, 64),
    ([(2, 100), (0, 50), (3, 3), (0, 0), (4, 200)], 32, 8, 1, 128),
    ([(5, 5), (1, 700), (17, 40), (32, 32)], 8, 8, 2, 80),
    ([(33, 90), (31, 31)], 64, 2, 2, 16),
    ([(130, 130), (1, 400), (63, 200)], 16, 6, 3, 96),
    ([(257, 300), (127, 127)], 128, 4, 2, 128),
    ([(100, 333)], 8, 14, 2, 112),
    ([(70, 150), (1, 150)], 16, 4, 4, 192),
    ([(40, 260), (129, 129), (1, 90)], 32, 4, 1, 256),
    ([(500, 1100)], 256, 8, 8, 64),
    ([(66, 70)], 16, 3, 3, 48),
    ([(1, 5000)], 16, 8, 1, 256),
    ([(20, 3000), (1, 3)], 16, 1, 1, 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(op, dev, shape, dtype):
    seqs, page, H, KV, d = SHAPES[shape]
    b = Batch(op, dev, seqs, page, KV, d, dtype, seed=shape, head_major=shape % 2 == 1, pad=shape % 3)
    q = (_randn(dev, 77, b.rows, H, d) * 2).to(dtype)
    out = torch.full_like(q, 7.0)
    y = op.paged_attention(q, b.kv, b.batch, out=out)
    assert y is out
    _check(y, _reference(b, q), b, dtype)
    assert bool((out[b.starts[-1] :] == 7).all())
    assert torch.equal(op.paged_attention(q, b.kv, b.batch)[: b.starts[-1]], y[: b.starts[-1]])


MASKS = [
    dict(window=1),
    dict(window=40),
    dict(window=64, softcap=20.0),
    dict(softcap=2.5),
    dict(alibi=True),
    dict(alibi=True, softcap=30.0, prefix=True),
    dict(prefix=True),
    dict(prefix=True, window=30),
    dict(docs=True),
    dict(docs=True, window=50, alibi=True),
    dict(empty=True),
    dict(scale=0.5),
    dict(scale=-0.1, alibi=True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("chunks", [False, True])
def test_masks(op, dev, mask, dtype, chunks):
    how = dict(MASKS[mask])
    seqs = [(130, 300), (65, 65), (0, 20), (1, 200), (7, 90)] if chunks else [(1, 300), (2, 65), (0, 9), (1, 1), (3, 777)]
    H, KV, d = (6, 2, 64) if mask % 2 else (4, 4, 128)
    b = Batch(op, dev, seqs, 16, KV, d, dtype, seed=mask)
    q = (_randn(dev, 5, b.rows, H, d) * 2).to(dtype)
    if how.pop("alibi", False):
        how["alibi_slopes"] = 0.3 ** (1 + torch.arange(H, device=dev)).float()
    if how.pop("prefix", False):
        how["prefix"] = _i32(dev, [200, 1000, 3, 0, 64])
    if how.pop("docs", False):
        first = [max(0, length - n + i - 37) // 20 * 20 for n, length in seqs for i in range(n)]
        how["first_key"] = _i32(dev, first)
    if how.pop("empty", False):  # some rows, whole tiles of them and a whole sequence see nothing
        first = [10**6 if i % 3 == 0 or 40 < i < 110 or n == 1 else -5 for n, _ in seqs for i in range(n)]
        how["first_key"] = _i32(dev, first)
    y = op.paged_attention(q, b.kv, b.batch, **how)
    _check(y, _reference(b, q, **how), b, dtype)
    if mask == 10:
        empty = how["first_key"] == 10**6
        assert bool((y[empty] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("seqs", [[(90, 250), (40, 40)], [(4, 250), (2, 40)], [(2, 250), (1, 40)]])
def test_not_finite_in_places_that_rows_do_not_see(op, dev, dtype, value, seqs):
    """A value or a key that is not finite reaches the rows that see it and no other."""
    H, KV, d = 4, 2, 128
    b = Batch(op, dev, seqs, 16, KV, d, dtype)
    n, length = seqs[0]
    for where, key in ((b.values, length - n // 2), (b.values, 100), (b.keys, min(length - n // 2 + 1, length - 1))):
        where[0][key, 1, 5] = value
    for where, pool in ((b.keys, b.k), (b.values, b.v)):
        j = torch.arange(length, device=dev)
        pool[b.table[0, j // 16].long(), j % 16] = where[0]
    first = _i32(dev, [101 if i % 2 else 0 for n, _ in seqs for i in range(n)])
    first[n:] = 0
    q = _randn(dev, 3, b.rows, H, d).to(dtype)
    y = op.paged_attention(q, b.kv, b.batch, first_key=first)
    ref = _reference(b, q, first_key=first)
    seen_by_none = torch.isfinite(ref[0])
    assert bool(torch.isfinite(y[: b.starts[-1]][seen_by_none[: b.starts[-1]]]).all())
    assert int(seen_by_none.sum()) > y.numel() // 4 and int((~seen_by_none).sum()) > 0
    # Rows that see the key have a NaN or what the exponentials make of it; the others are exact.
    clean = seen_by_none.all(-1, keepdim=True).expand_as(y)
    yy = torch.where(clean, y.double(), ref[0])
    _check(yy, ref, b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 60])
def test_not_finite_values_that_all_rows_see(op, dev, dtype, new):
    """An infinity among values makes that column infinite, of both signs or a NaN makes it a NaN."""
    b = Batch(op, dev, [(new, 300)], 16, 1, 64, dtype)
    v = b.values[0]
    v[7, 0, 1], v[7, 0, 2], v[90, 0, 2], v[30, 0, 3] = float("inf"), float("inf"), float("-inf"), float("nan")
    v[200, 0, 4] = float("-inf")
    j = torch.arange(300, device=dev)
    b.v[b.table[0, j // 16].long(), j % 16] = v
    q = _randn(dev, 3, new, 2, 64).to(dtype)
    y = op.paged_attention(q, b.kv, b.batch).float()
    assert bool((y[..., 1] == float("inf")).all()) and bool(y[..., 2].isnan().all()) and bool(y[..., 3].isnan().all())
    assert bool((y[..., 4] == float("-inf")).all())
    rest = [0] + list(range(5, 64))
    assert bool(torch.isfinite(y[..., rest]).all())
    out, A, ds, n = _reference(b, q)
    _check(torch.where(torch.isfinite(out), y.double(), out), (out, A, ds, n), b, dtype)


def test_a_tiny_cap(op, dev):
    b = Batch(op, dev, [(3, 40), (40, 40)], 16, 2, 64, torch.float32)
    q = _randn(dev, 3, b.rows, 4, 64)
    q[0] = 0
    y = op.paged_attention(q, b.kv, b.batch, softcap=1e-38)
    _check(y, _reference(b, q, softcap=1e-38), b, torch.float32)


@pytest.mark.parametrize("cap", [1024.0, 1e6, 1e30])
def test_a_wide_cap(op, dev, cap):
    """A cap that leaves the scores nearly as they are: each off by 2^-20 of itself at most in fp32 (of the cap, steps of
    2^-23 would be seen), which with (d + 8) >= 72 U of a score twice the uncapped bound covers."""
    dtype = torch.float32
    b = Batch(op, dev, [(3, 40), (70, 130), (1, 50)], 16, 2, 64, dtype)
    q = _randn(dev, 3, b.rows, 4, 64) * 8
    out, A, _, n = _reference(b, q, softcap=cap)
    ds = _reference(b, q)[2]
    _check(op.paged_attention(q, b.kv, b.batch, softcap=cap), (out, A, 2 * ds, n), b, dtype)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_the_widest_cap_in_16_bits(op, dev, dtype):
    b = Batch(op, dev, [(3, 40), (70, 130), (1, 50)], 16, 2, 64, dtype)
    q = (_randn(dev, 3, b.rows, 4, 64) * 8).to(dtype)
    _check(op.paged_attention(q, b.kv, b.batch, softcap=1024.0), _reference(b, q, softcap=1024.0), b, dtype)
    with pytest.raises(Exception, match="softcap past 1024"):
        op.paged_attention(q, b.kv, b.batch, softcap=1025.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_of_not_finite_queries(op, dev, dtype):
    b = Batch(op, dev, [(70, 200), (1, 100)], 16, 2, 64, dtype)
    q = _randn(dev, 3, b.rows, 4, 64).to(dtype)
    q[5, 1, 3] = float("nan")
    q[70, 2, 0] = float("nan")
    y = op.paged_attention(q, b.kv, b.batch)
    assert bool(y[5, 1].isnan().all()) and bool(y[70, 2].isnan().all())
    q2 = torch.where(q.isnan(), 0, q)
    ref = _reference(b, q2)
    y[5, 1], y[70, 2] = ref[0][5, 1].to(dtype), ref[0][70, 2].to(dtype)
    _check(y, ref, b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_apart(op, dev, dtype):
    """Maxima that grow, fall and jump from key to key: one key takes it all, weights vanish."""
    seqs = [(64, 400), (1, 400)]
    b = Batch(op, dev, seqs, 16, 2, 64, dtype)
    q = (_randn(dev, 3, b.rows, 2, 64) * 30).to(dtype)
    _check(op.paged_attention(q, b.kv, b.batch), _reference(b, q), b, dtype)
    _check(op.paged_attention(q, b.kv, b.batch, scale=2.0), _reference(b, q, scale=2.0), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_many_small_weights_beside_a_large_one(op, dev, dtype, new):
    """4095 weights of e^-14.5, between the steps that fp16 has near 2^-21, are all that the result is of."""
    n = 4096
    k, v = torch.zeros(n, 1, 64, dtype=dtype, device=dev), torch.ones(n, 1, 64, dtype=dtype, device=dev)
    k[0, 0, 0], v[0] = 1.8125, 0
    b = Batch(op, dev, [(new, n)], 16, 1, 64, dtype, kv=([k], [v]))
    q = torch.zeros(new, 2, 64, dtype=dtype, device=dev)
    q[:, :, 0] = 8
    _check(op.paged_attention(q, b.kv, b.batch, scale=1.0), _reference(b, q, scale=1.0), b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_bounds_of_the_device_arrays(op, dev, dtype, new):
    """Sequences that break a bound are NaN, the others as if alone."""
    seqs = [(new, 100), (new, 90), (new, 80)]
    b = Batch(op, dev, seqs, 16, 2, 64, dtype)
    q = _randn(dev, 3, b.rows, 4, 64).to(dtype)
    want = op.paged_attention(q, b.kv, b.batch)

    def run(table=b.table, lens=(100, 90, 80), starts=b.starts, max_len=100, max_new=new):
        batch = op.SequenceBatch(table, _i32(dev, lens), _i32(dev, starts), max_len, max_new)
        return op.paged_attention(q, b.kv, batch, out=torch.zeros_like(q))

    mid = slice(new, 2 * new)
    for page in (-1, b.k.shape[0], 2**31 - 1, -(2**31)):
        t = b.table.clone()
        t[1, 2] = page
        y = run(table=t)
        assert bool(y[mid].isnan().all())
        y[mid] = want[mid]
        assert torch.equal(y, want)
    for length in (new - 1, -3, 101, 2**31 - 1):
        y = run(lens=(100, length, 80))
        assert bool(y[mid].isnan().all())
        y[mid] = want[mid]
        assert torch.equal(y, want)
    y = run(max_len=95)
    assert bool(y[:new].isnan().all()) and torch.equal(y[new:], want[new:])
    y = run(lens=(100, 16 * b.table.shape[1] + 1, 80), max_len=10**6)  # more keys than a table's pages
    assert bool(y[mid].isnan().all())
    y = run(max_new=new - 1) if new > 1 else run(starts=[0, 0, 2, 3])
    assert bool(y.isnan().any())
    y = run(starts=[0, new, 2 * new, 10**6])  # past the rows: what there is of it is NaN
    assert bool(y[2 * new :].isnan().all()) and torch.equal(y[: 2 * new], want[: 2 * new])
    run(starts=[5, 2, -1, 1])  # anything may come of it, within the arrays
    torch.cuda.synchronize()


# ---- norm, rotation, append -------------------------------------------------


def _turned(x, norm, eps, freqs, pos, interleaved):
    """The head's values in 64 bits and the magnitude that their errors go with."""
    x = x.double()
    if norm is not None:
        x = x * norm.double() / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    half = 0 if freqs is None else freqs.numel()
    if half == 0:
        return x, x.abs()
    angle = (pos.double()[:, None] * freqs)[:, None]
    c, s = angle.cos(), angle.sin()
    a, b = (x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]) if interleaved else (x[..., :half], x[..., half : 2 * half])
    y, m = x.clone(), x.abs().clone()
    ya, yb, mag = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if interleaved:
        y[..., 0 : 2 * half : 2], y[..., 1 : 2 * half : 2] = ya, yb
        m[..., 0 : 2 * half : 2] = m[..., 1 : 2 * half : 2] = mag
    else:
        y[..., :half], y[..., half : 2 * half] = ya, yb
        m[..., :half] = m[..., half : 2 * half] = mag
    return y, m


def _close(y, ref, mag, d, dtype):
    # d / 8 + 16 roundings for the sum of squares, the root, the quotient, the products; 8 for the sine
    tol = (HALF[dtype] + U) * ref.abs() + (d / 8 + 24) * U * mag + TINY[dtype]
    assert bool(((y.double() - ref).abs() <= tol).all()), float(((y.double() - ref).abs() / tol).max())


ROPES = [  # heads, kv_heads, head_dim, rotary_dim
    (1, 1, 64, 64), (4, 2, 128, 128), (12, 3, 80, 48), (5, 5, 80, 20), (8, 1, 256, 64), (2, 2, 16, 16), (64, 8, 128, 128),
    (3, 1, 96, 24), (6, 2, 112, 112), (4, 4, 192, 0), (7, 1, 48, 2), (16, 16, 128, 126),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", range(len(ROPES)))
def test_norm_rope_append(op, dev, shape, interleaved, dtype):
    H, KV, d, rot = ROPES[shape]
    seqs = [(1, 1), (7, 40), (0, 12), (1, 17), (64, 64), (3, 100003)] if shape == 1 else [(1, 1), (7, 40), (0, 12), (33, 49)]
    hole = 3.0
    page = 8 << shape % 6
    b = Batch(op, dev, seqs, page, KV, d, dtype, hole=hole, head_major=shape % 2 == 0, pad=2)
    before = b.k.clone(), b.v.clone()
    qkv = _randn(dev, shape, b.rows, H + 2 * KV, d).to(dtype)
    q, k, v = qkv[:, :H], qkv[:, H : H + KV], qkv[:, H + KV :]
    freqs = op.rotary_frequencies(rot, device=dev) if rot else None
    norms = [None, None] if shape % 3 == 2 else [1 + 0.2 * _randn(dev, 1, d), 1 + 0.2 * _randn(dev, 2, d)]
    positions = _randn(dev, 4, b.rows).mul(1e5).int() if shape % 4 == 3 else None
    T = b.starts[-1]
    pos = torch.cat([torch.arange(n - m, n, device=dev) for m, n in seqs])
    out = torch.full((b.rows, H, d), 9.0, dtype=dtype, device=dev)
    how = dict(freqs=freqs, q_norm=norms[0], k_norm=norms[1], eps=1e-5, interleaved=interleaved, positions=positions)
    assert op.norm_rope_append(q, k, v, b.kv, b.batch, out=out, **how) is out
    assert bool((out[T:] == 9).all())
    at = pos if positions is None else positions[:T]
    _close(out[:T], *_turned(q[:T], norms[0], 1e-5, freqs, at, interleaved), d, dtype)
    # The new rows of the cache, and nothing else of it.
    seq = torch.cat([torch.full((m,), i, device=dev) for i, (m, _) in enumerate(seqs)])
    where = b.table[seq, pos // page].long(), pos % page
    _close(b.k[where], *_turned(k[:T], norms[1], 1e-5, freqs, at, interleaved), d, dtype)
    assert torch.equal(b.v[where], v[:T])
    for pool, old in ((b.k, before[0]), (b.v, before[1])):
        pool = pool.clone()
        pool[where] = old[where]
        assert torch.equal(pool, old)
    # In place.
    q2 = q
    y = op.norm_rope_append(q2, k, v, b.kv, b.batch, out=q2, **how)
    assert torch.equal(y[:T], out[:T])


@pytest.mark.parametrize("count", [64, 65, 130, 4200])
def test_append_of_many_sequences(op, dev, count):
    """A token finds its sequence among many, some without tokens."""
    dtype = torch.float32
    new = [(7 * i) % 3 for i in range(count)]
    table = torch.arange(count, dtype=torch.int32, device=dev)[:, None]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + 3
    kv = op.PagedKV(*(torch.full((count, 8, 1, 16), 5, dtype=dtype, device=dev) for _ in range(2)))
    batch = op.SequenceBatch(table, _i32(dev, [6] * count), _i32(dev, starts), 8, 2)
    q, k, v = _randn(dev, 1, rows, 2, 16), _randn(dev, 2, rows, 1, 16), _randn(dev, 3, rows, 1, 16)
    out = torch.full_like(q, 7)
    op.norm_rope_append(q, k, v, kv, batch, out=out)
    assert torch.equal(out[: rows - 3], q[: rows - 3]) and bool((out[rows - 3 :] == 7).all())
    want = torch.full_like(kv.k, 5), torch.full_like(kv.v, 5)
    seq = torch.repeat_interleave(torch.arange(count), torch.tensor(new)).to(dev)
    at = torch.cat([torch.arange(6 - n, 6) for n in new]).to(dev)
    want[0][seq, at], want[1][seq, at] = k[: rows - 3], v[: rows - 3]
    assert torch.equal(kv.k, want[0]) and torch.equal(kv.v, want[1])


def test_one_norm_of_two(op, dev):
    b = Batch(op, dev, [(5, 9)], 8, 2, 64, torch.float32)
    q, k, v = (_randn(dev, i, 5, 2, 64) for i in range(3))
    g = 1 + 0.1 * _randn(dev, 9, 64)
    y = op.norm_rope_append(q, k, v, b.kv, b.batch, k_norm=g)
    assert torch.equal(y, q)
    pos = torch.arange(4, 9, device=dev)
    where = b.table[0, pos // 8].long(), pos % 8
    _close(b.k[where], *_turned(k, g, 1e-5, None, pos, False), 64, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_bounds(op, dev, dtype):
    """No row is written for a sequence that breaks a bound, or outside the pool."""
    seqs = [(3, 20), (3, 30), (3, 40)]
    b = Batch(op, dev, seqs, 8, 2, 64, dtype, hole=1.0)
    qkv = _randn(dev, 1, b.rows, 4 + 4, 64).to(dtype)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]

    def run(table=b.table, lens=(20, 30, 40), starts=b.starts, max_len=40, max_new=3):
        b.k.fill_(1), b.v.fill_(1)
        y = op.norm_rope_append(q, k, v, b.kv, op.SequenceBatch(table, _i32(dev, lens), _i32(dev, starts), max_len, max_new))
        return y, (b.k != 1).any(-1).any(-1).sum().item()

    want, rows = run()
    assert rows == 9 and torch.equal(want, q)
    for page in (-1, b.k.shape[0], 2**31 - 1):
        t = b.table.clone()
        t[1, 3] = page  # keys 24 .. 31: all three
        y, rows = run(table=t)
        assert rows == 6 and bool(y[3:6].isnan().all()) and torch.equal(y[:3], want[:3]) and torch.equal(y[6:], want[6:])
    for length in (2, -1, 41, 2**31 - 1):
        y, rows = run(lens=(20, length, 40))
        assert rows == 6 and bool(y[3:6].isnan().all())
    y, rows = run(max_new=2)
    assert rows == 0 and bool(y.isnan().all())
    run(starts=[5, 2, -1, 1])
    run(starts=[0, 3, 6, 10**6])
    torch.cuda.synchronize()


# ---- together ---------------------------------------------------------------


def _layers(op, dev, dtype, D=256, H=8, KV=2, d=64, hidden=512, n=2):
    import soverign_grad_amd.w8a8 as w8a8

    out = []
    for i in range(n):
        w = [_randn(dev, 100 * i + j, *s) * s[0] ** -0.5 for j, s in
             enumerate([(D, H * d), (D, KV * d), (D, KV * d), (H * d, D), (D, hidden), (D, hidden), (hidden, D)])]
        norm = 1 + 0.1 * _randn(dev, 50 + i, D)
        attn = op.QuantizedAttentionInt8.from_float(*w[:4], norm, H, KV, freqs=op.rotary_frequencies(d, device=dev),
                                                    q_norm=1 + 0.1 * _randn(dev, 60 + i, d),
                                                    k_norm=1 + 0.1 * _randn(dev, 70 + i, d))
        out.append((attn, w8a8.QuantizedMLPInt8.from_float(*w[4:], norm)))
    return out


def _forward(layers, x, kvs, batch):
    h = None
    for (attn, mlp), kv in zip(layers, kvs):
        x, h = attn.forward(x, kv, batch, residual=h)
        x, h = mlp.forward(x, residual=h)
    return x + h


@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_in_chunks_and_tokens_give_what_whole_prompts_give(op, dev, dtype):
    """Two layers: prompts at once, in chunks beside another sequence's tokens, and token by token."""
    layers, page = _layers(op, dev, dtype), 16
    lens = [70, 45]
    x = [_randn(dev, i, n, 256).to(dtype) for i, n in enumerate(lens)]
    table = _i32(dev, [[3, 1, 4, 7, 9, 8], [2, 6, 5, 0, 11, 10]])

    def pools():
        return [op.PagedKV.empty(12, page, 2, 64, dtype, dev) for _ in layers]

    def step(kvs, spans):
        """spans: (first, end) of each sequence's tokens."""
        starts = [0, spans[0][1] - spans[0][0]]
        starts.append(starts[1] + spans[1][1] - spans[1][0])
        batch = op.SequenceBatch(table, _i32(dev, [e for _, e in spans]), _i32(dev, starts), max(e for _, e in spans),
                                 max(e - f for f, e in spans))
        y = _forward(layers, torch.cat([t[f:e] for t, (f, e) in zip(x, spans)]), kvs, batch)
        return y[: starts[1]], y[starts[1] :]

    whole = step(pools(), [(0, 70), (0, 45)])
    kvs = pools()
    for spans in ([(0, 40), (0, 44)], [(40, 69), (44, 45)], [(69, 70), (45, 45)]):
        parts = step(kvs, spans)
        for got, want, (f, e) in zip(parts, whole, spans):
            # The forms differ by roundings, which 8-bit codes may carry by a step of 1 / 127 of a row's
            # largest value, now and then.
            top = want.float().abs().max()
            assert got.shape[0] == e - f
            if e > f:
                diff = (got.float() - want[f:e].float()).abs()
                assert float(diff.max()) <= 0.06 * float(top) and float(diff.mean()) <= 0.01 * float(top)


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_steps(op, dev, dtype):
    """A decode step of two layers in a graph, replayed with other lengths and inputs."""
    layers, page, B = _layers(op, dev, dtype), 16, 3
    kvs = [op.PagedKV(*(_randn(dev, i, 30, page, 2, 64).to(dtype) for i in (1, 2))) for _ in layers]
    table = torch.arange(30, dtype=torch.int32, device=dev).reshape(3, 10)
    lens, starts = _i32(dev, [1, 1, 1]), torch.arange(B + 1, dtype=torch.int32, device=dev)
    x = torch.zeros(B, 256, dtype=dtype, device=dev)
    batch = op.SequenceBatch(table, lens, starts, 160, 1)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        _forward(layers, x, kvs, batch)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _forward(layers, x, kvs, batch)
    for i, now in enumerate([[1, 5, 160], [17, 33, 2], [160, 64, 65], [100, 1, 7]]):
        x.copy_(_randn(dev, 40 + i, B, 256))
        lens.copy_(_i32(dev, now))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, _forward(layers, x, kvs, batch))


def test_two_graphs_replayed_side_by_side(op, dev):
    """Each graph has a workspace of its own."""
    b = Batch(op, dev, [(1, 4000)], 16, 2, 128, torch.bfloat16)
    qs = [_randn(dev, i, 1, 8, 128).to(torch.bfloat16) for i in range(2)]
    want = [op.paged_attention(q, b.kv, b.batch) for q in qs]
    streams, graphs, outs = [torch.cuda.Stream(dev) for _ in qs], [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(op.paged_attention(q, b.kv, b.batch))
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_on_a_stream_of_its_own(op, dev):
    b = Batch(op, dev, [(1, 900), (50, 400)], 16, 2, 128, torch.bfloat16)
    q = _randn(dev, 1, b.rows, 8, 128).to(torch.bfloat16)
    want = op.paged_attention(q, b.kv, b.batch)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        y = op.paged_attention(q, b.kv, b.batch)
    s.synchronize()
    assert torch.equal(y, want)


def test_a_cache_past_32_bits(op, dev):
    """Pages whose offsets pass 2^32 bytes and 2^31 elements; a table that walks them."""
    dtype, page, KV, d = torch.bfloat16, 64, 8, 128
    pages = (2**31 // (page * KV * d)) + 300
    k = torch.empty(pages, page, KV, d, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    table = _i32(dev, [[pages - 1, 0, pages - 2, 5, pages - 300, pages // 2, 1, pages - 3]])
    small_k, small_v = _randn(dev, 1, 8, page, KV, d).to(dtype), _randn(dev, 2, 8, page, KV, d).to(dtype)
    k[table[0].long()], v[table[0].long()] = small_k, small_v
    for n in (1, 150):
        q = _randn(dev, 3, n, 16, d).to(dtype)
        nk, nv = _randn(dev, 4, n, KV, d).to(dtype), _randn(dev, 5, n, KV, d).to(dtype)
        args = _i32(dev, [500]), _i32(dev, [0, n]), 500, n
        far, near = op.PagedKV(k, v), op.PagedKV(small_k, small_v)
        here = torch.arange(8, dtype=torch.int32, device=dev)[None]
        f = op.rotary_frequencies(d, device=dev)
        got = [op.norm_rope_append(q, nk, nv, far, op.SequenceBatch(table, *args), freqs=f),
               op.paged_attention(q, far, op.SequenceBatch(table, *args))]
        want = [op.norm_rope_append(q, nk, nv, near, op.SequenceBatch(here, *args), freqs=f),
                op.paged_attention(q, near, op.SequenceBatch(here, *args))]
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(k[table[0].long()], small_k) and torch.equal(v[table[0].long()], small_v)


def test_few_tokens_in_a_batch_padded_to_many(op, dev):
    """One token of one long sequence among 2^21 rows of 8 heads: its row is right, the others stay."""
    dtype, rows = torch.float16, 2**21
    b = Batch(op, dev, [(1, 3000)], 16, 8, 16, dtype, pad=rows - 1)
    q = torch.zeros(rows, 8, 16, dtype=dtype, device=dev)
    q[0] = _randn(dev, 3, 8, 16)
    out = torch.full_like(q, 7)
    op.paged_attention(q, b.kv, b.batch, out=out)
    assert bool((out[1:] == 7).all())
    _check(out[:1], _reference(b, q[:1]), b, dtype)


def test_limits_past_32_bits(op, dev):
    """A prefix or a first key in 64 bits that 32 do not hold is past (or before) every key."""
    b = Batch(op, dev, [(4, 50), (1, 30)], 16, 2, 64, torch.float16)
    q = _randn(dev, 1, 5, 4, 64).half()
    for far, near in ((2**63 - 1, 50), (2**32 + 3, 50), (2**31, 50), (-(2**32) + 7, 0), (-(2**63), 0)):
        got = op.paged_attention(q, b.kv, b.batch, prefix=torch.tensor([far, far], device=dev))
        assert torch.equal(got, op.paged_attention(q, b.kv, b.batch, prefix=_i32(dev, [near, near])))
        got = op.paged_attention(q, b.kv, b.batch, first_key=torch.full((5,), far, device=dev))
        assert torch.equal(got, op.paged_attention(q, b.kv, b.batch, first_key=_i32(dev, [near] * 5)))
    assert bool((op.paged_attention(q, b.kv, b.batch, first_key=torch.full((5,), 2**40, device=dev)) == 0).all())


def test_heads_that_are_not_aligned_are_copied(op, dev):
    b = Batch(op, dev, [(4, 50)], 16, 2, 64, torch.float16)
    flat = _randn(dev, 1, 4 * 4 * 64 + 1).half()
    q = flat[1:].view(4, 4, 64)
    want = op.paged_attention(q.clone(), b.kv, b.batch)
    assert torch.equal(op.paged_attention(q, b.kv, b.batch), want)
    wide = _randn(dev, 2, 4, 4, 65).half()
    wide[..., :64] = q
    assert torch.equal(op.paged_attention(wide[..., :64], b.kv, b.batch), want)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(op.paged_attention(major, b.kv, b.batch), want)
    one = q[:1, :2].expand(4, 2, 64)
    assert torch.equal(op.paged_attention(one, b.kv, b.batch), op.paged_attention(one.clone(), b.kv, b.batch))


def test_refusals_on_the_device(op, dev):
    b = Batch(op, dev, [(4, 50)], 16, 2, 64, torch.float16)
    q = _randn(dev, 1, 4, 4, 64).half()
    kv, batch, run = b.kv, b.batch, op.paged_attention
    bad = [lambda: run(q.float(), kv, batch), lambda: run(q[:, :3], kv, batch), lambda: run(q[..., :48], kv, batch),
           lambda: run(q.cpu(), kv, batch), lambda: run(q, kv, batch, window=-1),
           lambda: run(q, kv, batch, out=torch.empty(4, 4, 65, device=dev).half()[..., :64]),
           lambda: run(q, kv, batch, out=torch.empty(5, 4, 64, device=dev).half()),
           lambda: run(q, kv, batch, alibi_slopes=torch.ones(3, device=dev)),
           lambda: run(q, kv, batch, prefix=torch.ones(2, device=dev).int()),
           lambda: run(q, kv, batch, first_key=torch.ones(4, device=dev)),
           lambda: op.PagedKV(b.k, b.v[:-1]), lambda: op.PagedKV(b.k, b.k), lambda: op.PagedKV(b.k[..., :40], b.v[..., :40]),
           lambda: op.PagedKV(b.k[:, :12], b.v[:, :12]), lambda: op.PagedKV(b.k.double(), b.v.double()),
           lambda: op.PagedKV(b.k[:, :, :1].expand(-1, -1, 2, -1), b.v[:, :, :1].expand(-1, -1, 2, -1)),
           lambda: op.SequenceBatch(b.table.long(), batch.lens, batch.starts, 50, 4),
           lambda: op.SequenceBatch(b.table, batch.lens, batch.lens, 50, 4),
           lambda: op.SequenceBatch(b.table, batch.lens, batch.starts, -1, 4),
           lambda: op.norm_rope_append(q, q, q, kv, batch),
           lambda: op.norm_rope_append(q, q[:, :2], q[:3, :2], kv, batch),
           lambda: op.norm_rope_append(q, q[:, :2], q[:, 2:], kv, batch, freqs=torch.ones(33, device=dev)),
           lambda: op.norm_rope_append(q, q[:, :2], q[:, 2:], kv, batch, q_norm=torch.ones(63, device=dev)),
           lambda: op.norm_rope_append(q, q[:, :2], q[:, 2:], kv, batch, positions=torch.ones(3, device=dev).int())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    import soverign_grad_amd as sgq

    x = _randn(dev, 2, 4, 12, 64).half()
    for call in (lambda: run(q, kv, batch, softcap=-1.0), lambda: run(q, kv, batch, softcap=float("nan")),
                 lambda: run(x[:, :4], kv, batch, out=x[:, 2:6]),
                 lambda: op.norm_rope_append(x[:, :4], x[:, 4:6], x[:, 6:8], kv, batch, out=x[:, 3:7])):
        with pytest.raises(sgq.SGQError):
            call()


def test_nothing_to_do(op, dev):
    b = Batch(op, dev, [(0, 5), (0, 0)], 16, 2, 64, torch.float16)
    q = torch.empty(0, 4, 64, dtype=torch.float16, device=dev)
    assert op.paged_attention(q, b.kv, b.batch).shape == (0, 4, 64)
    assert op.norm_rope_append(q, q[:, :2], q[:, :2], b.kv, b.batch).shape == (0, 4, 64)
    none = op.SequenceBatch(b.table[:0], b.batch.lens[:0], b.batch.starts[:1], 0, 0)
    x = torch.full((3, 4, 64), 2.0, dtype=torch.float16, device=dev)
    assert bool((op.paged_attention(x, b.kv, none, out=x) == 2).all())
