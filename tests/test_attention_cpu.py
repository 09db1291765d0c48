"""What the attention entry points refuse, found before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
P = 1 << 20  # an address that nothing reads


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.fixture(scope="module")
def lib(sgq):
    return sgq.load_library()


def _cache(op, **kw):
    a = dict(k=P, v=2 * P, pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, token_stride=128,
             head_stride=64, dtype=1)
    return op._PagedCache(**{**a, **kw})


def _seqs(op, **kw):
    a = dict(table=P, table_ld=4, table_pages=4, lens=P, starts=P, B=3, max_len=64, max_new=2)
    return op._Sequences(**{**a, **kw})


def _scores(op, **kw):
    return op._Scores(**{**dict(scale=0.125, softcap=0.0, window=0, alibi_slopes=None, prefix=None, first_key=None), **kw})


def _attend(op, lib, cache={}, seqs={}, scores={}, q=4 * P, q_row=256, q_head=64, out=8 * P, o_row=256, o_head=64, rows=5,
            heads=4, ws=None, nws=0):
    c, s, h = _cache(op, **cache), _seqs(op, **seqs), _scores(op, **scores)
    return lib.sgq_paged_attention(q, q_row, q_head, out, o_row, o_head, rows, heads, ctypes.addressof(c),
                                   ctypes.addressof(s), ctypes.addressof(h), ws, nws, None)


def _append(op, lib, cache={}, seqs={}, q=4 * P, q_row=512, q_head=64, k=4 * P + 512, v=4 * P + 768, out=8 * P, o_row=256,
            rows=5, heads=4, freqs=P, rot=64):
    c, s = _cache(op, **cache), _seqs(op, **seqs)
    return lib.sgq_norm_rope_append(q, q_row, q_head, k, q_row, q_head, v, q_row, q_head, out, o_row, 64, rows, heads,
                                    ctypes.addressof(c), ctypes.addressof(s), None, None, 1e-5, freqs, rot, 0, None, None)


SHARED = [
    (INVALID, dict(cache=dict(dtype=3))), (UNSUPPORTED, dict(cache=dict(head_dim=40))), (UNSUPPORTED, dict(cache=dict(head_dim=272))),
    (UNSUPPORTED, dict(cache=dict(head_dim=0))), (UNSUPPORTED, dict(cache=dict(page_size=12))),
    (UNSUPPORTED, dict(cache=dict(page_size=1 << 17))), (UNSUPPORTED, dict(cache=dict(page_size=0))), (UNSUPPORTED, dict(cache=dict(page_size=4))),
    (INVALID, dict(cache=dict(kv_heads=0))), (INVALID, dict(cache=dict(kv_heads=3, head_stride=64))), (INVALID, dict(cache=dict(pages=-1))),
    (INVALID, dict(cache=dict(token_stride=60))), (INVALID, dict(cache=dict(token_stride=56))),
    (INVALID, dict(cache=dict(head_stride=-64))), (INVALID, dict(cache=dict(page_stride=0))),
    (UNSUPPORTED, dict(cache=dict(page_stride=1 << 31))), (UNSUPPORTED, dict(cache=dict(token_stride=1 << 31))), (UNSUPPORTED, dict(cache=dict(head_stride=1 << 41))), (INVALID, dict(cache=dict(k=P + 8))), (INVALID, dict(cache=dict(v=None))),
    (INVALID, dict(seqs=dict(B=-1))), (INVALID, dict(seqs=dict(max_len=-1))), (INVALID, dict(seqs=dict(max_new=-1))),
    (INVALID, dict(seqs=dict(table_ld=3))), (INVALID, dict(seqs=dict(table=None))), (INVALID, dict(seqs=dict(lens=None))),
    (INVALID, dict(seqs=dict(starts=None))), (UNSUPPORTED, dict(seqs=dict(B=(1 << 20) + 1))),
    (UNSUPPORTED, dict(rows=(1 << 23) + 1)), (INVALID, dict(rows=-1)), (INVALID, dict(heads=3)), (INVALID, dict(heads=0)),
    (UNSUPPORTED, dict(heads=1026)), (UNSUPPORTED, dict(heads=512, rows=1 << 22)), (INVALID, dict(q=None)), (INVALID, dict(q=4 * P + 2)), (INVALID, dict(out=None)),
    (INVALID, dict(out=8 * P + 4)), (INVALID, dict(o_row=252)), (INVALID, dict(o_row=192)), (INVALID, dict(q_row=-512)),
    (INVALID, dict(q_head=32)), (INVALID, dict(q_row=1 << 31)),
]


@pytest.mark.parametrize("case", range(len(SHARED)))
def test_refused_by_both(op, lib, case):
    status, kw = SHARED[case]
    assert _attend(op, lib, **kw) == status, lib.sgq_last_error()
    assert _append(op, lib, **kw) == status, lib.sgq_last_error()


def test_refused_by_attention(op, lib):
    for kw in (dict(scores=dict(window=-1)), dict(scores=dict(softcap=-1.0)), dict(scores=dict(softcap=float("inf"))),
               dict(scores=dict(softcap=3e38)), dict(scores=dict(scale=3e38)), dict(scores=dict(scale=-3e38)),
               dict(scores=dict(softcap=float("nan"))), dict(out=4 * P + 128), dict(out=4 * P, o_row=320), dict(out=4 * P + 256)):
        assert _attend(op, lib, **kw) == INVALID, kw
    assert _attend(op, lib, scores=dict(softcap=1025.0)) == UNSUPPORTED
    c, s = _cache(op), _seqs(op)
    assert lib.sgq_paged_attention(P, 256, 64, 2 * P, 256, 64, 5, 4, ctypes.addressof(c), ctypes.addressof(s), None, None, 0,
                                   None) == INVALID
    assert lib.sgq_paged_attention(P, 256, 64, 2 * P, 256, 64, 5, 4, None, ctypes.addressof(s), None, None, 0, None) == INVALID


def test_refused_by_append(op, lib):
    for kw in (dict(rot=63), dict(rot=-2), dict(rot=66), dict(freqs=None), dict(k=None), dict(v=None), dict(k=4 * P + 520),
               dict(out=4 * P + 256, o_row=512), dict(out=4 * P + 512, o_row=512), dict(out=4 * P, o_row=256),
               dict(out=4 * P + 768, o_row=512), dict(cache=dict(k=2 * P))):
        assert _append(op, lib, **kw) == INVALID, kw


def test_nothing_to_do(op, lib):
    """Without rows or sequences no pointer is looked at."""
    none = dict(table=None, lens=None, starts=None)
    for kw in (dict(rows=0, seqs=none), dict(seqs=dict(B=0, **none))):
        assert _attend(op, lib, q=None, out=None, **kw) == OK
        assert _append(op, lib, q=None, out=None, k=None, v=None, freqs=None, **kw) == OK


def test_python_refuses_what_is_not_on_the_device(op):
    k, v = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError):
        op.PagedKV(k, v)
    t = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        op.SequenceBatch(t, t[:, 0], torch.zeros(3, dtype=torch.int32), 16, 1)
    for dim in (0, 3, -2):
        with pytest.raises(ValueError):
            op.rotary_frequencies(dim, device="cpu")
    f = op.rotary_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)


def test_limits_in_64_bits_do_not_wrap(op):
    t = torch.tensor([2**40, -(2**40), 2**31, 5])
    got = op._int32(t, 4, t.device, "prefix")
    assert got.dtype is torch.int32 and got.tolist() == [2**31 - 1, -(2**31), 2**31 - 1, 5]


def test_workspace(op, lib):
    """What a call needs it says beforehand, for a device of any size, and refuses to run without."""
    fn = lib.sgq_paged_attention_workspace_bytes
    seen = 0
    for cus in (1, 32, 256, 304):
        for heads, kv in ((1, 1), (32, 8), (16, 16), (28, 4)):
            for d in (16, 64, 80, 128, 192, 256):
                for dtype in (0, 1, 2):
                    for B, rows, length, new in ((1, 1, 1, 1), (1, 1, 131072, 1), (64, 64, 8192, 1), (1, 2048, 2048, 2048), (5, 100, 900, 33)):
                        for window in (0, 100):
                            need = fn(heads, kv, d, dtype, B, rows, length, new, window, cus)
                            per = rows * heads * (4 * d + 8)
                            assert need == 0 or need % per == 0 and 2 <= need // per <= 256
                            seen += need > 0
    assert seen > 100
    # Rows behind the last sequence: a gibibyte at most, however many.
    for heads, d, new in ((1, 16, 1), (32, 128, 1), (8, 256, 4), (32, 128, 100), (1024, 16, 1)):
        for rows in (1, 1000, 30000, 2**30 // 1024):
            assert fn(heads, 1, d, 1, 1, rows, 131072, new, 0, 0) <= 2**30
    for bad in ((0, 1, 64, 0, 1, 1, 1, 1, 0, 0), (3, 2, 64, 0, 1, 1, 1, 1, 0, 0), (2, 2, 60, 0, 1, 1, 1, 1, 0, 0), (2, 2, 64, 3, 1, 1, 1, 1, 0, 0),
                (2, 2, 64, 0, -1, 1, 1, 1, 0, 0), (2, 2, 64, 0, 1, -1, 1, 1, 0, 0), (2, 2, 64, 0, 1, 1, -1, 1, 0, 0),
                (2, 2, 64, 0, 1, 1, 1, -1, 0, 0), (2, 2, 64, 0, 1, 1, 1, 1, -1, 0), (2, 2, 64, 0, 1, 1, 1, 1, 0, -1)):
        assert fn(*bad) == -1, bad
    assert fn(2, 2, 64, 0, 0, 5, 1, 1, 0, 0) == 0 and fn(2, 2, 64, 0, 5, 0, 1, 1, 0, 0) == 0
    # One sequence of many keys is shared out: no workspace, too small a one, one at an odd address.
    long = dict(seqs=dict(B=1, max_len=60000, table_ld=4096, table_pages=4096, max_new=1), rows=1)
    need = fn(4, 2, 64, 1, 1, 1, 60000, 1, 0, 0)
    assert need > 0
    for ws, nws in ((None, need), (P, need - 1), (P + 8, need)):
        assert _attend(op, lib, ws=ws, nws=nws, **long) == WORKSPACE
    for scale in (float("inf"), float("nan")):
        assert _attend(op, lib, scores=dict(scale=scale)) == INVALID
