"""Rows of codes without columns still take sgq_tokens_row_bytes(0) bytes, which the quantizers fill with zeros: closer
rows are refused.  No call here launches a kernel."""
import helpers  # noqa: F401

P = 4096  # an aligned address that no call here reaches


def test_rows_without_columns_need_their_bytes(sgq):
    lib = sgq.load_library()
    assert lib.sgq_tokens_row_bytes(0) == 128
    for fn in (lib.sgq_quantize_tokens, lib.sgq_quantize_tokens_keep_nan):
        for ldc in (0, 16, 64, 112, 120):
            assert fn(None, 0, 0, 3, 0, P, ldc, P, None) == 1, ldc
            assert b"128" in lib.sgq_last_error()
        assert fn(None, 0, 0, 3, 0, None, 128, P, None) == 1 and fn(None, 0, 0, 0, 0, None, 0, None, None) == 0
    # What neither reads nor writes codes looks at none of it.
    assert lib.sgq_dequantize_tokens(None, 0, None, 3, 0, None, 0, 0, None) == 0
    assert lib.sgq_rms_norm_tokens(None, 0, 0, None, 0, None, 0, None, 1e-5, 3, 0, None, 0, None, None) == 0
