"""Refusals at the limits of 8-bit tokens, and the launch plans that the host alone answers.  No call here launches a
kernel: the addresses are never read."""
import pytest

import helpers  # noqa: F401

P = 4096  # an aligned address that no call here reaches
FAR = 2**21  # bytes between two rows of codes, at most


@pytest.fixture(scope="module")
def lib(sgq):
    return sgq.load_library()


def test_rows_of_codes_farther_apart_than_offsets_reach(lib):
    """The products take a row of codes through a 32-bit offset from its block's first: strides past 2^21 are refused."""
    q = dict(x=P, dtype=0, ldx=64, M=2, K=64, codes=P, ldc=FAR + 16, scales=P)
    n = dict(x=P, dtype=1, ldx=64, r=None, ldr=0, h=None, ldh=0, g=P, eps=1e-5, M=2, K=64, codes=P, ldc=FAR + 16, scales=P)
    d = dict(codes=P, ldc=FAR + 16, scales=P, M=2, K=64, out=P, dtype=0, ldo=64)
    y = dict(codes=P, ldc=FAR + 16, sx=P, M=2, K=64, N=32, packed=P, sw=P, bias=None, y=P, dtype=0, ldy=32, ws=P, nws=1 << 40)
    g = dict(codes=P, ldc=FAR + 16, sx=P, M=2, K=64, N=32, pg=P, sg=P, bg=None, pu=P, su=P, bu=None, h=P, dtype=0, ldh=32,
             ws=P, nws=1 << 40)
    calls = [(lib.sgq_quantize_tokens, q), (lib.sgq_quantize_tokens_keep_nan, q), (lib.sgq_rms_norm_tokens, n), (lib.sgq_dequantize_tokens, d), (lib.sgq_linear_w8a8, y),
             (lib.sgq_swiglu_w8a8, g)]
    for fn, kw in calls:
        for far in (FAR + 16, FAR * 2, 2**31, 2**40):
            assert fn(*{**kw, "ldc": far}.values(), None) == 2, (fn, far)
            assert str(FAR).encode() in lib.sgq_last_error()
        for bad in (FAR + 8, FAR - 8, 0, -128):
            assert fn(*{**kw, "ldc": bad}.values(), None) == 1, (fn, bad)
