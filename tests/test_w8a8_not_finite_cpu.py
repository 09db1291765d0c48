"""sgq_quantize_tokens_keep_nan refuses what sgq_quantize_tokens does.  No call here launches a kernel."""
import helpers  # noqa: F401

P = 4096  # an aligned address that no call here reaches


def test_refusals(sgq):
    lib = sgq.load_library()
    good = dict(x=P, dtype=0, ldx=64, M=2, K=64, codes=P, ldc=128, scales=P)
    for bad, status in [(dict(M=-1), 1), (dict(K=-1), 1), (dict(K=131072, ldx=131072, ldc=131072), 2), (dict(dtype=3), 1),
                        (dict(ldx=63), 1), (dict(x=None), 1), (dict(x=P + 2), 1), (dict(codes=None), 1), (dict(codes=P + 8), 1),
                        (dict(ldc=64), 1), (dict(ldc=136), 1), (dict(scales=None), 1), (dict(ldc=2**21 + 16), 2)]:
        for fn in (lib.sgq_quantize_tokens, lib.sgq_quantize_tokens_keep_nan):
            assert fn(*{**good, **bad}.values(), None) == status, bad
    assert b"sgq_quantize_tokens_keep_nan" in lib.sgq_last_error()
    assert lib.sgq_quantize_tokens_keep_nan(None, 1, 0, 0, 64, None, 0, None, None) == 0
