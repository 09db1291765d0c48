"""The 8-bit token and channel entry points refuse bad arguments before any GPU work, and their size queries answer on
the host.  No call here launches a kernel: the addresses are never read."""
import pytest
import torch

import helpers  # noqa: F401

P = 4096  # an aligned address that no call here reaches


@pytest.fixture(scope="module")
def lib(sgq):
    return sgq.load_library()


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.w8a8 as w8a8

    return w8a8


def test_sizes(lib):
    assert [lib.sgq_tokens_row_bytes(k) for k in (0, 1, 128, 129, 131071)] == [128, 128, 128, 256, 131072]
    assert lib.sgq_tokens_row_bytes(131072) == -1 and lib.sgq_tokens_row_bytes(-1) == -1
    for K, N in [(1, 1), (128, 16), (129, 17), (4096, 11008)]:
        assert lib.sgq_channels_packed_bytes(K, N) == -(-N // 16) * 16 * (-(-K // 128) * 128)
        assert lib.sgq_channels_workspace_bytes(K, N) >= 4 * N + 4
    assert lib.sgq_channels_packed_bytes(0, 5) == 0 and lib.sgq_channels_packed_bytes(5, 0) == 0
    assert lib.sgq_channels_packed_bytes(131072, 16) == -1 and lib.sgq_channels_packed_bytes(16, -1) == -1
    for fn in (lib.sgq_linear_w8a8_workspace_bytes, lib.sgq_swiglu_w8a8_workspace_bytes):
        for shape in [(0, 0, 0), (1, 1, 1), (1, 4096, 4096), (128, 1024, 1024), (2048, 4096, 11008), (3, 0, 5)]:
            assert fn(*shape, 256) >= 0
        assert fn(1, 131072, 16, 256) == -1 and fn(-1, 1, 1, 256) == -1 and fn(1, 1, 1, -1) == -1


def _plan(lib, gated, M, K, N, cus=256):
    import ctypes

    form, ks = ctypes.c_int(-1), ctypes.c_int(-1)
    assert lib.sgq_w8a8_plan(gated, M, K, N, cus, ctypes.byref(form), ctypes.byref(ks)) == 0
    return form.value, ks.value


def test_plans(lib):
    """Every form has shapes of its own, every split of K its stages of 128, and the workspace is the partial sums'."""
    seen = set()
    for cus in (1, 32, 64, 128, 256, 304):
        for gated in (0, 1):
            for K in (0, 1, 100, 640, 1024, 2043, 4096, 11008, 14336, 131071):
                for N in (1, 40, 1024, 4096, 5001, 28672):
                    for M in (1, 16, 17, 32, 33, 64, 100, 128, 200, 333, 512, 1000, 2048, 8192):
                        form, ks = _plan(lib, gated, M, K, N, cus)
                        seen.add(form)
                        assert (form == 0) == (K == 0) and (form == 1) == (K > 0 and M <= 16)
                        stages = -(-K // 128)
                        assert ks == 1 or (form >= 5 and (ks - 1) * -(-stages // ks) < stages)
                        fn = lib.sgq_swiglu_w8a8_workspace_bytes if gated else lib.sgq_linear_w8a8_workspace_bytes
                        want = 0 if ks == 1 else ks * (1 + gated) * M * -(-N // 16) * 64
                        assert fn(M, K, N, cus) == want
    assert seen == set(range(10))
    assert _plan(lib, 0, 8192, 8192, 28672) == (9, 1)
    import ctypes

    i = ctypes.c_int()
    assert lib.sgq_w8a8_plan(0, 1, 131072, 1, 256, ctypes.byref(i), ctypes.byref(i)) == 1
    assert lib.sgq_w8a8_plan(0, 1, 1, 1, 256, None, ctypes.byref(i)) == 1


def test_tokens_refusals(lib):
    q = lib.sgq_quantize_tokens
    good = dict(x=P, dtype=0, ldx=64, M=2, K=64, codes=P, ldc=128, scales=P)

    def call(fn=q, **kw):
        return fn(*{**good, **kw}.values(), None)

    assert call(M=-1) == 1 and call(K=-1) == 1 and call(K=131072, ldx=131072, ldc=131072) == 2
    assert call(dtype=3) == 1 and call(dtype=-1) == 1
    assert call(ldx=63) == 1 and call(x=None) == 1 and call(x=P + 2) == 1 and call(dtype=1, x=P + 1) == 1
    assert call(codes=None) == 1 and call(codes=P + 8) == 1
    assert call(ldc=64) == 1 and call(ldc=136) == 1 and call(K=129, ldx=129, ldc=128) == 1
    assert b"128" in lib.sgq_last_error() or b"256" in lib.sgq_last_error()
    assert call(scales=None) == 1
    assert call(M=0, x=None, codes=None, scales=None) == 0
    d = dict(codes=P, ldc=128, scales=P, M=2, K=64, out=P, dtype=0, ldo=64)
    deq = lambda **kw: lib.sgq_dequantize_tokens(*{**d, **kw}.values(), None)  # noqa: E731
    assert deq(dtype=9) == 1 and deq(out=None) == 1 and deq(ldo=63) == 1 and deq(codes=P + 4) == 1
    assert deq(scales=None) == 1 and deq(K=-1) == 1 and deq(M=0) == 0 and deq(K=0) == 0


def test_norm_refusals(lib):
    good = dict(x=P, dtype=1, ldx=64, r=P, ldr=64, h=P, ldh=64, g=P, eps=1e-5, M=2, K=64, codes=P, ldc=128, scales=P)

    def call(**kw):
        return lib.sgq_rms_norm_tokens(*{**good, **kw}.values(), None)

    assert call(dtype=5) == 1 and call(M=-3) == 1 and call(K=200000) == 2
    assert call(g=None) == 1 and call(scales=None) == 1 and call(x=None) == 1 and call(h=None) == 1
    assert call(r=None) == 1  # h without a residual
    assert call(ldh=65) == 1  # h over x, with another stride
    assert call(ldr=60) == 1 and call(ldx=10) == 1 and call(ldh=3, h=2 * P) == 1
    assert call(codes=P + 1) == 1 and call(ldc=120) == 1
    assert call(M=0) == 0


def test_norm_refuses_h_across_an_input(lib):
    """h is an input, with its stride, or shares nothing with either."""
    good = dict(x=P, dtype=1, ldx=64, r=16 * P, ldr=64, h=P, ldh=64, g=P, eps=1e-5, M=4, K=64, codes=P, ldc=128,
                scales=P)

    def clash(**kw):
        st = lib.sgq_rms_norm_tokens(*{**good, **kw}.values(), None)
        return st == 1 and b"over an input" in lib.sgq_last_error()

    for d in (2, 128, 2 * 64 * 3, 2 * (64 * 3 + 63)):  # an element, a row, the last row, the last element
        assert clash(h=P + d) and clash(h=P - d) and clash(h=16 * P + d) and clash(h=16 * P - d)
    assert clash(h=P + 2, M=1) and clash(h=P - 126, M=1, ldx=4096, ldr=64, ldh=4096)
    wide = dict(ldx=200, ldr=64, ldh=200)
    for d in (1, 63, 137, 199):
        assert clash(h=P + 2 * d, **wide) and clash(h=P - 2 * d, **wide)
    assert clash(h=P, ldh=65) and clash(h=P + 2 * 64, ldh=65)


def test_channels_refusals(lib):
    ws = lib.sgq_channels_workspace_bytes(64, 32)
    assert lib.sgq_quantize_channels(P, 64, 32, None, P, P, None, 0, None) == 3
    assert lib.sgq_quantize_channels(P, 64, 32, None, P, P, P, ws - 1, None) == 3
    assert lib.sgq_quantize_channels(P, 64, 32, None, P, P, P + 4, ws, None) == 3
    assert lib.sgq_quantize_channels(P, 64, 32, None, None, P, P, ws, None) == 1
    assert lib.sgq_quantize_channels(None, 64, 32, None, P, P, P, ws, None) == 1
    assert lib.sgq_quantize_channels(P, 64, 32, None, P, P + 8, P, ws, None) == 1
    assert lib.sgq_quantize_channels(P, 131072, 32, None, P, P, P, ws, None) == 2
    assert lib.sgq_quantize_channels(P, 64, 0, None, None, None, None, 0, None) == 0
    assert lib.sgq_pack_channels(P, 64, 32, None, P, ws, None) == 1
    assert lib.sgq_pack_channels(P, 64, 32, P, None, 0, None) == 3
    assert lib.sgq_pack_channels(P, -64, 32, P, P, ws, None) == 1
    assert lib.sgq_unpack_channels(P + 1, 64, 32, P, None) == 1
    assert lib.sgq_dequantize_channels(P, None, 64, 32, P, None) == 1


def test_product_refusals(lib):
    good = dict(codes=P, ldc=128, sx=P, M=2, K=64, N=32, packed=P, sw=P, bias=None, y=P, dtype=0, ldy=32, ws=P,
                nws=1 << 40)

    def call(**kw):
        return lib.sgq_linear_w8a8(*{**good, **kw}.values(), None)

    assert call(M=-1) == 1 and call(N=-1) == 1 and call(K=131072, ldc=131072) == 2
    assert call(dtype=3) == 1 and call(y=None) == 1 and call(y=P + 2) == 1 and call(ldy=31) == 1
    assert call(codes=None) == 1 and call(codes=P + 8) == 1 and call(ldc=127) == 1 and call(ldc=100) == 1
    assert call(sx=None) == 1 and call(packed=None) == 1 and call(packed=P + 8) == 1 and call(sw=None) == 1
    assert call(M=0) == 0 and call(N=0, ldy=0) == 0
    g = dict(codes=P, ldc=128, sx=P, M=2, K=64, N=32, pg=P, sg=P, bg=None, pu=P, su=P, bu=None, h=P, dtype=0, ldh=32,
             ws=P, nws=1 << 40)
    sw = lambda **kw: lib.sgq_swiglu_w8a8(*{**g, **kw}.values(), None)  # noqa: E731
    assert sw(pu=None) == 1 and sw(su=None) == 1 and sw(pu=P + 1) == 1 and sw(h=None) == 1 and sw(K=-5) == 1
    assert sw(M=0) == 0


def test_python_refuses_host_tensors(op):
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="device"):
        op.quantize_int8_tokens(x)
    with pytest.raises(ValueError, match="device"):
        op.rms_norm_int8_tokens(x, torch.ones(64))
    with pytest.raises(ValueError, match="device"):
        op.quantize_int8_channels(x)
    t = op.TokensInt8(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), 64)
    with pytest.raises(ValueError, match="device"):
        op.dequantize_int8_tokens(t)
