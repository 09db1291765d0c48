"""Norms of heads whose squares fp32 does not hold."""
import pytest
import torch

from test_attention_gpu import TYPES, Batch, _close, _randn, _turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


# (size of the elements, eps): squares past fp32's range, at its border, ordinary beside both, below it
SIZES = [(1e36, 1e-5), (2e18, 1e-5), (1e-19, 0.0), (1e-30, 0.0), (1e-30, 1e-5), (1e-10, 1e-35)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", range(len(SIZES)))
@pytest.mark.parametrize("shape", [(4, 2, 128, 128, False), (3, 1, 80, 20, False), (2, 2, 16, 16, True), (1, 1, 256, 0, False)])
def test_sizes(op, dev, shape, size, dtype):
    """Every second head of ordinary size, so that a wavefront has both."""
    H, KV, d, rot, interleaved = shape
    scale, eps = SIZES[size]
    if dtype is torch.float16:
        scale = 3e4 if scale > 1 else 2e-6  # whose squares fp32 has: nothing changes
    b = Batch(op, dev, [(5, 40), (1, 7)], 16, KV, d, dtype)
    qk = (_randn(dev, 1, b.rows, H + KV, d) / 4).clamp(-1, 1)
    qk[:, ::2] *= scale
    qk = qk.to(dtype)
    q, k, v = qk[:, :H], qk[:, H:], _randn(dev, 2, b.rows, KV, d).to(dtype)
    g = 1 + 0.2 * _randn(dev, 3, d)
    freqs = op.rotary_frequencies(rot, device=dev) if rot else None
    out = op.norm_rope_append(q, k, v, b.kv, b.batch, freqs, g, g, eps, interleaved)
    pos = torch.tensor([35, 36, 37, 38, 39, 6], device=dev)
    seq = torch.tensor([0, 0, 0, 0, 0, 1], device=dev)
    _close(out, *_turned(q, g, eps, freqs, pos, interleaved), d, dtype)
    _close(b.k[b.table[seq, pos // 16].long(), pos % 16], *_turned(k, g, eps, freqs, pos, interleaved), d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_heads_that_are_not_finite_or_zero(op, dev, dtype):
    """As the formula has them: x / inf, inf / inf, 0 / sqrt(eps), 0 / 0."""
    b = Batch(op, dev, [(3, 9)], 16, 1, 64, dtype)
    q = _randn(dev, 1, 3, 2, 64).to(dtype)
    q[0, 0, 5], q[1, 0, 7], q[2, 0] = float("inf"), float("nan"), 0
    g = torch.ones(64, device=dev)
    kv = q[:, 1:].contiguous()
    y = op.norm_rope_append(q, kv, kv, b.kv, b.batch, q_norm=g)
    assert bool(y[0, 0, 5].isnan()) and int((y[0, 0] == 0).sum()) == 63 and bool(y[1, 0].isnan().all()) and bool((y[2, 0] == 0).all())
    y0 = op.norm_rope_append(q, kv, kv, b.kv, b.batch, q_norm=g, eps=0.0)
    assert bool(y0[2, 0].isnan().all())
    want, mag = _turned(q[:, 1:], g, 1e-5, None, None, False)
    _close(y[:, 1:], want, mag, 64, dtype)
