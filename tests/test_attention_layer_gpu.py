"""QuantizedAttentionInt8 as a layer of a program."""
import pytest
import torch

import attention_layer_reference as R
from test_attention_gpu import TYPES, _i32, _layers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences", [0, 2])
@pytest.mark.parametrize("added", [False, True])
def test_no_tokens(op, dev, dtype, sequences, added):
    """A step without tokens is one like any other."""
    attn, mlp = _layers(op, dev, dtype, n=1)[0]
    kv = op.PagedKV(*(torch.full((4, 16, 2, 64), 3, dtype=dtype, device=dev) for _ in range(2)))
    batch = op.SequenceBatch(torch.zeros(sequences, 2, dtype=torch.int32, device=dev), _i32(dev, [5] * sequences),
                             _i32(dev, [0] * (sequences + 1)), 16, 1)
    x = torch.empty(0, 256, dtype=dtype, device=dev)
    y, h = attn.forward(x, kv, batch, residual=x.clone() if added else None)
    assert y.shape == h.shape == (0, 256) and y.dtype == dtype
    y, h = mlp.forward(y, residual=h)
    assert y.shape == (0, 256)
    assert bool((kv.k == 3).all() and (kv.v == 3).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", R.VARIANTS)
@pytest.mark.parametrize("steps", [1, 3])
def test_the_layer_against_64_bits(op, dev, name, dtype, steps):
    """Outputs of three sequences, at once and in steps (what a prefix shows ahead has to be there: at once)."""
    import soverign_grad_amd.w8a8 as w8a8

    K, H, KV, d, page, lens = 64, 4, 2, 16, 8, [40, 1, 23]
    parts, proj, norm = R.weights(K, H, KV, d, 1)
    made, window, calls = R.variant(name, K, H, KV, d, lens)
    there = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in made.items()}
    attn = op.QuantizedAttentionInt8.from_float(*(w.to(dev) for w in parts + [proj]), norm.to(dev), H, KV, window=window, **there)
    held = [w8a8.dequantize_int8_channels(w8a8.quantize_int8_channels(w.to(dev))).cpu().double() for w in parts + [proj]]
    added = R.VARIANTS[name].get("added", True)
    made = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in made.items()}
    tokens, want = [], []
    for i, (n, call) in enumerate(zip(lens, calls)):
        x, res, total = R.inputs(n, K, 20 + i)
        tokens.append((x if added else total, res))
        normed = total / torch.sqrt(total.pow(2).mean(-1, keepdim=True) + 1e-5) * norm.double()
        pos = torch.arange(n) if call["positions"] is None else call["positions"]
        want.append(R.layer(normed, held[:3], held[3], H, KV, pos, call["seen"], R.HALF[dtype], **made) + (total,))
    kv = op.PagedKV(*(torch.full((16, page, KV, d), float("nan"), dtype=dtype, device=dev) for _ in range(2)))
    table = torch.randperm(16, generator=torch.Generator().manual_seed(5))[:15].reshape(3, 5).int().to(dev)
    cuts = [[n * s // steps for s in range(steps + 1)] for n in lens]
    if "prefix" in R.VARIANTS[name]:
        cuts = [[0, n] for n in lens]
    for s in range(len(cuts[0]) - 1):
        spans = [slice(c[s], c[s + 1]) for c in cuts]
        starts = [0]
        for span in spans:
            starts.append(starts[-1] + span.stop - span.start)
        batch = op.SequenceBatch(table, _i32(dev, [span.stop for span in spans]), _i32(dev, starts), 40, max(b - a for a, b in zip(starts, starts[1:])))
        take = lambda key: None if calls[0][key] is None else torch.cat([c[key][span] for c, span in zip(calls, spans)]).to(dev)
        x, res = (torch.cat([t[i][span] for t, span in zip(tokens, spans)]).to(dev, dtype) for i in range(2))
        prefix = _i32(dev, [c["prefix"] for c in calls]) if "prefix" in calls[0] else None
        y, h = attn.forward(x, kv, batch, residual=res if added else None, positions=take("positions"), prefix=prefix,
                            first_key=take("first_key"))
        for i, span in enumerate(spans):
            out, bound, total = (t[span] for t in want[i])
            assert torch.equal(h[starts[i] : starts[i + 1]].cpu().double(), total)
            got = y[starts[i] : starts[i + 1]].cpu().double()
            over = ((got - out).abs() / bound).nan_to_num(9.0)
            assert not over.numel() or float(over.max()) <= 1, (s, i, float(over.max()))
