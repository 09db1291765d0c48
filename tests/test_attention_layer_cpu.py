"""The bounds that QuantizedAttentionInt8 is held to are narrow enough to show its mistakes: they are made here, in the
reference.  In fp32 all of them show (in 16 bits the bounds are wider, and the layer's steps the same)."""
import pytest
import torch

import attention_layer_reference as R

K, HEADS, KV, D, T = 64, 4, 2, 16, 40


def _run(name, dtype, change=None):
    parts, proj, norm = R.weights(K, HEADS, KV, D, 1)
    made, _, calls = R.variant(name, K, HEADS, KV, D, [T])
    _, _, total = R.inputs(T, K, 2)
    made = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in made.items()}
    a = dict(n=total / torch.sqrt(total.pow(2).mean(-1, keepdim=True) + 1e-5) * norm.double(), parts=[w.double() for w in parts],
             proj=proj.double(), pos=torch.arange(T) if calls[0]["positions"] is None else calls[0]["positions"],
             seen=calls[0]["seen"], **made)
    if change:
        change(a, total, norm)
    return R.layer(heads=HEADS, kv_heads=KV, h=R.HALF[dtype], **a)


def _swap(a, *_):
    a["parts"] = [a["parts"][0], a["parts"][2], a["parts"][1]]


def _no(key):
    def change(a, *_):
        a[key] = None
    return change


def _late(a, *_):
    a["pos"] = a["pos"] + torch.arange(len(a["pos"]))


def _without_residual(a, total, norm):
    x = R.inputs(T, K, 2)[0]
    a["n"] = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * norm.double()


def _without_norm(a, total, norm):
    a["n"] = a["n"] / norm.double()


def _sees_more(a, *_):
    a["seen"] = torch.ones_like(a["seen"]).tril()


def _set(**values):
    return lambda a, *_: a.update(values)


MISTAKES = [("plain", _swap), ("plain", _without_residual), ("plain", _without_norm), ("turned", _no("freqs")), ("turned", _late),
            ("turned", _set(interleaved=True)), ("norms", _no("q_norm")), ("norms", _no("k_norm")), ("biases", _no("qkv_bias")),
            ("biases", _no("proj_bias")), ("interleaved", _set(interleaved=False)),
            ("cap and window", _set(softcap=0.0)), ("cap and window", _sees_more), ("distance and documents", _no("alibi_slopes")),
            ("distance and documents", _sees_more), ("prefix", _sees_more), ("prefix", _set(scale=None)), ("all", _swap)]


@pytest.mark.parametrize("case", range(len(MISTAKES)))
def test_a_mistake_is_seen(case):
    name, change = MISTAKES[case]
    (want, bound), (got, _) = _run(name, torch.float32), _run(name, torch.float32, change)
    assert bool(torch.isfinite(want).all()) and float(bound.min()) > 0
    assert int(((got - want).abs() > bound).sum()) > want.numel() // 50
