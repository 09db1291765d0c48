"""The attention half of a block over a paged key/value cache, as cases to time and to compare.

The cache is a pool of pages, [pages, page, kv_heads, head_dim] for keys and for values;
a sequence's table names its pages in order.  A batch holds some new tokens of each
sequence, one sequence after the other: new token i of a sequence with n new tokens
and `len` keys (the new ones included) stands at position len - n + i.  The plain forms
below are elementary torch operations; with `own` true the same passes go through the
package's entry points.

Kinds:
  append  RMSNorm of every head of q and k, the position rotation, and the new keys
          and values into their pages
  attend  attention of the new tokens over the cache
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

PKG_DIR = Path(__file__).resolve().parents[1] / "soverign-grad_amd"
EPS = 1e-5
BASE = 10000.0
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def attention():
    """soverign-grad_amd/ as the package `soverign_grad_amd` (its folder's name is no identifier)."""
    name = "soverign_grad_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, PKG_DIR / "__init__.py",
                                                      submodule_search_locations=[str(PKG_DIR)])
        sys.modules[name] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    import soverign_grad_amd.attention as mod

    return mod


# ---- the cases -------------------------------------------------------------


def append(name, B, new, past, heads, kv_heads, d, dtype, page=16, rot=None, interleaved=False, norm=True,
           ragged=False):
    """B sequences of up to `past` cached and `new` new tokens; rot: how much of a head is rotated."""
    return {"name": name, "kind": "append", "B": B, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "d": d, "dtype": dtype, "page": page, "rot": d if rot is None else rot, "interleaved": interleaved,
            "norm": norm, "ragged": ragged}


def attend(name, B, new, past, heads, kv_heads, d, dtype, page=16, softcap=0.0, alibi=False, window=0, prefix=0,
           docs=1, ragged=False):
    """docs: documents that a sequence is packed from; prefix: keys that every token sees."""
    return {"name": name, "kind": "attend", "B": B, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "d": d, "dtype": dtype, "page": page, "softcap": softcap, "alibi": alibi, "window": window,
            "prefix": prefix, "docs": docs, "ragged": ragged}


def listed():
    return [
        # A decode step of eight sequences of a 2048-wide model in fp32: launch and latency.
        append("append_step", 8, 1, 511, 16, 16, 128, "fp32"),
        # A prompt's chunk on grouped heads.
        append("append_prompt", 1, 2048, 0, 32, 8, 128, "bf16"),
        # Ragged prompts, heads of no power of two, part of a head rotated, neighbours in pairs.
        append("append_odd", 5, 333, 77, 12, 3, 80, "fp16", rot=48, interleaved=True, ragged=True),
        # Several long prompts at once on the widest model.
        append("append_large", 4, 4096, 0, 64, 8, 128, "bf16", page=64),
        # A decode step of eight sequences of a 2048-wide model in fp32.
        attend("decode_step", 8, 1, 511, 16, 16, 128, "fp32"),
        # A served batch, each sequence with a cache of its own length.
        attend("decode_batch", 64, 1, 8191, 32, 8, 128, "bf16", ragged=True),
        # One sequence with a very long cache: few rows, the keys to be shared out.
        attend("decode_long", 1, 1, 131071, 32, 8, 128, "bf16", page=64),
        # A prompt from its start.
        attend("chunk_prompt", 1, 2048, 0, 32, 8, 128, "bf16"),
        # A chunk of a long prompt: wide heads, capped scores, a sliding window.
        attend("chunk_window", 1, 1024, 15000, 16, 8, 256, "fp16", softcap=50.0, window=4096, page=32),
        # A chunk in fp32 with a bias by distance, ragged lengths.
        attend("chunk_distance", 2, 333, 1000, 16, 16, 128, "fp32", alibi=True, ragged=True),
        # Ragged sequences packed from documents, after a prefix that both sides see.
        attend("chunk_documents", 7, 777, 300, 12, 4, 64, "bf16", prefix=100, docs=3, ragged=True),
        # Several long prompts on the widest model: the largest call.
        attend("chunk_large", 4, 8192, 0, 64, 8, 128, "bf16", page=64),
    ]


LARGEST_PAIRS = 4 * 8192 * 8193 // 2 * 64 * 128  # pairs of a row and a key, times heads and width
LARGEST_KEYS = 64 * 8192 * 8 * 128  # a cache's keys, times heads and width
LARGEST_ROWS = 4 * 4096 * (64 + 2 * 8) * 128


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7, 8]) if kv_heads <= 8 else kv_heads
    d = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    c = {"kind": rng.choice(["append", "attend", "attend", "attend"]), "heads": heads, "kv_heads": kv_heads, "d": d,
         "dtype": dtype, "page": rng.choice([16, 32, 64, 128]), "ragged": rng.random() < 0.6}
    c["B"] = rng.choice([1, _log_int(rng, 2, 8), _log_int(rng, 8, 64)])
    c["new"] = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 512), _log_int(rng, 513, 8192)])
    c["past"] = rng.choice([0, _log_int(rng, 1, 1024), _log_int(rng, 1025, 131071)])
    B, size = c["B"], BYTES[dtype] // 2
    if c["kind"] == "append":
        c["new"] = max(1, min(c["new"], LARGEST_ROWS // size // (B * (heads + 2 * kv_heads) * d)))
        c["past"] = min(c["past"], 4096)
        c["rot"] = rng.choice([d, d, d // 2, 32])
        return dict(c, interleaved=rng.random() < 0.5, norm=rng.random() < 0.7)
    keys = max(2, LARGEST_KEYS // size // (B * kv_heads * d))
    c["new"] = min(c["new"], keys // 2)
    c["past"] = min(c["past"], keys - c["new"])
    # fp32 runs at a sixteenth of the 16-bit matrix rate
    pairs = LARGEST_PAIRS // (4 if size == 1 else 32) // (B * heads * d)
    while c["new"] > 1 and c["new"] * (c["past"] + c["new"]) > pairs:
        c["new"] = (c["new"] + 1) // 2
        if c["new"] == 1:
            c["past"] = min(c["past"], max(1, pairs))
    return dict(c, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3,
                window=rng.choice([0, 0, _log_int(rng, 16, 4096)]), prefix=rng.choice([0, 0, _log_int(rng, 1, 1000)]),
                docs=rng.choice([1, 1, 3]))


# ---- a batch's lengths (of the case alone) ---------------------------------


def _lengths(c):
    """(new tokens, keys) of every sequence; the first one's are the largest."""
    rng = random.Random(1000003 * c["B"] + 1009 * c["new"] + c["past"])
    out = [(c["new"], c["past"] + c["new"])]
    for _ in range(c["B"] - 1):
        n, p = c["new"], c["past"]
        if c["ragged"]:
            n, p = rng.randint(1, n), rng.randint(0, p)
        out.append((n, p + n))
    return out


def _document_starts(c, n, length):
    """First key of the document of each of a sequence's n new tokens."""
    rng = random.Random(31 * length + n)
    cuts = sorted({0, *(rng.randrange(length) for _ in range(c["docs"] - 1))})
    starts, i = [], 0
    for p in range(length - n, length):
        while i + 1 < len(cuts) and cuts[i + 1] <= p:
            i += 1
        starts.append(cuts[i])
    return starts


def _intervals(c):
    """For each sequence the first key and the end of the keys of every new token."""
    out = []
    for n, length in _lengths(c):
        first = _document_starts(c, n, length) if c["docs"] > 1 else [0] * n
        lo, hi = [], []
        for i in range(n):
            p = length - n + i
            lo.append(max(first[i], p - c["window"] + 1 if c["window"] else 0))
            hi.append(max(p + 1, min(c["prefix"], length)))
        out.append((lo, hi))
    return out


# ---- inputs ----------------------------------------------------------------


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda:0", dtype=torch.float32) * std


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda:0")


def prepare(case, seed):
    c, dtype = case, TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(int(seed))
    H, KV, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    lengths = _lengths(c)
    used = [-(-length // page) for _, length in lengths]
    # Pages of the sequences in no order, a few of the pool free; the rows behind a
    # sequence's end hold what an earlier one left.
    pool = sum(used) + 4
    order = torch.randperm(pool, generator=gen, device="cuda:0").to(torch.int32)
    table = torch.zeros(c["B"], max(used), dtype=torch.int32, device="cuda:0")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at : at + n]
        at += n
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    T = starts[-1]
    s = {"case": c, "dtype": dtype, "lengths": lengths, "starts": starts, "table": table}
    s["k_cache"] = _normal(gen, pool, page, KV, d).to(dtype)
    s["v_cache"] = _normal(gen, pool, page, KV, d).to(dtype)
    if own:  # a serving program makes them once, the batch for each step of all layers
        s["kv"] = attention().PagedKV(s["k_cache"], s["v_cache"])
        s["batch"] = attention().SequenceBatch(table, _ints([n for _, n in lengths]), _ints(starts),
                                               max_len=max(n for _, n in lengths), max_new=c["new"])
    if c["kind"] == "append":
        # What a fused projection leaves: q, k and v side by side in a row.
        qkv = _normal(gen, T, H + 2 * KV, d).to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H : H + KV], qkv[:, H + KV :]
        half = c["rot"] // 2
        s["freqs"] = BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda:0") / half)
        s["q_norm"] = 1 + _normal(gen, d, std=0.1) if c["norm"] else None
        s["k_norm"] = 1 + _normal(gen, d, std=0.1) if c["norm"] else None
        return s
    s["q"] = _normal(gen, T, H, d, std=2.0).to(dtype)
    intervals = _intervals(c)
    s["lo"], s["hi"] = _ints([v for lo, _ in intervals for v in lo]), _ints([v for _, hi in intervals for v in hi])
    s["slopes"] = (2.0 ** (-8.0 * (torch.arange(H, device="cuda:0") + 1) / H)).float() if c["alibi"] else None
    s["prefix"] = _ints([min(c["prefix"], n) for _, n in lengths]) if c["prefix"] else None
    first = [v for n, length in lengths for v in _document_starts(c, n, length)] if c["docs"] > 1 else None
    s["first_key"] = None if first is None else _ints(first)
    return s


# ---- one pass --------------------------------------------------------------


def _plain_rotate(x, s, norm, cos, sin):
    c, half = s["case"], s["case"]["rot"] // 2
    u = x.float()
    if norm is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * norm
    if c["interleaved"]:
        a, b = u[..., 0 : 2 * half : 2], u[..., 1 : 2 * half : 2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = u[..., :half], u[..., half : 2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, u[..., 2 * half :]], -1).to(s["dtype"])


def _plain_append(s):
    c, dev = s["case"], s["q"].device
    pos = torch.cat([torch.arange(length - n, length, device=dev) for n, length in s["lengths"]])
    seq = torch.cat([torch.full((n,), b, device=dev) for b, (n, _) in enumerate(s["lengths"])])
    angle = pos.double()[:, None] * s["freqs"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    page, row = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k_cache"][page, row] = _plain_rotate(s["k"], s, s["k_norm"], cos, sin)
    s["v_cache"][page, row] = s["v"]
    return {"q": _plain_rotate(s["q"], s, s["q_norm"], cos, sin), "k": s["k_cache"], "v": s["v_cache"]}


def _plain_attend(s):
    c = s["case"]
    H, KV, d = c["heads"], c["kv_heads"], c["d"]
    g = H // KV
    out = torch.empty_like(s["q"])
    for b, (n, length) in enumerate(s["lengths"]):
        rows = slice(s["starts"][b], s["starts"][b + 1])
        pages = s["table"][b, : -(-length // c["page"])].long()
        k = s["k_cache"][pages].flatten(0, 1)[:length].float()
        v = s["v_cache"][pages].flatten(0, 1)[:length].float()
        j = torch.arange(length, device=k.device)
        seen = (j >= s["lo"][rows, None]) & (j < s["hi"][rows, None])
        away = (torch.arange(length - n, length, device=k.device)[:, None] - j).abs().float()
        some = max(1, 2**29 // (g * n * length))  # kv heads at a time
        for h0 in range(0, KV, some):
            h1 = min(KV, h0 + some)
            q = s["q"][rows, h0 * g : h1 * g].float().transpose(0, 1).reshape(h1 - h0, g * n, d)
            score = torch.matmul(q, k[:, h0:h1].permute(1, 2, 0).contiguous()).view(h1 - h0, g, n, length)
            score = score / math.sqrt(d)
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            if c["alibi"]:
                score = score - s["slopes"][h0 * g : h1 * g].view(h1 - h0, g, 1, 1) * away
            score = score.masked_fill(~seen, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = p.view(h1 - h0, g * n, length)
            o = torch.matmul(p, v[:, h0:h1].transpose(0, 1).contiguous()).view(h1 - h0, g, n, d)
            o = torch.where(total > 0, o / total, 0.0)
            out[rows, h0 * g : h1 * g] = o.reshape((h1 - h0) * g, n, d).transpose(0, 1).to(s["dtype"])
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_append(s) if c["kind"] == "append" else _plain_attend(s)
    op = attention()
    if c["kind"] == "append":
        q = op.norm_rope_append(s["q"], s["k"], s["v"], s["kv"], s["batch"], freqs=s["freqs"], q_norm=s["q_norm"],
                                k_norm=s["k_norm"], eps=EPS, interleaved=c["interleaved"])
        return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}
    return op.paged_attention(s["q"], s["kv"], s["batch"], softcap=c["softcap"], alibi_slopes=s["slopes"],
                              window=c["window"], prefix=s["prefix"], first_key=s["first_key"])


# ---- what a pass cannot do without -----------------------------------------


def work(case):
    c, e = case, BYTES[case["dtype"]]
    H, KV, d = c["heads"], c["kv_heads"], c["d"]
    rows = sum(n for n, _ in _lengths(c))
    if c["kind"] == "append":
        n = rows * (H + 2 * KV) * d
        return {"bytes": 2 * e * n, "flops": 8 * n}
    pairs = keys = 0
    for lo, hi in _intervals(c):
        pairs += sum(max(0, b - a) for a, b in zip(lo, hi))
        keys += max(0, max(hi) - min(lo))
    return {"bytes": 2 * e * (rows * H * d + keys * KV * d), "flops": 4 * pairs * H * d}


# ---- the same in 64 bits ---------------------------------------------------


def _exact_head(x, weight, c, angle):
    """One kind of head's rows [T, heads, d] after norm and rotation, by complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["d"] + EPS) * weight.double()
    rot, half = c["rot"], c["rot"] // 2
    pairs = x[..., :rot].unflatten(-1, (half, 2)) if c["interleaved"] else x[..., :rot].unflatten(-1, (2, half)).mT
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z if c["interleaved"] else z.mT
    return torch.cat([z.flatten(-2), x[..., rot:]], -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lengths = s["lengths"]
    if c["kind"] == "append":
        pos = [p for n, length in lengths for p in range(length - n, length)]
        angle = torch.tensor(pos, dtype=torch.float64, device="cuda:0").outer(s["freqs"])
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        k, v = _exact_head(s["k"], s["k_norm"], c, angle), s["v"].double()
        at = 0
        for b, (n, length) in enumerate(lengths):
            for page in range((length - n) // c["page"], -(-length // c["page"])):
                first, end = max(length - n, page * c["page"]), min(length, (page + 1) * c["page"])
                rows = slice(at + first - (length - n), at + end - (length - n))
                where = (int(s["table"][b, page]), slice(first - page * c["page"], end - page * c["page"]))
                k_cache[where], v_cache[where] = k[rows], v[rows]
            at += n
        return {"q": _exact_head(s["q"], s["q_norm"], c, angle), "k": k_cache, "v": v_cache}
    g, at, parts = c["heads"] // c["kv_heads"], 0, []
    for b, ((n, length), (lo, hi)) in enumerate(zip(lengths, _intervals(c))):
        pages = s["table"][b, : -(-length // c["page"])].long()
        j = torch.arange(length, device="cuda:0", dtype=torch.float64)
        lo, hi = (torch.tensor(v, device="cuda:0", dtype=torch.float64)[:, None] for v in (lo, hi))
        here = torch.arange(length - n, length, device="cuda:0", dtype=torch.float64)[:, None]
        hidden = (j < lo) | (j >= hi)
        heads = []
        for h in range(c["heads"]):
            key = s["k_cache"][pages, :, h // g].reshape(-1, c["d"])[:length].double()
            value = s["v_cache"][pages, :, h // g].reshape(-1, c["d"])[:length].double()
            score = s["q"][at : at + n, h].double() @ key.T * c["d"] ** -0.5
            if c["softcap"]:
                score = torch.tanh(score / c["softcap"]) * c["softcap"]
            if c["alibi"]:
                score = score - (here - j).abs() * s["slopes"][h].double()
            weight = torch.softmax(score.masked_fill_(hidden, -math.inf), -1).nan_to_num_(nan=0.0)
            heads.append(weight @ value)
        parts.append(torch.stack(heads, 1))
        at += n
    return torch.cat(parts)
