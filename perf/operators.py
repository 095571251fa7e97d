"""Head norms with rotation, rotated appends and attention of several tokens, as cases to time and compare.

A case is a dict of plain values; ``prepare`` makes the tensors (and, where the framework's own calls are asked for, the
plan and the rotation) that a serving program holds before a call, ``run`` is one pass, ``exact`` the same result in
64 bits. Three kinds of pass:

* ``rotate``: each head of new queries and keys is normed and turned by its token's position;
* ``append``: the same, with the keys and the values written into the paged cache;
* ``tokens``: several new tokens of each sequence attend to its pages, causally or (an encoder's states) to all of them.

With ``own`` false the passes are elementary torch operations in 32 bits; with ``own`` true they are the framework's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

# fmt -> (type of queries and new tokens, type of the cache)
_TYPES = {
    "f32": (torch.float32, torch.float32),
    "f16": (torch.float16, torch.float16),
    "bf16": (torch.bfloat16, torch.bfloat16),
    "e4m3": (torch.float16, torch.float8_e4m3fn),
    "e5m2": (torch.float16, torch.float8_e5m2),
    "bf16_e4m3": (torch.bfloat16, torch.float8_e4m3fn),
}

# What a case holds unless it says otherwise: 32 query and 8 KV heads of 128 dims, pages of 16 tokens. `context` is the
# longest sequence after the new tokens; `counts`: every sequence brings `tokens` new ones, or from one to that many.
_DEFAULTS = {"fmt": "bf16", "batch": 4, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "context": 4096, "tokens": 1,
             "lengths": "uniform", "counts": "full", "causal": True, "norm": True, "style": "half", "rotary": 1.0,
             "fused": False, "base": 500000.0, "heavy": 0.0}
_EPS = 1e-6


def listed():
    return [
        # One decode step's queries and keys of a serving batch, normed and rotated.
        {"name": "rotate_bf16_b64_n1", "kind": "rotate", "batch": 64, "context": 32768, "lengths": "ragged"},
        # Prompts of four users, straight from a fused projection's rows.
        {"name": "rotate_f16_b4_n2048", "kind": "rotate", "fmt": "f16", "tokens": 2048, "context": 2048, "fused": True},
        # The precise path: neighbouring dims paired, half of them rotated, an odd number of tokens.
        {"name": "rotate_f32_b3_n333", "kind": "rotate", "fmt": "f32", "batch": 3, "q_heads": 8, "kv_heads": 2, "dim": 64,
         "tokens": 333, "context": 100000, "norm": False, "style": "interleaved", "rotary": 0.5},
        # The write of a decode step: one token of each of four sequences, rotated without norms. The smallest call.
        {"name": "append_f16_b4_n1", "kind": "append", "fmt": "f16", "fused": True, "norm": False},
        # Prompts of uneven lengths written into a quantised cache.
        {"name": "append_e4m3_b8_n1024", "kind": "append", "fmt": "e4m3", "batch": 8, "tokens": 1024, "context": 2048,
         "counts": "ragged", "fused": True},
        # Drafted tokens, scored in one pass over 4K contexts.
        {"name": "tokens_f16_b4_n4_l4096", "kind": "tokens", "fmt": "f16", "tokens": 4},
        # The same over a quantised cache: a serving batch of uneven contexts and numbers of drafts.
        {"name": "tokens_e4m3_b16_n8_l8192", "kind": "tokens", "fmt": "e4m3", "batch": 16, "tokens": 8, "context": 8192,
         "page": 32, "lengths": "ragged", "counts": "ragged"},
        # A chunk of a long prompt: its tokens see what came before them and each other.
        {"name": "tokens_bf16_b1_n2048_l8192", "kind": "tokens", "batch": 1, "tokens": 2048, "context": 8192, "heavy": 0.05},
        # Whole prompts: the largest pass.
        {"name": "tokens_f16_b2_n4096_l4096", "kind": "tokens", "fmt": "f16", "batch": 2, "tokens": 4096},
        # Odd numbers of tokens over a quantised cache, heads of 64 dims, seven query heads to a KV head.
        {"name": "tokens_bf16_e4m3_b5_n301_l1777", "kind": "tokens", "fmt": "bf16_e4m3", "batch": 5, "q_heads": 28,
         "kv_heads": 4, "dim": 64, "tokens": 301, "context": 1777, "lengths": "ragged", "counts": "ragged"},
        # A decoder's tokens over an encoder's states: no order between them, one KV head to a query head.
        {"name": "tokens_f16_b8_n96_l1500_full", "kind": "tokens", "fmt": "f16", "batch": 8, "q_heads": 16, "kv_heads": 16,
         "dim": 64, "tokens": 96, "context": 1500, "causal": False},
        # The precise path.
        {"name": "tokens_f32_b2_n33_l1000", "kind": "tokens", "fmt": "f32", "batch": 2, "q_heads": 8, "kv_heads": 2,
         "dim": 64, "tokens": 33, "context": 1000, "page": 32, "lengths": "ragged"},
    ]


_HEADS = [(32, 8, 128), (32, 8, 64), (32, 4, 128), (28, 4, 128), (40, 8, 128), (8, 2, 64), (16, 1, 64), (16, 16, 64),
          (16, 16, 128), (24, 3, 128), (64, 8, 128)]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: any kind, type, head layout and page size, 1 to 64 sequences, 1 to 4096 new tokens of each."""
    while True:
        q_heads, kv_heads, dim = rng.choice(_HEADS)
        case = {"kind": rng.choice(["rotate", "append", "tokens", "tokens", "tokens"]),
                "fmt": rng.choice(["f16", "f16", "bf16", "bf16", "e4m3", "e5m2", "bf16_e4m3", "f32"]),
                "batch": _between(rng, 1, 64), "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32]), "tokens": _between(rng, 1, 4096), "lengths": rng.choice(["uniform", "ragged"]),
                "counts": rng.choice(["full", "full", "ragged"])}
        case["context"] = max(case["tokens"], _between(rng, 17, 32768))
        if case["kind"] == "tokens":
            case["causal"] = rng.choice([True, True, True, False])
            case["heavy"] = rng.choice([0.0, 0.0, 0.05])
        else:
            case["norm"] = rng.choice([True, True, False])
            case["style"] = rng.choice(["half", "half", "interleaved"])
            case["rotary"] = rng.choice([1.0, 1.0, 0.5, 0.25])
            case["fused"] = rng.choice([True, False])
            case["base"] = rng.choice([10000.0, 500000.0])
        c = _full(case)
        scores = c["batch"] * c["q_heads"] * c["tokens"] * c["context"] if c["kind"] == "tokens" else 0
        cache = 2 * c["batch"] * c["context"] * kv_heads * dim * _TYPES[c["fmt"]][1].itemsize if c["kind"] != "rotate" else 0
        rows = c["batch"] * c["tokens"] * (q_heads + 2 * kv_heads) * dim
        w = work(case)
        if scores <= 1 << 30 and cache <= 1 << 29 and rows <= 1 << 27 and w["flops"] <= 1.3e11 and \
                w["flops"] / 1e15 + w["bytes"] / 6e12 <= 1.4e-4 and (c["fmt"] != "f32" or w["flops"] <= 1e10):
            return case


def _full(case):
    return {**_DEFAULTS, **case}


def _metadata(c):
    """Lengths after the new tokens, and the new tokens of each sequence: the case's own, so that each seed's pass is
    the same amount of work."""
    rng = np.random.default_rng(c["batch"] * 65537 + c["context"] * 31 + c["tokens"])
    counts = np.full(c["batch"], c["tokens"], dtype=np.int32)
    if c["counts"] == "ragged":
        counts[1:] = rng.integers(1, c["tokens"] + 1, size=c["batch"] - 1)
    lengths = np.full(c["batch"], c["context"], dtype=np.int32)
    if c["lengths"] == "ragged":  # a quarter of the context to all of it
        lengths[1:] = rng.integers(max(1, c["context"] // 4), c["context"] + 1, size=c["batch"] - 1)
    if c.get("causal", True):
        lengths = np.maximum(lengths, counts)
    return lengths, counts


def _table(c, seed):
    width = -(-c["context"] // c["page"])
    return np.random.default_rng(seed).permutation(c["batch"] * width).astype(np.int32).reshape(c["batch"], width)


def _values(shape, dtype, gen, heavy=0.0):
    """N(0, 1) values in the stored type with their scale (1 for unquantised types)."""
    if dtype.itemsize > 1:
        x = torch.randn(shape, device="cuda", dtype=dtype, generator=gen)
        if heavy:
            x.mul_(torch.where(torch.rand(shape, device="cuda", generator=gen) < heavy, 4.0, 1.0).to(dtype))
        return x, 1.0
    x = torch.randn(shape, device="cuda", dtype=torch.float16, generator=gen)
    return x.div_(_scale(dtype)).clamp_(-_largest(dtype), _largest(dtype)).to(dtype), _scale(dtype)


def _largest(dtype):
    return float(torch.finfo(dtype).max)


def _scale(dtype):
    """A calibrated scale, as a checkpoint carries it."""
    return 5.5 / _largest(dtype) if dtype.itemsize == 1 else 1.0


def prepare(case, seed):
    c = _full(case)
    x_type, kv_type = _TYPES[c["fmt"]]
    lengths, counts = _metadata(c)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    s["counts"] = torch.from_numpy(counts).cuda() if c["counts"] == "ragged" else None
    if c["kind"] != "rotate":
        table = _table(c, seed)
        s["table"] = torch.from_numpy(table).cuda()
    if c["kind"] == "tokens":
        s["lengths"] = torch.from_numpy(lengths).cuda()
        cache, s["scale"] = _values((2, table.size, c["page"], c["kv_heads"], c["dim"]), kv_type, gen, c["heavy"])
        s["k"], s["v"] = cache[0], cache[1]
        s["q"] = torch.randn((c["batch"], c["tokens"], c["q_heads"], c["dim"]), device="cuda", dtype=x_type, generator=gen)
        s["out"] = torch.empty_like(s["q"])
        if own:
            Layout, DecodePlan = _framework()[:2]
            layout = Layout(c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["page"], table.size)
            s["plan"] = DecodePlan(layout, table, lengths, query_tokens=c["tokens"])
        return s
    # The rows of the projections: fused in one tensor, or each in its own.
    heads = (c["q_heads"], c["kv_heads"], c["kv_heads"])
    rows = (c["batch"], c["tokens"])
    if c["fused"]:
        wide = torch.randn((*rows, sum(heads), c["dim"]), device="cuda", dtype=x_type, generator=gen)
        s["q"], s["k_new"], s["v_new"] = torch.split(wide, heads, dim=2)
    else:
        s["q"], s["k_new"], s["v_new"] = (torch.randn((*rows, h, c["dim"]), device="cuda", dtype=x_type, generator=gen)
                                          for h in heads)
    s["positions"] = torch.from_numpy((lengths - counts).astype(np.int32)).cuda()
    turned = int(c["dim"] * c["rotary"])
    s["frequencies"] = torch.pow(c["base"], -torch.arange(0, turned, 2, device="cuda", dtype=torch.float64) / turned)
    s["q_weight"] = s["k_weight"] = None
    if c["norm"]:
        s["q_weight"], s["k_weight"] = (1 + 0.2 * torch.randn((2, c["dim"]), device="cuda", generator=gen)).to(x_type)
    if c["kind"] == "append":
        s["k"], s["v"] = torch.zeros((2, table.size, c["page"], c["kv_heads"], c["dim"]), device="cuda", dtype=x_type).to(kv_type)
        s["scale"] = _scale(kv_type)
        # The program knows on the host how many tokens each prompt brings: their rows among all of them.
        j = np.arange(c["tokens"])
        s["rows"] = torch.from_numpy(np.flatnonzero(j[None, :] < counts[:, None])).cuda()
    if own:
        Layout, _, Rotary, s["rotate_heads"], s["append_rotated"] = _framework()
        s["rotation"] = Rotary(s["frequencies"], style=c["style"])
        if c["kind"] == "append":
            s["layout"] = Layout(c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["page"], table.size)
    return s


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paged-decode-lab_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from paged_decode.layout import Layout
    from paged_decode.rotary import Rotary, append_rotated, rotate_heads
    from paged_decode.runtime import DecodePlan
    return Layout, DecodePlan, Rotary, rotate_heads, append_rotated


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_tokens(state) if kind == "tokens" else _own_heads(state)
    return {"rotate": _rotate, "append": _append, "tokens": _tokens}[kind](state)


def _own_heads(s):
    if s["case"]["kind"] == "rotate":
        return s["rotate_heads"](s["q"], s["k_new"], s["positions"], s["rotation"], q_weight=s["q_weight"],
                                 k_weight=s["k_weight"], eps=_EPS)
    q = s["append_rotated"](s["layout"], s["k"], s["v"], s["table"], s["positions"], s["k_new"], s["v_new"],
                            s["rotation"], q=s["q"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS,
                            k_scale=s["scale"], v_scale=s["scale"], counts=s["counts"])
    return q, s["k"], s["v"]


def _own_tokens(s):
    return s["plan"].run_tokens(s["q"], s["k"], s["v"], causal=s["case"]["causal"], counts=s["counts"],
                                k_scale=s["scale"], v_scale=s["scale"], out=s["out"])


def _token_positions(s):
    return s["positions"].long()[:, None] + torch.arange(s["case"]["tokens"], device="cuda")


def _turned(x, weight, s):
    """The heads of x in 32 bits, normed and rotated; the angles in 64, which far positions need."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    angle = (_token_positions(s).double()[..., None] * s["frequencies"])[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    turned = 2 * s["frequencies"].numel()
    if s["case"]["style"] == "half":
        a, b = x[..., :turned // 2], x[..., turned // 2:turned]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., turned:]), -1)
    a, b = x[..., 0:turned:2], x[..., 1:turned:2]
    pairs = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((pairs, x[..., turned:]), -1)


def _rotate(s):
    return (_turned(s["q"], s["q_weight"], s).to(s["q"].dtype), _turned(s["k_new"], s["k_weight"], s).to(s["q"].dtype))


def _stored(x, scale, dtype):
    if dtype.itemsize == 1:
        x = (x / scale).clamp(-_largest(dtype), _largest(dtype))
    return x.to(dtype)


def _bytes(x):
    """FP8 pages as bytes, which every kind of indexing takes."""
    return x.view(torch.uint8) if x.dtype.itemsize == 1 else x


def _append(s):
    c = s["case"]
    position = _token_positions(s)
    page = torch.gather(s["table"].long(), 1, torch.clamp(position // c["page"], max=s["table"].shape[1] - 1))
    row = (page * c["page"] + position % c["page"]).flatten()[s["rows"]]
    for cache, new in ((s["k"], _turned(s["k_new"], s["k_weight"], s)), (s["v"], s["v_new"].float())):
        new = _stored(new.flatten(0, 1)[s["rows"]], s["scale"], cache.dtype)
        _bytes(cache.flatten(0, 1))[row] = _bytes(new)
    q = _turned(s["q"], s["q_weight"], s)
    if s["counts"] is not None:  # rows past a sequence's tokens are zeros
        live = torch.arange(c["tokens"], device="cuda") < s["counts"][:, None]
        q = torch.where(live[..., None, None], q, 0.0)
    return q.to(s["q"].dtype), s["k"], s["v"]


def _tokens(s):
    c = s["case"]
    batch, n, group = c["batch"], c["tokens"], c["q_heads"] // c["kv_heads"]
    at = s["table"].long()

    def dense(cache):  # [batch, kv_heads, tokens, dim] in 32 bits
        return _bytes(cache)[at].view(cache.dtype).flatten(1, 2).float().transpose(1, 2).contiguous()

    k, v = dense(s["k"]), dense(s["v"])
    q = s["q"].float().view(batch, n, c["kv_heads"], group, c["dim"]).permute(0, 2, 1, 3, 4).reshape(batch, c["kv_heads"], -1, c["dim"])
    scores = torch.matmul(q * (s["scale"] / math.sqrt(c["dim"])), k.transpose(2, 3).contiguous())
    lengths = s["lengths"].long()[:, None]
    counts = s["counts"].long()[:, None] if s["counts"] is not None else torch.full_like(lengths, n)
    j = torch.arange(n, device="cuda")
    sees = torch.minimum(lengths - counts + j + 1, lengths) if c["causal"] else lengths.expand(batch, n)
    sees = torch.where(j < counts, sees, 0)  # tokens that row j of each sequence attends to
    hidden = torch.arange(k.shape[2], device="cuda") >= sees[..., None]
    scores = scores.view(batch, c["kv_heads"], n, group, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = scores.sum(-1, keepdim=True).clamp_(min=1e-30)
    out = torch.matmul(scores.flatten(2, 3), v).view(batch, c["kv_heads"], n, group, -1) / total * s["scale"]
    return out.permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(s["q"].dtype)


def work(case):
    c = _full(case)
    x, kv = (t.itemsize for t in _TYPES[c["fmt"]])
    lengths, counts = (m.astype(np.int64) for m in _metadata(c))
    if c["kind"] == "tokens":
        j = np.arange(c["tokens"])[None, :]
        sees = np.minimum(lengths[:, None] - counts[:, None] + j + 1, lengths[:, None]) if c["causal"] else lengths[:, None] + 0 * j
        visible = int(np.where(j < counts[:, None], sees, 0).sum())
        row = c["q_heads"] * c["dim"] * x
        return {"bytes": 2 * int(lengths.sum()) * c["kv_heads"] * c["dim"] * kv + (int(counts.sum()) + c["batch"] * c["tokens"]) * row
                + 4 * int((-(-lengths // c["page"])).sum()),
                "flops": 4 * visible * c["q_heads"] * c["dim"]}
    if c["kind"] == "rotate":
        return {"bytes": 2 * c["batch"] * c["tokens"] * (c["q_heads"] + c["kv_heads"]) * c["dim"] * x, "flops": 0}
    live = int(counts.sum())
    return {"bytes": c["dim"] * (live * ((c["q_heads"] + 2 * c["kv_heads"]) * x + 2 * c["kv_heads"] * kv)
                                 + c["batch"] * c["tokens"] * c["q_heads"] * x), "flops": 0}


def _turned_64(x, weight, s):
    """The rotation as a product of complex numbers, in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * weight.double()
    turned = 2 * s["frequencies"].numel()
    angle = _token_positions(s).double()[:, :, None, None] * s["frequencies"]
    turn = torch.polar(torch.ones_like(angle), angle)
    part = x[..., :turned]
    pairs = part.unflatten(-1, (2, turned // 2)).transpose(-1, -2) if s["case"]["style"] == "half" else part.unflatten(-1, (turned // 2, 2))
    done = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    done = done.transpose(-1, -2) if s["case"]["style"] == "half" else done
    return torch.cat((done.flatten(-2), x[..., turned:]), -1)


def exact(case, seed):
    c = _full(case)
    s = prepare(case, seed)
    if c["kind"] == "rotate":
        return _turned_64(s["q"], s["q_weight"], s), _turned_64(s["k_new"], s["k_weight"], s)
    if c["kind"] == "append":
        lengths, counts = _metadata(c)
        caches = []
        for cache, new in ((s["k"], _turned_64(s["k_new"], s["k_weight"], s)), (s["v"], s["v_new"].double())):
            cells = cache.double()
            if cache.dtype.itemsize == 1:
                new = torch.clamp(new / s["scale"], -_largest(cache.dtype), _largest(cache.dtype))
            for b in range(c["batch"]):
                at = torch.arange(int(lengths[b] - counts[b]), int(lengths[b]), device="cuda")
                cells[s["table"][b].long()[at // c["page"]], at % c["page"]] = new[b, :int(counts[b])]
            caches.append(cells)
        q = _turned_64(s["q"], s["q_weight"], s)
        for b in range(c["batch"]):
            q[b, int(counts[b]):] = 0
        return q, *caches
    if work(case)["flops"] > 4e11:
        return None
    lengths, counts = _metadata(c)
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    group = c["q_heads"] // c["kv_heads"]
    for b in range(c["batch"]):
        n, new = int(lengths[b]), int(counts[b])
        pages = s["table"][b, :-(-n // c["page"])].long()
        for h in range(c["kv_heads"]):
            k, v = (_bytes(x)[pages, :, h].contiguous().view(x.dtype).reshape(-1, c["dim"])[:n].double() * s["scale"]
                    for x in (s["k"], s["v"]))
            for g in range(group):
                at = h * group + g
                weights = torch.mm(s["q"][b, :new, at].double(), k.T.contiguous()) / math.sqrt(c["dim"])
                if c["causal"]:
                    weights += torch.full_like(weights, -math.inf).triu(n - new + 1)
                out[b, :new, at] = torch.mm(torch.softmax(weights, -1), v)
    return out
