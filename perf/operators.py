"""Operators of paged generation: cases, their plain forms, and their definition in 64 bits.

``kind`` names the operator:

  append   paged_qkv_append: one new token per sequence: QK norm, RoPE, k and v into the pages
  write    paged_write: the prompts' k and v into the pages
  attend   paged_attention: one new token per sequence over its pages, with or without the
           accumulated weights
  evict    paged_evict: every layer of a cache bounded by accumulated weight
  sample   sample_tokens: temperature, top-k, top-p and min-p from given random numbers

Head counts and dims are the package's presets (20m: 8/4 heads of 40, 150m: 12/4 of 64, 350m:
16/4 of 80, 1b: 16/8 of 128), vocabularies the presets' 100000 and the benchmark's 32000.
Pages are handed out in random order from a pool that is somewhat larger than the batch needs,
as a server's pool looks after a while.  Nothing that an operator overwrites feeds its own
inputs, so a pass can be repeated on the same state.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
HEADS = {"20m": (8, 4, 40), "tiny": (4, 2, 64), "150m": (12, 4, 64), "350m": (16, 4, 80), "1b": (16, 8, 128)}
LARGEST = 1.2e9  # bytes: no drawn case costs more than the largest listed ones


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One user of the smallest preset, 500 tokens in: a call whose latency is all it costs.
        {"name": "append-20m-1", "kind": "append", "preset": "20m", "B": 1, "max": 500, "page": 16, "ragged": False,
         "norm": True},
        # A serving batch of the 1B preset, every sequence at a length of its own.
        {"name": "append-1b-256", "kind": "append", "preset": "1b", "B": 256, "max": 512, "page": 64, "ragged": True,
         "norm": True},
        # Eight right-padded prompts of the 1B preset, up to its 2048 positions.
        {"name": "write-1b-prompts", "kind": "write", "preset": "1b", "B": 8, "max": 2048, "page": 64, "ragged": True},
        # One user of the smallest preset: heads of 40, pages of 16 tokens.
        {"name": "attend-20m-1", "kind": "attend", "preset": "20m", "B": 1, "max": 500, "page": 16, "ragged": False,
         "weights": False},
        # Heads of 80 in groups of 4, ragged lengths up to an odd 4099, with the weights that eviction goes by.
        {"name": "attend-350m-weights", "kind": "attend", "preset": "350m", "B": 16, "max": 4099, "page": 32,
         "ragged": True, "weights": True},
        # A serving batch of the 1B preset at ragged lengths up to its 2048 positions.
        {"name": "attend-1b-ragged", "kind": "attend", "preset": "1b", "B": 64, "max": 2048, "page": 64, "ragged": True,
         "weights": False},
        # Few sequences over long documents.
        {"name": "attend-1b-long", "kind": "attend", "preset": "1b", "B": 4, "max": 65536, "page": 128, "ragged": False,
         "weights": False},
        # A bounded cache of the 150M preset in its steady state: each step evicts one token a head.
        {"name": "evict-150m-one", "kind": "evict", "preset": "150m", "layers": 12, "B": 4, "max": 1025, "keep": 1024,
         "recent": 256, "page": 64, "mixed": True, "ragged": False},
        # Prompts of the 1B preset cut to half their length once.
        {"name": "evict-1b-half", "kind": "evict", "preset": "1b", "layers": 24, "B": 8, "max": 2048, "keep": 1024,
         "recent": 128, "page": 64, "mixed": False, "ragged": True},
        # generate()'s defaults for one user.
        {"name": "sample-1-topk", "kind": "sample", "B": 1, "V": 100000, "dtype": "bf16", "temperature": 1.0,
         "top_k": 50, "top_p": 0.9, "min_p": 0.0, "rows": False},
        # A batch of logits that a caller post-processed in fp32, cut by min-p alone.
        {"name": "sample-64-minp", "kind": "sample", "B": 64, "V": 32000, "dtype": "fp32", "temperature": 0.8,
         "top_k": 0, "top_p": 1.0, "min_p": 0.05, "rows": False},
        # A serving batch, each row with settings of its own.
        {"name": "sample-256-rows", "kind": "sample", "B": 256, "V": 100000, "dtype": "bf16", "temperature": 0.9,
         "top_k": 0, "top_p": 0.95, "min_p": 0.0, "rows": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "write", "attend", "attend", "evict", "sample", "sample"])
    if kind == "sample":
        V = _log(rng, 50, 131000)
        case = {"kind": kind, "B": _log(rng, 1, 300), "V": V, "dtype": rng.choice(["bf16", "fp32"]),
                "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]) if rng.random() < 0.5 else rng.uniform(0.2, 2.0),
                "top_k": rng.choice([0, 1, _log(rng, 2, V), _log(rng, 2, 200)]),
                "top_p": rng.choice([1.0, rng.uniform(0.05, 1.0), 0.9]),
                "min_p": rng.choice([0.0, 0.0, rng.uniform(0.001, 0.5)]), "rows": rng.random() < 0.4}
        return case
    preset = rng.choice(list(HEADS))
    nq, nkv, D = HEADS[preset]
    page = rng.choice([16, 32, 64, 128, 256])
    ragged = rng.random() < 0.7
    token = nkv * D * 4  # bytes of k and v
    while True:
        if kind == "append":
            case = {"kind": kind, "preset": preset, "B": _log(rng, 1, 512), "max": _log(rng, 1, 1024), "page": page,
                    "ragged": ragged, "norm": rng.random() < 0.8}
            size = case["B"] * case["max"] * token
        elif kind == "write":
            case = {"kind": kind, "preset": preset, "B": _log(rng, 1, 32), "max": _log(rng, 1, 4096), "page": page,
                    "ragged": ragged}
            size = 2 * case["B"] * case["max"] * token
        elif kind == "attend":
            case = {"kind": kind, "preset": preset, "B": _log(rng, 1, 256), "max": _log(rng, 1, 65536), "page": page,
                    "ragged": ragged, "weights": rng.random() < 0.4}
            size = case["B"] * case["max"] * token
        else:
            n = _log(rng, 2, 4096)
            keep = max(1, min(n, n - _log(rng, 1, n) + 1))
            case = {"kind": kind, "preset": preset, "layers": rng.choice([1, 2, 6, 12, 24]), "B": _log(rng, 1, 32),
                    "max": n, "keep": keep, "recent": rng.randint(0, keep), "page": page, "mixed": rng.random() < 0.5,
                    "ragged": ragged}
            size = case["layers"] * case["B"] * case["max"] * token
        if size <= LARGEST:
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """Tokens of each sequence, from the case alone: the longest is the case's ``max``."""
    B, n = case["B"], case["max"]
    if not case["ragged"]:
        return [n] * B
    # Evenly spread over 1 .. max in a fixed, unsorted order.
    return [1 + (n - 1) * ((b * 37 + B - 1) % B if math.gcd(37, B) == 1 else B - 1 - b) // max(1, B - 1) if B > 1 else n
            for b in range(B)]


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _pool(case, g, layers=None):
    """Pages [.., pages, nkv, page, D] of random values and a block table into them."""
    _, nkv, D = HEADS[case["preset"]]
    page, B = case["page"], case["B"]
    width = -(-case["max"] // page)
    pages = B * width + max(1, B * width // 16)
    shape = ([] if layers is None else [layers]) + [pages, nkv, page, D]
    k = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    v = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    order = torch.randperm(pages, generator=g, device=DEV)[:B * width]
    return k, v, order.view(B, width).to(torch.int32)


def _rotary(n, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32).to(DEV).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "sample":
        B, V = case["B"], case["V"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # Logits of a language model: a broad body and a few tokens well above it.
        x = torch.randn(B, V, generator=g, device=DEV) * 2.0
        few = torch.randint(0, V, (B, 8), generator=g, device=DEV)
        x.scatter_add_(1, few, 4.0 + 3.0 * torch.rand(B, 8, generator=g, device=DEV))
        st["logits"] = x.to(dt)
        st["uniforms"] = torch.rand(B, generator=g, device=DEV)
        names = ("temperature", "top_k", "top_p", "min_p")
        if case["rows"]:
            r = torch.rand(4, B, generator=g, device=DEV)
            st["temperature"] = (case["temperature"] * (0.5 + r[0])).contiguous()
            st["top_k"] = (case["top_k"] * (0.5 + r[1])).to(torch.int32)
            st["top_p"] = torch.clamp(case["top_p"] * (0.8 + 0.3 * r[2]), max=1.0)
            st["min_p"] = (case["min_p"] * r[3]).contiguous()
        else:
            st.update({n: case[n] for n in names})
        return st
    nq, nkv, D = HEADS[case["preset"]]
    B = case["B"]
    lens = _lengths(case)
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["k_pages"], st["v_pages"], st["table"] = _pool(case, g, case.get("layers"))
    bf = {"generator": g, "device": DEV, "dtype": torch.bfloat16}
    if kind == "append":
        st["qkv"] = torch.randn(B, (nq + 2 * nkv) * D, **bf)
        st["positions"] = st["lengths"] - 1
        st["cos_sin"] = _rotary(case["max"], D)
        w = 1.0 + 0.1 * torch.randn(2, D, generator=g, device=DEV)
        w = w.to(torch.bfloat16)
        st["q_norm"], st["k_norm"] = (w[0], w[1]) if case["norm"] else (None, None)
    elif kind == "write":
        st["k"] = torch.randn(B, nkv, case["max"], D, **bf)
        st["v"] = torch.randn(B, nkv, case["max"], D, **bf)
    elif kind == "attend":
        # Queries somewhat larger than the keys: weights as uneven as a trained head's.
        st["q"] = (1.5 * torch.randn(B, nq, D, generator=g, device=DEV)).to(torch.bfloat16)
        cap = st["table"].shape[1] * case["page"]
        st["weights"] = torch.rand(B, nkv, cap, generator=g, device=DEV) if case["weights"] else None
    else:
        L, cap = case["layers"], st["table"].shape[1] * case["page"]
        at = torch.arange(cap, device=DEV)
        n = st["lengths"].view(1, B, 1, 1)
        pos = at.expand(L, B, nkv, cap)
        if case["mixed"]:
            # After earlier evictions any slot holds any position; the newest token is in the last slot.
            shuffle = torch.rand(L, B, nkv, cap, generator=g, device=DEV)
            shuffle = torch.where(at < n - 1, shuffle, 2.0 + at.float())
            pos = torch.argsort(shuffle, -1)
        live = at < n
        st["slot_positions"] = torch.where(live, pos, -1).to(torch.int32).contiguous()
        st["positions"] = st["lengths"] - 1
        # Attention received so far: heavy-tailed, growing with a token's age; some got none.
        age = (n - pos).clamp(min=0).float() / case["max"]
        u = torch.rand(L, B, nkv, cap, generator=g, device=DEV)
        w = age * u.pow(4) * 10.0
        st["weights"] = torch.where(live & (u > 0.02), w, 0.0).contiguous()
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_package = None


def _cdx():
    global _package
    if _package is None:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "complexity-deep_amd"))
        import complexity_deep
        _package = complexity_deep
    return _package


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["kind"]](state, case)


def _own_append(st, case):
    q = _cdx().paged_qkv_append(st["qkv"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["positions"],
                                HEADS[case["preset"]][0], st["cos_sin"], st["q_norm"], st["k_norm"], EPS)
    return q, st["k_pages"], st["v_pages"]


def _own_write(st, case):
    _cdx().paged_write(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["lengths"])
    return st["k_pages"], st["v_pages"]


def _own_attend(st, case):
    return _cdx().paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"],
                                  weights=st["weights"])


def _own_evict(st, case):
    new = _cdx().paged_evict(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["positions"], st["weights"],
                             st["slot_positions"], case["keep"], case["recent"])
    return (*new, st["k_pages"], st["v_pages"])


def _own_sample(st, case):
    return _cdx().sample_tokens(st["logits"], st["uniforms"], temperature=st["temperature"], top_k=st["top_k"],
                                top_p=st["top_p"], min_p=st["min_p"])


_OWN = {"append": _own_append, "write": _own_write, "attend": _own_attend, "evict": _own_evict, "sample": _own_sample}


def _slots(table, page, slots):
    """(page, row in it) of slots [B, n]."""
    return torch.gather(table.long(), 1, slots // page), slots % page


def _norm_rope(x, w, cs):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    x1, x2 = x.chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _plain_append(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    x = st["qkv"].float().view(-1, nq + 2 * nkv, D)
    cs = st["cos_sin"][st["positions"].long()].unsqueeze(1)
    q = _norm_rope(x[:, :nq], st["q_norm"], cs).to(torch.bfloat16)
    k = _norm_rope(x[:, nq:nq + nkv], st["k_norm"], cs)
    pg, row = _slots(st["table"], case["page"], (st["lengths"].long() - 1).unsqueeze(1))
    st["k_pages"][pg[:, 0], :, row[:, 0]] = k.to(torch.bfloat16)
    st["v_pages"][pg[:, 0], :, row[:, 0]] = x[:, nq + nkv:].to(torch.bfloat16)
    return q, st["k_pages"], st["v_pages"]


def _plain_write(st, case):
    page, table = case["page"], st["table"].long()
    B, nkv, S, D = st["k"].shape
    pad = table.shape[1] * page - S
    live = (torch.arange(S + pad, device=DEV) < st["lengths"].unsqueeze(1)).view(B, -1, 1, page, 1)
    for new, pages in ((st["k"], st["k_pages"]), (st["v"], st["v_pages"])):
        x = torch.nn.functional.pad(new, (0, 0, 0, pad)).view(B, nkv, -1, page, D).transpose(1, 2)
        pages[table] = torch.where(live, x, pages[table])
    return st["k_pages"], st["v_pages"]


def _plain_attend(st, case):
    q, table, lens = st["q"].float(), st["table"].long(), st["lengths"].long()
    B, nq, D = q.shape
    nkv, page = st["k_pages"].shape[1:3]
    cap = table.shape[1] * page
    k = st["k_pages"][table].transpose(1, 2).reshape(B, nkv, cap, D).float()
    s = torch.matmul(q.view(B, nkv, nq // nkv, D), k.transpose(-1, -2).contiguous()) * D ** -0.5
    del k
    seen = (torch.arange(cap, device=DEV) < lens.unsqueeze(1)).view(B, 1, 1, cap)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = st["v_pages"][table].transpose(1, 2).reshape(B, nkv, cap, D).float()
    v = v.masked_fill(~seen.view(B, 1, cap, 1), 0.0)
    o = torch.matmul(p, v).reshape(B, nq * D).to(torch.bfloat16)
    if st["weights"] is None:
        return o
    return o, st["weights"] + p.sum(2)


def _plain_evict(st, case):
    table, lens, keep = st["table"].long(), st["lengths"].long(), case["keep"]
    L, B, nkv, cap = st["weights"].shape
    page = case["page"]
    at = torch.arange(cap, device=DEV)
    live = (at < lens.unsqueeze(1)).view(1, B, 1, cap)
    recent = st["slot_positions"] > (st["positions"] - case["recent"]).view(1, B, 1, 1)
    rank = torch.where(live, 1 + recent.int(), 0)
    w = torch.nan_to_num(st["weights"], nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    order = torch.argsort(w, dim=-1, descending=True, stable=True)
    order = torch.gather(order, -1, torch.argsort(torch.gather(rank, -1, order), dim=-1, descending=True, stable=True))
    count = lens.clamp(max=keep).view(1, B, 1, 1)
    kept = torch.zeros(L, B, nkv, cap, dtype=torch.bool, device=DEV)
    kept.scatter_(-1, order, (at < count).expand(L, B, nkv, cap))
    # Slot j < keep takes its own row, or the next kept row of the slots from keep on.
    n = min(keep, cap)
    hole = live & ~kept & (at < n)
    movers = torch.where(kept & (at >= n), at, cap).sort(-1).values
    nth = (torch.cumsum(hole, -1) - 1).clamp(min=0)
    source = torch.where(hole, torch.gather(movers, -1, nth), at)[..., :n]
    src_page = torch.gather(table.view(1, B, 1, -1).expand(L, B, nkv, -1), -1, source // page)
    dst_page = table[:, at[:n] // page].view(1, B, 1, n).expand(L, B, nkv, n)
    layer = torch.arange(L, device=DEV).view(L, 1, 1, 1)
    head = torch.arange(nkv, device=DEV).view(1, 1, nkv, 1)
    for pages in (st["k_pages"], st["v_pages"]):
        pages[layer, dst_page, head, at[:n] % page] = pages[layer, src_page, head, source % page]
    new_w = torch.zeros_like(st["weights"])
    new_p = torch.full_like(st["slot_positions"], -1)
    inside = at[:n] < count
    new_w[..., :n] = torch.where(inside, torch.gather(st["weights"], -1, source), 0.0)
    new_p[..., :n] = torch.where(inside, torch.gather(st["slot_positions"], -1, source), -1)
    return lens.clamp(max=keep).to(torch.int32), new_w, new_p, st["k_pages"], st["v_pages"]


def _column(x, B, dt):
    # Settings are taken in 32 bits, as numbers and as tensors.
    if not torch.is_tensor(x):
        x = torch.full((B,), x, dtype=torch.int32 if isinstance(x, int) else torch.float32, device=DEV)
    return x.to(dt).view(B, 1)


def _plain_sample(st, case):
    # In 64 bits: a token's share of the sum is compared with a random number.
    x = st["logits"].double()
    B, V = x.shape
    T, p, mp = (_column(st[n], B, torch.float64) for n in ("temperature", "top_p", "min_p"))
    k = _column(st["top_k"], B, torch.int64)
    srt, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    top = srt[:, :1]
    kth = torch.gather(srt, 1, torch.where((k > 0) & (k < V), k, V) - 1)
    w = torch.exp((srt - top) / torch.where(T > 0, T, 1.0))
    w = torch.where(srt >= kth, w, 0.0)
    before = torch.cumsum(w, -1) - w
    keep = (before <= p * w.sum(-1, keepdim=True)) | (p >= 1)
    w = torch.where(keep & (w >= mp), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, idx, w)
    cum = torch.cumsum(w, -1)
    drawn = (cum > st["uniforms"].double().unsqueeze(1) * cum[:, -1:]).int().argmax(-1)
    return torch.where(T[:, 0] > 0, drawn, idx[:, 0])


_PLAIN = {"append": _plain_append, "write": _plain_write, "attend": _plain_attend, "evict": _plain_evict,
          "sample": _plain_sample}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 12 * case["B"], "flops": 4 * n}
    nq, nkv, D = HEADS[case["preset"]]
    B, lens = case["B"], _lengths(case)
    table = 4 * sum(-(-n // case["page"]) for n in lens) + 4 * B
    if kind == "append":
        values = (nq + 2 * nkv) * D
        return {"bytes": B * (4 * values + 4 * D + 12), "flops": 10 * B * values}
    if kind == "write":
        return {"bytes": 8 * nkv * D * sum(lens) + table, "flops": 0}
    if kind == "attend":
        extra = 8 * nkv * sum(lens) if case["weights"] else 0
        return {"bytes": 4 * nkv * D * sum(lens) + 4 * B * nq * D + table + extra, "flops": 4 * nq * D * sum(lens)}
    moved = 0.0
    for n in lens:
        over = n - case["keep"]
        if over <= 0:
            continue
        rec = min(case["recent"], over)
        old = n - case["recent"]
        moved += rec + ((case["keep"] - case["recent"]) * max(0, over - rec) / old if old > 0 else 0)
    cap = -(-case["max"] // case["page"]) * case["page"]
    rows = case["layers"] * nkv
    return {"bytes": int(rows * (8 * sum(lens) + 8 * B * cap + moved * 8 * D)) + table, "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _exact_append(st, case)
    if kind == "write":
        return _exact_write(st, case)
    if kind == "attend":
        return _exact_attend(st, case)
    if kind == "evict":
        return _exact_evict(st, case)
    return _exact_sample(st, case)


def _exact_append(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    x = st["qkv"].double().reshape(case["B"], nq + 2 * nkv, D)
    pos = st["positions"].long()
    cos, sin = st["cos_sin"].double()[pos, :, 0], st["cos_sin"].double()[pos, :, 1]

    def head(i, w):
        y = x[:, i]
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * w.double()
        a, b = y[:, :D // 2], y[:, D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], 1)

    q = torch.stack([head(i, st["q_norm"]) for i in range(nq)], 1)
    k, v = st["k_pages"].double(), st["v_pages"].double()
    rows = torch.stack([head(nq + i, st["k_norm"]) for i in range(nkv)], 1)
    table = st["table"].cpu().numpy()
    for b, n in enumerate(_lengths(case)):
        page, row = divmod(n - 1, case["page"])
        k[table[b, page], :, row] = rows[b]
        v[table[b, page], :, row] = x[b, nq + nkv:]
    return q, k, v


def _exact_write(st, case):
    k, v = st["k_pages"], st["v_pages"]
    table = st["table"].cpu().numpy()
    for b, n in enumerate(_lengths(case)):
        for i in range(-(-n // case["page"])):
            lo = i * case["page"]
            hi = min(n, lo + case["page"])
            k[table[b, i], :, :hi - lo] = st["k"][b, :, lo:hi]
            v[table[b, i], :, :hi - lo] = st["v"][b, :, lo:hi]
    return k, v


def _exact_attend(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    out = torch.empty(case["B"], nq, D, dtype=torch.float64, device=DEV)
    weights = None if st["weights"] is None else st["weights"].double()
    for b, n in enumerate(_lengths(case)):
        used = st["table"][b, :-(-n // case["page"])].long()
        for h in range(nkv):
            k = st["k_pages"][used, h].reshape(-1, D)[:n].double()
            v = st["v_pages"][used, h].reshape(-1, D)[:n].double()
            heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            p = torch.softmax(k @ st["q"][b, heads].double().t().contiguous() / math.sqrt(D), 0)
            out[b, heads] = p.t().contiguous() @ v
            if weights is not None:
                weights[b, h, :n] += p.sum(1)
    out = out.view(case["B"], nq * D)
    return out if weights is None else (out, weights)


def _exact_evict(st, case):
    L, B, nkv, cap = st["weights"].shape
    keep, page = case["keep"], case["page"]
    w, pos = st["weights"].cpu().numpy(), st["slot_positions"].cpu().numpy()
    last, table = st["positions"].cpu().numpy(), st["table"].cpu().numpy()
    new_w, new_p = np.zeros_like(w), np.full_like(pos, -1)
    lens = _lengths(case)
    at = {n: [] for n in ("layer", "head", "dst", "dst_row", "src", "src_row")}
    for l in range(L):
        for b, n in enumerate(lens):
            for h in range(nkv):
                m = min(n, keep)
                old = pos[l, b, h, :n] <= last[b] - case["recent"]
                best = np.lexsort((np.arange(n), -w[l, b, h, :n].astype(np.float64), old))[:m]
                src = np.arange(m)
                if n > keep:
                    holes = np.setdiff1d(src, best)
                    src[holes] = np.sort(best[best >= keep])
                    at["layer"].append(np.full(len(holes), l))
                    at["head"].append(np.full(len(holes), h))
                    for name, slots in (("dst", holes), ("src", src[holes])):
                        at[name].append(table[b, slots // page])
                        at[name + "_row"].append(slots % page)
                new_w[l, b, h, :m] = w[l, b, h, src]
                new_p[l, b, h, :m] = pos[l, b, h, src]
    k, v = st["k_pages"], st["v_pages"]
    if at["layer"]:
        i = {n: torch.from_numpy(np.concatenate(a).astype(np.int64)).to(DEV) for n, a in at.items()}
        for pages in (k, v):
            pages[i["layer"], i["dst"], i["head"], i["dst_row"]] = pages[i["layer"], i["src"], i["head"], i["src_row"]]
    return (torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device=DEV), torch.from_numpy(new_w).to(DEV),
            torch.from_numpy(new_p).to(DEV), k, v)


def _exact_sample(st, case):
    x = st["logits"].float().cpu().numpy().astype(np.float64)
    B, V = x.shape
    u = st["uniforms"].cpu().numpy().astype(np.float64)

    def rows(name, dt):
        s = st[name]
        return np.full(B, np.float32(s) if dt != np.int64 else s, dt) if not torch.is_tensor(s) else \
            s.cpu().numpy().astype(dt)

    T, p, mp, k = rows("temperature", np.float64), rows("top_p", np.float64), rows("min_p", np.float64), \
        rows("top_k", np.int64)
    out = np.empty(B, np.int64)
    for b in range(B):
        if not T[b] > 0:
            out[b] = int(x[b].argmax())
            continue
        w = np.exp((x[b] - x[b].max()) / T[b])
        if 0 < k[b] < V:
            w[x[b] < np.partition(x[b], V - k[b])[V - k[b]]] = 0.0
        if p[b] < 1:
            order = np.argsort(-x[b], kind="stable")
            run_ = np.cumsum(w[order])
            first_out = 1 + int(np.searchsorted(run_, p[b] * run_[-1], side="right"))
            w[order[first_out:]] = 0.0
        w[w < mp[b]] = 0.0
        run_ = np.cumsum(w)
        out[b] = int(np.searchsorted(run_, u[b] * run_[-1], side="right"))
    return torch.from_numpy(out).to(DEV)
