"""Operators of several new tokens per sequence on a paged cache: cases, plain forms, definition in 64 bits.

``kind`` names the operator:

  reserve   paged_reserve: pages from a shared pool for the new tokens, and the map of their rows
  truncate  paged_truncate: sequences cut back, their pages returned to the pool
  append    paged_chunk_append: the projections of the new tokens: QK norm, RoPE, k and v into the pages
  attend    paged_chunk_attention: the new tokens over all tokens up to themselves

Head counts and dims are the package's presets (20m: 8/4 heads of 40, tiny: 4/2 of 64, 150m: 12/4
of 64, 350m: 16/4 of 80, 1b: 16/8 of 128).  How many tokens each sequence brings goes by ``mix``:

  even     ``new`` each
  ragged   1 .. ``new``, evenly spread in an unsorted order
  mixed    ``new`` for every sixteenth sequence, one for the others: prompts among running generations

and the tokens that it has already by ``old`` (0 .. ``old`` spread likewise, or ``old`` each if even).
``padded`` batches give every sequence ``new`` rows; others lie one behind the other.  Nothing that an operator
overwrites feeds its own inputs, so a pass can be repeated on the same state.
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
MOST_SCORES = 2.2e9  # of a padded batch: the largest listed one's
MOST_VALUES = 3.4e7  # of a projection


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One user's next token, the pool's pages of 16: a call whose latency is all it costs.
        {"name": "reserve-1", "kind": "reserve", "B": 1, "old": 511, "new": 1, "mix": "even", "page": 16,
         "padded": False, "short": False},
        # A server's batch: running generations with new prompts among them, the pool nearly used up.
        {"name": "reserve-256-mixed", "kind": "reserve", "B": 256, "old": 2048, "new": 512, "mix": "mixed", "page": 64,
         "padded": False, "short": True},
        # A padded batch of first prompts.
        {"name": "reserve-64-prompts", "kind": "reserve", "B": 64, "old": 0, "new": 2048, "mix": "ragged", "page": 64,
         "padded": True, "short": False},
        # Speculated tokens taken back, up to 8 of each sequence.
        {"name": "truncate-256", "kind": "truncate", "B": 256, "old": 2048, "drop": 8, "every": 1, "page": 16},
        # A quarter of a large batch has ended and gives all of its pages back.
        {"name": "truncate-1024-ended", "kind": "truncate", "B": 1024, "old": 4096, "drop": 4096, "every": 4,
         "page": 16},
        # Five speculated tokens of one user of the smallest preset.
        {"name": "append-20m-5", "kind": "append", "preset": "20m", "B": 1, "old": 500, "new": 5, "mix": "even",
         "page": 16, "norm": True},
        # Second turns of eight users of the 1B preset.
        {"name": "append-1b-turns", "kind": "append", "preset": "1b", "B": 8, "old": 1024, "new": 1024, "mix": "even",
         "page": 64, "norm": True},
        # The five tokens' attention: heads of 40, pages of 16.
        {"name": "attend-20m-5", "kind": "attend", "preset": "20m", "B": 1, "old": 500, "new": 5, "mix": "even",
         "page": 16, "padded": False},
        # Heads of 80 in groups of 4, chunks and contexts of all lengths in a padded batch.
        {"name": "attend-350m-ragged", "kind": "attend", "preset": "350m", "B": 16, "old": 3322, "new": 777,
         "mix": "ragged", "page": 32, "padded": True},
        # Four prompts of 512 among sixty running generations of the 1B preset.
        {"name": "attend-1b-mixed", "kind": "attend", "preset": "1b", "B": 64, "old": 1536, "new": 512, "mix": "mixed",
         "page": 64, "padded": False},
        # Second turns of eight users, to the preset's 2048 positions.
        {"name": "attend-1b-turns", "kind": "attend", "preset": "1b", "B": 8, "old": 1024, "new": 1024, "mix": "even",
         "page": 64, "padded": False},
        # The last piece of one long document.
        {"name": "attend-1b-long", "kind": "attend", "preset": "1b", "B": 1, "old": 63488, "new": 2048, "mix": "even",
         "page": 128, "padded": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["reserve", "truncate", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128, 256])
    mix = rng.choice(["even", "ragged", "mixed"])
    while True:
        B, old = _log(rng, 1, 1024), _log(rng, 1, 65536) - 1
        if kind == "truncate":
            case = {"kind": kind, "B": B, "old": old, "drop": rng.choice([_log(rng, 1, 16), _log(rng, 1, old + 1)]),
                    "every": _log(rng, 1, 16), "page": page}
            if B * old <= 8e6 and old > 0:
                return case
            continue
        new = _log(rng, 1, 4096)
        case = {"kind": kind, "B": B, "old": old, "new": new, "mix": mix, "page": page}
        if kind == "reserve":
            case.update(padded=rng.random() < 0.4, short=rng.random() < 0.4)
            if B * (old + new) <= 8e6 and B * new <= 262144:
                return case
            continue
        preset = rng.choice(list(HEADS))
        nq, nkv, D = HEADS[preset]
        case["preset"] = preset
        tokens = B * (old + new)
        if tokens * nkv * D > 1.4e8:  # K and V of 268 MB each
            continue
        if kind == "append":
            case["norm"] = rng.random() < 0.8
            if B * new * (nq + 2 * nkv) * D <= MOST_VALUES:
                return case
            continue
        case["padded"] = rng.random() < 0.3
        if B * nq * new * (old + new + page) <= MOST_SCORES and B * new * nq * D <= MOST_VALUES:
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _spread(B, lo, hi, step):
    """lo .. hi evenly over B sequences, in a fixed, unsorted order; hi for one alone."""
    if B == 1:
        return [hi]
    order = [(b * step + B - 1) % B if math.gcd(step, B) == 1 else B - 1 - b for b in range(B)]
    return [lo + (hi - lo) * o // (B - 1) for o in order]


def _counts(case):
    B, new = case["B"], case["new"]
    if case["mix"] == "even":
        return [new] * B
    if case["mix"] == "ragged":
        return _spread(B, 1, new, 37)
    return [new if b % 16 == 0 else 1 for b in range(B)]


def _before(case):
    """Tokens that each sequence has before the call."""
    if case.get("mix") == "even":
        return [case["old"]] * case["B"]
    return _spread(case["B"], 0 if case["kind"] != "truncate" else 1, case["old"], 59)


def _starts(case):
    if case.get("padded"):
        return [b * case["new"] for b in range(case["B"])]
    at, starts = 0, []
    for n in _counts(case):
        starts.append(at)
        at += n
    return starts


def _rows(case):
    return case["B"] * case["new"] if case.get("padded") else sum(_counts(case))


def _pages(n, page):
    return -(-n // page)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _rotary(n, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32).to(DEV).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, B, page = case["kind"], case["B"], case["page"]
    old = _before(case)
    st = {"case": case}
    if kind in ("reserve", "truncate"):
        # A pool in the order that its pages came back in.
        longest = case["old"] + case.get("new", 0)
        width = _pages(longest, page) + 1
        used = [_pages(n, page) for n in old]
        if kind == "reserve":
            need = [_pages(n + c, page) - u for n, c, u in zip(old, _counts(case), used)]
            free = max(1, sum(need) * 2 // 3 if case["short"] else sum(need) + 7)
        else:
            free = 11
        pool = sum(used) + free
        order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
        table = torch.full((B, width), -1, dtype=torch.int32)
        at, host = free, order.cpu()
        for b, u in enumerate(used):
            table[b, :u] = host[at:at + u]
            at += u
        st.update(free_pages=order.clone(), free_count=_ints([free]), block_table=table.to(DEV), lengths=_ints(old),
                  positions=_ints(old) - 1, num_pages=pool)
        if kind == "reserve":
            st["counts"] = _ints(_counts(case))
        else:
            # What stays of each: everything, or up to ``drop`` tokens less.
            gone = (torch.rand(B, generator=g, device=DEV) * (case["drop"] + 1)).long()
            if case["drop"] >= case["old"]:
                gone = torch.full_like(gone, case["drop"])
            gone[torch.arange(B, device=DEV) % case["every"] != 0] = 0
            st["to"] = (st["lengths"] - gone).clamp(min=0).to(torch.int32)
        return st
    nq, nkv, D = HEADS[case["preset"]]
    counts, R = _counts(case), _rows(case)
    longest = max(n + c for n, c in zip(old, counts))
    width = _pages(longest, page)
    pages = B * width + max(1, B * width // 16)
    bf = {"generator": g, "device": DEV, "dtype": torch.bfloat16}
    st["k_pages"] = torch.randn(pages, nkv, page, D, **bf)
    st["v_pages"] = torch.randn(pages, nkv, page, D, **bf)
    table = torch.randperm(pages, generator=g, device=DEV)[:B * width].view(B, width).to(torch.int32)
    if kind == "append":
        st["qkv"] = torch.randn(R, (nq + 2 * nkv) * D, **bf)
        before = torch.repeat_interleave(_ints(old, torch.int64), _ints(counts, torch.int64))
        first = torch.repeat_interleave(_ints(_starts(case), torch.int64), _ints(counts, torch.int64))
        seq = torch.repeat_interleave(torch.arange(B, device=DEV), _ints(counts, torch.int64))
        slot = before + torch.arange(R, device=DEV) - first
        st["row_slots"] = table[seq, slot // page].long() * page + slot % page
        st["row_positions"] = slot.to(torch.int32)
        st["cos_sin"] = _rotary(longest, D)
        w = (1.0 + 0.1 * torch.randn(2, D, generator=g, device=DEV)).to(torch.bfloat16)
        st["q_norm"], st["k_norm"] = (w[0], w[1]) if case["norm"] else (None, None)
    else:
        # Queries somewhat larger than the keys: weights as uneven as a trained head's.
        st["q"] = (1.5 * torch.randn(R, nq, D, generator=g, device=DEV)).to(torch.bfloat16)
        st["block_table"] = table
        st["starts"], st["counts"] = _ints(_starts(case)), _ints(counts)
        st["lengths"] = _ints([n + c for n, c in zip(old, counts)])
        st["most"] = max(counts)
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


def _own_reserve(st, case):
    rows = _cdx().paged_reserve(st["counts"], st["lengths"], st["positions"], st["block_table"], case["page"],
                                _rows(case), stride=case["new"] if case["padded"] else None,
                                free_pages=st["free_pages"], free_count=st["free_count"])
    return (rows.starts, rows.counts, rows.lengths, rows.positions, rows.free_count, rows.row_slots,
            rows.row_positions, st["block_table"])


def _own_truncate(st, case):
    new = _cdx().paged_truncate(st["to"], st["lengths"], st["positions"], st["block_table"], case["page"],
                                st["free_pages"], st["free_count"])
    return (*new, st["free_pages"])


def _own_append(st, case):
    q = _cdx().paged_chunk_append(st["qkv"], st["k_pages"], st["v_pages"], st["row_slots"], st["row_positions"],
                                  HEADS[case["preset"]][0], st["cos_sin"], st["q_norm"], st["k_norm"], EPS)
    return q, st["k_pages"], st["v_pages"]


def _own_attend(st, case):
    return _cdx().paged_chunk_attention(st["q"], st["k_pages"], st["v_pages"], st["block_table"], st["starts"],
                                        st["counts"], st["lengths"], max_tokens=st["most"])


_OWN = {"reserve": _own_reserve, "truncate": _own_truncate, "append": _own_append, "attend": _own_attend}


def _plain_reserve(st, case):
    page, R, table = case["page"], _rows(case), st["block_table"]
    B, width = table.shape
    n, length = st["counts"].long().clamp(min=0), st["lengths"].long()
    starts = torch.arange(B, device=DEV) * case["new"] if case["padded"] else torch.cumsum(n, 0) - n
    fits = (starts + n <= R) & (length + n <= width * page)
    if case["padded"]:
        fits &= n <= case["new"]
    have = (length + page - 1) // page
    need = torch.where(fits, (length + n + page - 1) // page - have, 0)
    upto = torch.cumsum(need, 0)
    free = st["free_count"].long()
    ok = fits & ((need == 0) | (upto <= free))
    n = torch.where(ok, n, 0)
    taken = torch.where(ok, need, 0)
    # The j-th new page of a sequence, in the table's columns.
    col = torch.arange(width, device=DEV)
    nth = col - have.unsqueeze(1)
    fresh = (nth >= 0) & (nth < taken.unsqueeze(1))
    at = (free - 1 - ((upto - need).unsqueeze(1) + nth)).clamp(0, st["free_pages"].numel() - 1)
    table.copy_(torch.where(fresh, st["free_pages"][at], table))
    row = torch.arange(R, device=DEV)
    seq = torch.searchsorted(starts, row, right=True) - 1
    i = row - starts[seq]
    slot = length[seq] + i
    pg = table[seq, (slot // page).clamp(max=width - 1)].long()
    mapped = i < n[seq]
    row_slots = torch.where(mapped & (pg >= 0), pg * page + slot % page, -1)
    row_positions = torch.where(mapped, st["positions"][seq] + 1 + i, -1).to(torch.int32)
    free = free - taken.sum()
    return (starts.to(torch.int32), n.to(torch.int32), (length + n).to(torch.int32),
            (st["positions"] + n).to(torch.int32), free.to(torch.int32), row_slots, row_positions, table)


def _plain_truncate(st, case):
    page, table, pool = case["page"], st["block_table"], st["free_pages"]
    width = table.shape[1]
    length = st["lengths"].long()
    new = torch.minimum(length, st["to"].long().clamp(min=0))
    have, keep = (length + page - 1) // page, (new + page - 1) // page
    gone = have - keep
    upto = torch.cumsum(gone, 0)
    free = st["free_count"].long()
    nth = torch.arange(width, device=DEV) - keep.unsqueeze(1)
    back = (nth >= 0) & (nth < gone.unsqueeze(1))
    at = free + upto[-1] - 1 - ((upto - gone).unsqueeze(1) + nth)
    # (One place behind the list for the entries that stay.)
    longer = torch.cat([pool, pool[:1]])
    longer[torch.where(back, at, pool.numel())] = table
    pool.copy_(longer[:-1])
    return (new.to(torch.int32), (st["positions"] - (length - new)).to(torch.int32),
            (free + upto[-1]).to(torch.int32), pool)


def _norm_rope(x, w, cs):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    x1, x2 = x.chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _plain_append(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    x = st["qkv"].float().view(-1, nq + 2 * nkv, D)
    cs = st["cos_sin"][st["row_positions"].long()].unsqueeze(1)
    q = _norm_rope(x[:, :nq], st["q_norm"], cs).to(torch.bfloat16)
    k = _norm_rope(x[:, nq:nq + nkv], st["k_norm"], cs)
    pg, row = st["row_slots"] // case["page"], st["row_slots"] % case["page"]
    st["k_pages"][pg, :, row] = k.to(torch.bfloat16)
    st["v_pages"][pg, :, row] = x[:, nq + nkv:].to(torch.bfloat16)
    return q, st["k_pages"], st["v_pages"]


def _plain_attend(st, case):
    table, starts, counts = st["block_table"].long(), st["starts"].long(), st["counts"].long()
    R, nq, D = st["q"].shape
    nkv, page = st["k_pages"].shape[1:3]
    B, cap, most, G = table.shape[0], table.shape[1] * page, st["most"], nq // nkv
    # A padded batch [B, nkv, most * G, D] of the rows.
    i = torch.arange(most, device=DEV)
    q = st["q"][(starts.unsqueeze(1) + i).clamp(max=R - 1)].float()
    q = q.view(B, most, nkv, G, D).transpose(1, 2).reshape(B, nkv, most * G, D)
    k = st["k_pages"][table].transpose(1, 2).reshape(B, nkv, cap, D).float()
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5)
    del k
    last = (st["lengths"].long() - counts).unsqueeze(1) + i
    seen = torch.arange(cap, device=DEV) <= last.unsqueeze(-1)
    s.view(B, nkv, most, G, cap).masked_fill_(~seen.view(B, 1, most, 1, cap), -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    v = st["v_pages"][table].transpose(1, 2).reshape(B, nkv, cap, D).float()
    o = torch.matmul(s, v).div_(total)
    del s, v
    o = o.view(B, nkv, most, G, D).transpose(1, 2).reshape(B, most, nq * D)
    row = torch.arange(R, device=DEV)
    seq = torch.searchsorted(starts, row, right=True) - 1
    at = row - starts[seq]
    o = o[seq, at.clamp(max=most - 1)]
    return o.masked_fill((at >= counts[seq]).unsqueeze(1), 0.0).to(torch.bfloat16)


_PLAIN = {"reserve": _plain_reserve, "truncate": _plain_truncate, "append": _plain_append, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, B, page = case["kind"], case["B"], case["page"]
    old = _before(case)
    if kind == "truncate":
        mean = case["drop"] if case["drop"] >= case["old"] else case["drop"] // 2
        pages = sum(_pages(n, page) - _pages(max(0, n - mean), page) for b, n in enumerate(old) if b % case["every"] == 0)
        return {"bytes": 20 * B + 8 + 8 * pages, "flops": 0}
    counts, R = _counts(case), _rows(case)
    pages = sum(_pages(n + c, page) - _pages(n, page) for n, c in zip(old, counts))
    if kind == "reserve":
        return {"bytes": 28 * B + 8 + 12 * R + 8 * pages, "flops": 0}
    nq, nkv, D = HEADS[case["preset"]]
    if kind == "append":
        values = (nq + 2 * nkv) * D
        longest = max(n + c for n, c in zip(old, counts))
        return {"bytes": R * (4 * values + 12) + 4 * D * min(R, longest), "flops": 10 * R * values}
    tokens = sum(n + c for n, c in zip(old, counts))
    pairs = sum(c * n + c * (c + 1) // 2 for n, c in zip(old, counts))
    table = 4 * sum(_pages(n + c, page) for n, c in zip(old, counts)) + 12 * B
    return {"bytes": 4 * nkv * D * tokens + 2 * nq * D * (sum(counts) + R) + table, "flops": 4 * nq * D * pairs}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"reserve": _exact_reserve, "truncate": _exact_truncate, "append": _exact_append,
            "attend": _exact_attend}[case["kind"]](st, case)


def _exact_reserve(st, case):
    page, R = case["page"], _rows(case)
    table, pool = st["block_table"].cpu().numpy(), st["free_pages"].cpu().numpy()
    B, width = table.shape
    length, pos = st["lengths"].tolist(), st["positions"].tolist()
    free = int(st["free_count"])
    asked = 0
    starts, granted, new_len, new_pos, gone = [], [], [], [], 0
    slots, where_to = np.full(R, -1, np.int64), np.full(R, -1, np.int32)
    at = 0
    for b, n in enumerate(st["counts"].tolist()):
        first = b * case["new"] if case["padded"] else at
        at += n
        starts.append(first)
        have = _pages(length[b], page)
        need = _pages(length[b] + n, page) - have
        if first + n > R or length[b] + n > width * page or (case["padded"] and n > case["new"]):
            n = need = 0
        before, asked = asked, asked + need
        if need and asked > free:
            n = need = 0
        for j in range(need):
            table[b, have + j] = pool[free - 1 - before - j]
        gone += need
        slot = length[b] + np.arange(n)
        slots[first:first + n] = table[b, slot // page].astype(np.int64) * page + slot % page
        where_to[first:first + n] = pos[b] + 1 + np.arange(n)
        granted.append(n)
        new_len.append(length[b] + n)
        new_pos.append(pos[b] + n)
    small = [np.array(x, np.int32) for x in (starts, granted, new_len, new_pos, [free - gone])]
    return (*small, slots, where_to, table)


def _exact_truncate(st, case):
    page = case["page"]
    table, pool = st["block_table"].cpu().numpy(), st["free_pages"].cpu().numpy()
    length, to, pos = st["lengths"].tolist(), st["to"].tolist(), st["positions"].tolist()
    free = int(st["free_count"])
    new = [min(n, t) for n, t in zip(length, to)]
    back = [table[b, _pages(m, page):_pages(n, page)] for b, (n, m) in enumerate(zip(length, new))]
    back = np.concatenate(back)[::-1]
    pool[free:free + len(back)] = back
    small = [np.array(x, np.int32) for x in (new, [p - n + m for p, n, m in zip(pos, length, new)], [free + len(back)])]
    return (*small, pool)


def _exact_append(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    x = st["qkv"].double().reshape(-1, nq + 2 * nkv, D)
    pos = st["row_positions"].long()
    cos, sin = st["cos_sin"].double()[pos, :, 0], st["cos_sin"].double()[pos, :, 1]

    def head(i, w):
        y = x[:, i]
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * w.double()
        a, b = y[:, :D // 2], y[:, D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], 1)

    q = torch.stack([head(i, st["q_norm"]) for i in range(nq)], 1)
    page = case["page"]
    k, v = st["k_pages"].double(), st["v_pages"].double()
    for h in range(nkv):
        k[st["row_slots"] // page, h, st["row_slots"] % page] = head(nq + h, st["k_norm"])
        v[st["row_slots"] // page, h, st["row_slots"] % page] = x[:, nq + nkv + h]
    return q, k, v


def _exact_attend(st, case):
    nq, nkv, D = HEADS[case["preset"]]
    page, G = case["page"], nq // nkv
    out = torch.zeros(_rows(case), nq, D, dtype=torch.float64, device=DEV)
    for b, (first, c, old) in enumerate(zip(_starts(case), _counts(case), _before(case))):
        used = st["block_table"][b, :_pages(old + c, page)].long()
        hidden = torch.arange(old + c, device=DEV) > old + torch.arange(c, device=DEV).unsqueeze(1)
        for h in range(nkv):
            k = st["k_pages"][used, h].reshape(-1, D)[:old + c].double().t().contiguous()
            v = st["v_pages"][used, h].reshape(-1, D)[:old + c].double()
            for j in range(h * G, h * G + G):
                s = st["q"][first:first + c, j].double() @ k / math.sqrt(D)
                p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
                out[first:first + c, j] = p @ v
    return out.view(-1, nq * D)
