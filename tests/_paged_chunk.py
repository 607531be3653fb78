"""Plain forms of the operators of several new tokens per sequence: pages as lists of integers, attention in
64 bits row by row."""

from __future__ import annotations

import torch

import _paged as ref


def pages(n, page):
    return -(-n // page)


def reserve(counts, lengths, positions, table, page, rows, stride=None, free=None):
    """(starts, counts, lengths, positions, pages left, row slots, row positions, table) of lists; free: the
    list's valid part, or None."""
    table = [list(r) for r in table]
    width = len(table[0])
    slots, where_to = [-1] * rows, [-1] * rows
    out = [[], [], [], []]
    at = asked = gone = 0
    for b, (n, given, pos) in enumerate(zip(counts, lengths, positions)):
        n, have = max(n, 0), max(given, 0)
        first = b * stride if stride else at
        at += n
        fits = first + n <= rows and have + n <= width * page and not (stride and n > stride)
        need = pages(have + n, page) - pages(have, page) if free is not None and fits else 0
        before, asked = asked, asked + need
        if not fits or (need and asked > len(free)):
            n = need = 0
        for j in range(need):
            table[b][pages(have, page) + j] = free[len(free) - 1 - before - j]
        gone += need
        for i in range(n):
            slot = have + i
            p = table[b][slot // page]
            slots[first + i] = p * page + slot % page if p >= 0 else -1
            where_to[first + i] = pos + 1 + i
        for o, x in zip(out, (min(first, rows), n, have + n if n else given, pos + n)):
            o.append(x)
    return (*out, None if free is None else len(free) - gone, slots, where_to, table)


def truncate(to, lengths, positions, table, page, free, room):
    """(lengths, positions, list)."""
    cap = len(table[0]) * page
    new_len, new_pos, back = [], [], []
    for t, n, pos, row in zip(to, lengths, positions, table):
        t = max(t, 0)
        m = min(n, t)
        new_len.append(m)
        new_pos.append(pos - (n - m))
        had = min(max(n, 0), cap)
        back += row[pages(min(had, t), page):pages(had, page)]
    return new_len, new_pos, (list(free) + back[::-1])[:room]


def attention(q, k_pages, v_pages, table, starts, counts, lengths, scale=None, rounded_p=True):
    """(out [rows, nq, D], bound [rows, nq, D]) in 64 bits on q's device: row starts[b] + i attends to the slots
    up to lengths[b] - counts[b] + i; and a bound of a bf16 kernel's error.

    The kernel's scores are fp32 sums of D exact products (each partial sum rounded: D 2^-24 of the sum
    of magnitudes), its sums over slots fp32.  Where few queries share a tile its weights enter the product
    with v as two bf16 parts (2^-16 of a weight is lost); else they are rounded to bf16 (2^-8 of each, in the
    product and in the sum that divides it: ``rounded_p``).  The result is rounded once (2^-8 of it)."""
    rows, nq, D = q.shape
    nkv, page = k_pages.shape[1:3]
    cap = table.shape[1] * page
    out = torch.zeros(rows, nq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    scale = D ** -0.5 if scale is None else scale
    for b, (first, c, n) in enumerate(zip(starts, counts, lengths)):
        last = min(n, cap)
        if c <= 0 or last <= 0:
            continue
        k, v = ref.slots(k_pages, table, b, last).double(), ref.slots(v_pages, table, b, last).double()
        seen = torch.clamp(torch.arange(c, device=q.device) + n - c + 1, 0, cap)
        hidden = torch.arange(last, device=q.device) >= seen.unsqueeze(1)
        some = (seen > 0).unsqueeze(1)
        for h in range(nq):
            g = h // (nq // nkv)
            x = q[first:first + c, h].double()
            s = scale * (x @ k[g].t().contiguous())
            p = torch.softmax(s.masked_fill(hidden, -torch.inf), 1).masked_fill(~some, 0.0)
            size = x.abs() @ k[g].abs().t().contiguous()
            delta = (D + 8) * 2.0 ** -24 * scale * size.masked_fill(hidden, 0.0).amax(1, keepdim=True) + 2.0 ** -19
            # Infinite values and NaN count where they are seen only (0 * NaN is NaN).
            plain = torch.where(v[g].isfinite(), v[g], 0.0)
            o, a = p @ plain, p @ plain.abs()
            for t in (~v[g].isfinite()).any(1).nonzero().flatten().tolist():
                x = torch.where(v[g, t].isfinite(), 0.0, v[g, t])
                o += torch.where(hidden[:, t:t + 1] | (x == 0), 0.0, p[:, t:t + 1] * x)
            out[first:first + c, h] = o
            part = 2.0 ** -8 if rounded_p else 2.0 ** -16
            sums = (last / 32 + 64) * 2.0 ** -23
            bound[first:first + c, h] = (part + 2 * delta + sums) * a + (2.0 ** -8 + (part if rounded_p else 0)) * o.abs()
    return out, bound
