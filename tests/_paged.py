"""Plain 64-bit forms of the paged operators, slot by slot, and the caches the tests use."""

from __future__ import annotations

import math

import torch

bf16 = torch.bfloat16


def cache(B, nkv, D, page, width, layers=None, spare=3, seed=0, device="cuda", fill=None):
    """(k_pages, v_pages, table): a pool with pages in random order; ``fill`` replaces the values."""
    g = torch.Generator().manual_seed(seed)
    pages = B * width + spare
    shape = (() if layers is None else (layers,)) + (pages, nkv, page, D)
    k, v = (torch.randn(shape, generator=g).to(bf16) for _ in range(2))
    if fill is not None:
        k.fill_(fill), v.fill_(fill)
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32)
    return k.to(device), v.to(device), table.to(device)


def slots(pages, table, b, n):
    """Rows [nkv, n, D] of sequence b's first n slots."""
    page = pages.shape[-2]
    used = pages[table[b, :-(-n // page)].long()] if n else pages[:0]
    return used.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[-1])[:, :n]


def rope(x, pos):
    """x [..., D] rotated at one position, in 64 bits."""
    D = x.shape[-1]
    a = pos * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    x1, x2 = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1)


def attention(q, k_pages, v_pages, table, lengths, scale=None):
    """(out [B, nq, D], weights [B, nkv, capacity], bound [B, nq, D]) in 64 bits: the softmax
    attention, what each slot received, and a bound of a bf16 kernel's error.

    The kernel's scores are fp32 sums of D exact products (each partial sum rounded: D 2^-24 of
    the sum of magnitudes); its weights enter the product with v as two bf16 parts (each rounding
    2^-8: 2^-16 of a weight is lost), summed in fp32 over tiles of 32 slots, waves and splits;
    the result is rounded once (2^-8 of it)."""
    q, k_pages, v_pages, table = q.double().cpu(), k_pages.double().cpu(), v_pages.double().cpu(), table.cpu()
    B, nq, D = q.shape
    nkv, page = k_pages.shape[1:3]
    cap = table.shape[1] * page
    out, bound = torch.zeros(B, nq, D, dtype=torch.float64), torch.zeros(B, nq, D, dtype=torch.float64)
    weights = torch.zeros(B, nkv, cap, dtype=torch.float64)
    scale = D ** -0.5 if scale is None else scale
    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), cap)
        if n == 0:
            continue
        k, v = slots(k_pages, table, b, n), slots(v_pages, table, b, n)
        for h in range(nq):
            g = h // (nq // nkv)
            p = torch.softmax(scale * (k[g] @ q[b, h]), 0)
            delta = (D + 8) * 2.0 ** -24 * scale * float((k[g].abs() @ q[b, h].abs()).max()) + 2.0 ** -19
            out[b, h] = p @ v[g]
            weights[b, g, :n] += p
            sums = (n / 32 + 64) * 2.0 ** -23
            bound[b, h] = (2.0 ** -16 + 2 * delta + sums) * (p @ v[g].abs()) + 2.0 ** -8 * out[b, h].abs()
    return out, weights, bound


def evict(lengths, positions, weights, slot_positions, keep, recent):
    """(new lengths, weights, slot positions, moves [(row index, hole, mover)]) by sorting."""
    L, B, nkv, cap = weights.shape
    new_w, new_p = torch.zeros_like(weights), torch.full_like(slot_positions, -1)
    moves, new_len = [], [min(max(int(n), 0), cap, keep) for n in lengths]
    for l in range(L):
        for b in range(B):
            n = min(max(int(lengths[b]), 0), cap)
            for h in range(nkv):
                w, p = weights[l, b, h].tolist(), slot_positions[l, b, h].tolist()

                def rank(i):
                    value = -math.inf if math.isnan(w[i]) else w[i]
                    return (p[i] <= int(positions[b]) - recent, -value, i)

                kept = set(sorted(range(n), key=rank)[:keep])
                holes = [i for i in range(min(n, keep)) if i not in kept] if n > keep else []
                movers = sorted(i for i in kept if i >= keep)
                assert len(holes) == len(movers)
                source = list(range(min(n, keep)))
                for i, j in zip(holes, movers):
                    source[i] = j
                    moves.append(((l, b, h), i, j))
                new_w[l, b, h, :len(source)] = weights[l, b, h, source]
                new_p[l, b, h, :len(source)] = slot_positions[l, b, h, source]
    return new_len, new_w, new_p, moves


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row of logits (any float tensor), by sorting, in 64 bits."""
    x = x.double().cpu().tolist()
    V = len(x)
    x = [-math.inf if math.isnan(v) else v for v in x]
    top = max(x)
    if top == -math.inf:
        return -1
    if not temperature > 0:
        return x.index(top)
    none = {-math.inf} if top < math.inf else set(x) - {top}
    w = [1.0 if v == top else (0.0 if v in none else math.exp((v - top) / temperature)) for v in x]
    order = sorted(range(V), key=lambda i: (-x[i], i))
    if 0 < top_k < V:
        kth = x[order[top_k - 1]]
        w = [a if v >= kth else 0.0 for a, v in zip(w, x)]
    if top_p < 1:
        total, before = math.fsum(w), 0.0
        for i in order:
            a = w[i]
            if before > max(top_p, 0.0) * total:
                w[i] = 0.0
            before += a
    w = [a if a >= min_p or v == top else 0.0 for a, v in zip(w, x)]
    total, run = math.fsum(w), 0.0
    for i in range(V):
        run += w[i]
        if w[i] > 0 and run > u * total:
            return i
    return max(i for i in range(V) if w[i] > 0)
