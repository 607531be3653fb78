"""The paged KV cache's operators against plain 64-bit forms (tests/_paged.py): the append of a
step, the write of prompts, attention over the pages, and eviction by accumulated weight."""

from __future__ import annotations

import math

import pytest
import torch

import _paged as ref

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(n, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    return torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()


def _check_attention(out, q, k, v, table, lengths, scale=None):
    want, weights, bound = ref.attention(q, k, v, table, lengths, scale)
    got = out.double().cpu().view(want.shape)
    assert bool((((got - want).abs() <= bound) | (want.isnan() & got.isnan())).all()), \
        f"off by {float(((got - want).abs() / bound.clamp_min(1e-30)).max())} of the bound"
    return weights


# ---- the append ---------------------------------------------------------------

@pytest.mark.parametrize("nq,nkv,D,page,norm,dtype", [
    (16, 8, 128, 64, True, bf16), (12, 4, 64, 16, True, torch.float32), (16, 4, 80, 32, True, bf16),
    (8, 4, 40, 256, True, torch.float32), (4, 2, 64, 128, False, bf16), (3, 1, 8, 16, True, bf16),
    (5, 5, 104, 32, False, torch.float32),
])
def test_append(cdx, nq, nkv, D, page, norm, dtype):
    print(f"append {nq}/{nkv} D={D} page={page} norm={norm} {dtype}", flush=True)
    B, width = 6, 3
    g = torch.Generator().manual_seed(D + nq)
    k, v, table = ref.cache(B, nkv, D, page, width, seed=D)
    k0, v0 = k.clone(), v.clone()
    qkv = torch.randn(B, (nq + 2 * nkv) * D, generator=g).to(dtype)
    wq, wk = ((1 + 0.1 * torch.randn(2, D, generator=g)).to(bf16)) if norm else (None, None)
    # An empty sequence, the first slot, a page's last and first, the last slot, one past it.
    lens = [0, 1, page, page + 1, width * page, width * page + 1]
    pos = [3, 0, page - 1, 9000, width * page - 1, 77]
    cs = _table(9001, D)
    q = cdx.paged_qkv_append(qkv.cuda(), k, v, table, _ints(lens), _ints(pos), nq, cs,
                             wq.cuda() if norm else None, wk.cuda() if norm else None)
    x = qkv.double().view(B, nq + 2 * nkv, D)
    ek, ev = k0.cpu().clone(), v0.cpu().clone()
    for b in range(B):
        def head(i, w):
            y = x[b, i]
            if w is not None:
                y = y * torch.rsqrt(y.square().mean() + 1e-6) * w.double()
            return ref.rope(y, pos[b])

        def close(got, want):
            # One rounding of the result, and fp32 arithmetic (and a table rounded to fp32) on
            # values of the row's size.
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().max()
            assert bool(((got.double().cpu() - want).abs() <= tol).all())

        for i in range(nq):
            close(q[b, i], head(i, wq))
        slot = lens[b] - 1
        if not 0 <= slot < width * page:
            continue
        pg, row = int(table[b, slot // page]), slot % page
        for h in range(nkv):
            close(k[pg, h, row], head(nq + h, wk))
            ek[pg, h, row] = k[pg, h, row].cpu()
            ev[pg, h, row] = x[b, nq + nkv + h].to(bf16)
    assert torch.equal(k.cpu(), ek) and torch.equal(v.cpu(), ev)  # v exactly, and nothing else written


def test_append_unknown_position_and_missing_page(cdx):
    print("append: positions outside the table, pages outside the pool", flush=True)
    B, nq, nkv, D, page = 5, 4, 2, 64, 16
    k, v, table = ref.cache(B, nkv, D, page, 2)
    k0, v0 = k.clone(), v.clone()
    table[2, 0], table[3, 0] = -1, k.shape[0]
    qkv = torch.randn(B, (nq + 2 * nkv) * D, device="cuda").to(bf16)
    q = cdx.paged_qkv_append(qkv, k, v, table, _ints([1, 1, 1, 1, 1]), _ints([-1, 10, 0, 0, 9]), nq, _table(10, D))
    nan = q.isnan().all(-1).all(-1).cpu().tolist()
    assert nan == [True, True, False, False, False] and not q[2:].isnan().any()
    for b in (0, 1):  # k cannot be rotated, v needs no angle
        assert bool(k[int(table[b, 0]), :, 0].isnan().all())
        assert torch.equal(v[int(table[b, 0]), :, 0], qkv.view(B, -1, D)[b, nq + nkv:])
    changed = {int(table[b, 0]) for b in (0, 1, 4)}
    rest = [i for i in range(k.shape[0]) if i not in changed]
    assert torch.equal(k[rest], k0[rest]) and torch.equal(v[rest], v0[rest])


def test_append_takes_strided_rows_and_tables(cdx):
    print("append: strided operands", flush=True)
    B, nq, nkv, D, page = 4, 4, 2, 64, 16
    k, v, table = ref.cache(B, nkv, D, page, 2)
    wide = torch.randn(B, 3 * (nq + 2 * nkv) * D + 8, device="cuda").to(bf16)
    qkv = wide[:, 8:8 + (nq + 2 * nkv) * D]
    odd = wide[:, 3:3 + (nq + 2 * nkv) * D]
    tables = torch.full((B, 7), -1, dtype=torch.int32, device="cuda")
    tables[:, 2:4] = table
    lens, cs = _ints([1, 5, 17, 32]), _table(40, D)
    both = torch.stack([lens, lens - 1], 1)  # strided lengths and positions
    for x in (qkv, odd):
        k1, v1, k2, v2 = k.clone(), v.clone(), k.clone(), v.clone()
        a = cdx.paged_qkv_append(x.contiguous(), k1, v1, table, lens, lens - 1, nq, cs)
        b = cdx.paged_qkv_append(x, k2, v2, tables[:, 2:4], both[:, 0], both[:, 1], nq, cs)
        assert torch.equal(a, b) and torch.equal(k1, k2) and torch.equal(v1, v2)


# ---- prompts ------------------------------------------------------------------

@pytest.mark.parametrize("nkv,D,page,S", [(8, 128, 64, 200), (4, 80, 16, 77), (2, 64, 32, 1), (3, 40, 256, 300),
                                          (1, 8, 128, 513)])
def test_write(cdx, nkv, D, page, S):
    print(f"write nkv={nkv} D={D} page={page} S={S}", flush=True)
    lens = [S, 0, (S + 1) // 2, -3, S + 5, 1]
    B, width = len(lens), -(-S // page)
    k, v, table = ref.cache(B, nkv, D, page, width, seed=S)
    table[3] = -1  # an empty sequence needs no pages
    ek, ev = k.cpu().clone(), v.cpu().clone()
    nk, nv = (torch.randn(B, nkv, S, D, device="cuda").to(bf16) for _ in range(2))
    cdx.paged_write(nk, nv, k, v, table, _ints(lens))
    for b, n in enumerate(lens):
        for t in range(max(0, min(n, S))):
            ek[int(table[b, t // page]), :, t % page] = nk[b, :, t].cpu()
            ev[int(table[b, t // page]), :, t % page] = nv[b, :, t].cpu()
    assert torch.equal(k.cpu(), ek) and torch.equal(v.cpu(), ev)


def test_write_past_the_capacity_and_missing_pages(cdx):
    print("write: longer than the table, pages outside the pool", flush=True)
    B, nkv, D, page, S = 3, 2, 64, 16, 50
    k, v, table = ref.cache(B, nkv, D, page, 2)
    table[1, 1], table[2, 0] = k.shape[0] + 5, -7
    ek, ev = k.cpu().clone(), v.cpu().clone()
    nk, nv = (torch.randn(B, S, nkv, D, device="cuda").to(bf16).transpose(1, 2) for _ in range(2))
    cdx.paged_write(nk, nv, k, v, table, _ints([S, S, S]))
    for b in range(B):
        for t in range(2 * page):
            pg = int(table[b, t // page])
            if 0 <= pg < k.shape[0]:
                ek[pg, :, t % page], ev[pg, :, t % page] = nk[b, :, t].cpu(), nv[b, :, t].cpu()
    assert torch.equal(k.cpu(), ek) and torch.equal(v.cpu(), ev)


# ---- attention ----------------------------------------------------------------

@pytest.mark.parametrize("nq,nkv,D,page,lens", [
    (16, 8, 128, 64, [1, 31, 32, 33, 64, 65, 700]), (12, 4, 64, 16, [1, 15, 16, 17, 47, 128, 129, 130]),
    (16, 4, 80, 32, [500, 3, 97]), (8, 4, 40, 256, [1, 300, 511]), (4, 4, 32, 128, [90, 1000]),
    (32, 2, 96, 16, [33, 200]), (34, 2, 104, 64, [5, 260]), (40, 1, 128, 16, [77]), (6, 2, 8, 16, [1, 2, 50]),
    (2, 2, 24, 32, [0, 40, 0]), (16, 8, 128, 128, [5000]), (3, 1, 120, 16, [4099, 2]), (16, 1, 56, 64, [129]),
    # many short sequences, some empty, beside a long one
    (4, 2, 64, 16, [0, 700, 0, 1, 2, 3, 900, 0] + [33 * (i % 7) for i in range(90)] + [0]),
    (2, 1, 32, 16, [i % 40 for i in range(1030)]), (2, 1, 16, 32, [i % 70 for i in range(300)]),
    (4, 2, 128, 256, [20000, 1, 0, 257]), (2, 2, 64, 16, [9000]),  # many splits
])
def test_attention(cdx, nq, nkv, D, page, lens):
    print(f"attention {nq}/{nkv} D={D} page={page} lengths={lens}", flush=True)
    B, width = len(lens), -(-max(lens) // page) + 1
    g = torch.Generator().manual_seed(D + page)
    k, v, table = ref.cache(B, nkv, D, page, width, seed=nq)
    q = (1.5 * torch.randn(B, nq, D, generator=g)).to(bf16).cuda()
    lengths = _ints(lens)
    out = cdx.paged_attention(q, k, v, table, lengths)
    weights = _check_attention(out, q, k, v, table, lengths)
    # With the weights: the same output, and what each slot received added to what was there.
    w0 = torch.rand(B, nkv, width * page, generator=g).cuda()
    again, w1 = cdx.paged_attention(q, k, v, table, lengths, weights=w0)
    assert torch.equal(again, out) and w1 is not w0
    want = w0.double().cpu() + weights
    # p in fp32: (D + 8) 2^-24 of scores of at most ~50, twice, and the sums' roundings.
    tol = weights * (2 * (D + 8) * 50 * 2.0 ** -24 + 2.0 ** -18) + 2.0 ** -22 * want.abs()
    assert bool(((w1.double().cpu() - want).abs() <= tol).all())
    for b, n in enumerate(lens):
        assert torch.equal(w1[b, :, n:], w0[b, :, n:])
    inplace = w0.clone()
    cdx.paged_attention(q, k, v, table, lengths, weights=inplace, weights_out=inplace)
    assert torch.equal(inplace, w1)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3e38])
def test_attention_ignores_what_lies_behind_a_sequence(cdx, value):
    print(f"attention: {value} behind the lengths", flush=True)
    nq, nkv, D, page = 8, 2, 64, 16
    lens = [0, 1, 15, 16, 17, 33, 48, -2]
    B, width = len(lens), 4
    k, v, table = ref.cache(B, nkv, D, page, width)
    q = torch.randn(B, nq, D, device="cuda").to(bf16)
    clean = cdx.paged_attention(q, k, v, table, _ints(lens))
    assert bool((clean[0] == 0).all()) and bool((clean[7] == 0).all())
    for b, n in enumerate(lens):
        for t in range(max(n, 0), width * page):
            k[int(table[b, t // page]), :, t % page] = value
            v[int(table[b, t // page]), :, t % page] = value
        used = -(-max(n, 0) // page)
        table[b, used:] = torch.tensor([-1, 10 ** 9, 5, -2 ** 31])[:width - used].int()
    assert torch.equal(cdx.paged_attention(q, k, v, table, _ints(lens)), clean)
    _check_attention(clean, q, k, v, table.clamp(0, k.shape[0] - 1), _ints(lens))


def test_attention_over_a_missing_page_is_nan(cdx):
    print("attention: pages outside the pool", flush=True)
    k, v, table = ref.cache(4, 2, 64, 16, 3)
    q = torch.randn(4, 4, 64, device="cuda").to(bf16)
    table[1, 1], table[2, 0], table[3, 2] = -1, k.shape[0], 2 ** 31 - 1
    out = cdx.paged_attention(q, k, v, table, _ints([40, 40, 1, 32]))
    assert out.isnan().all(-1).cpu().tolist() == [False, True, True, False]
    assert not out[0].isnan().any() and not out[3].isnan().any()


def test_attention_scores_of_minus_infinity(cdx):
    """Scores of -inf weigh nothing beside a finite one (also when they come first, and when a
    whole tile or split has no other), and alone give NaN, as softmax does."""
    print("attention: infinite scores", flush=True)
    nq, nkv, D, page, n = 4, 2, 64, 32, 700
    k, v, table = ref.cache(4, nkv, D, page, 22)
    q = torch.ones(4, nq, D, device="cuda").to(bf16)
    for b, hidden in enumerate((range(0, 1), range(0, 699), range(0, 700), range(300, 301))):
        for t in hidden:
            k[int(table[b, t // page]), :, t % page, 5] = math.inf if b == 3 else -math.inf
    lengths = _ints([n] * 4)
    out = cdx.paged_attention(q, k, v, table, lengths)
    assert out.isnan().all(-1).cpu().tolist() == [False, False, True, True]
    _check_attention(out[:2], q[:2], k, v, table[:2], lengths[:2])
    _, w = cdx.paged_attention(q, k, v, table, lengths, weights=torch.zeros(4, nkv, 704, device="cuda"))
    assert bool((w[1, :, :699] == 0).all()) and bool((w[1, :, 699] == 2).all())


def test_attention_large_scores_and_scale(cdx):
    print("attention: scores of thousands, a scale of its own", flush=True)
    k, v, table = ref.cache(2, 2, 128, 64, 5)
    q = (100 * torch.randn(2, 4, 128, device="cuda")).to(bf16)
    lengths = _ints([300, 64])
    for scale in (None, 1.0, 1e-3):
        _check_attention(cdx.paged_attention(q, k, v, table, lengths, scale), q, k, v, table, lengths, scale)


def test_attention_of_one_row_does_not_depend_on_the_others(cdx):
    print("attention: rows on their own, strided operands, length past the capacity", flush=True)
    nq, nkv, D, page, width = 16, 8, 128, 32, 9
    k, v, table = ref.cache(3, nkv, D, page, width)
    wide = torch.randn(3, nq + 1, 2 * D, device="cuda").to(bf16)
    q = wide[:, 1:, 4:4 + D]  # strided, and not on 16 bytes
    lens = _ints([10 ** 9, 100, 288])
    out = cdx.paged_attention(q, k, v, table, lens)
    assert torch.equal(out, cdx.paged_attention(q.contiguous(), k, v, table, _ints([288, 100, 288])))
    _check_attention(out, q, k, v, table, lens)
    big = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    big[:, 1:1 + width] = table
    assert torch.equal(cdx.paged_attention(q, k, v, big[:, 1:1 + width], lens), out)
    # Two sequences that share their pages (a common prefix).
    shared = table[[0, 0, 0]].clone()
    assert torch.equal(cdx.paged_attention(q[[1, 1, 1]], k, v, shared, lens[[1, 1, 1]])[0],
                       cdx.paged_attention(q[[1, 1, 1]], k, v, shared, lens[[1, 1, 1]])[2])


def test_attention_past_32_bits(cdx):
    """A pool of more than 4 GB (and 2^31 values): pages at its end."""
    print("paged: a pool of 5 GB", flush=True)
    nq, nkv, D, page = 4, 2, 128, 256
    pages = 5 * 2 ** 30 // (nkv * page * D * 2)
    k = torch.zeros(pages, nkv, page, D, dtype=bf16, device="cuda")
    v = torch.zeros_like(k)
    small_k, small_v, _ = ref.cache(1, nkv, D, page, 3, spare=0)
    at = [pages - 1, 0, pages - 2]
    k[at], v[at] = small_k, small_v
    table = _ints([at])
    q = torch.randn(1, nq, D, device="cuda").to(bf16)
    out = cdx.paged_attention(q, k, v, table, _ints([700]))
    assert torch.equal(out, cdx.paged_attention(q, small_k, small_v, _ints([[0, 1, 2]]), _ints([700])))
    nk = torch.randn(1, nkv, 600, D, device="cuda").to(bf16)
    cdx.paged_write(nk, nk, k, v, table, _ints([600]))
    assert torch.equal(ref.slots(k, table, 0, 600), nk[0]) and torch.equal(ref.slots(v, table, 0, 600), nk[0])
    qkv = torch.randn(1, (nq + 2 * nkv) * D, device="cuda").to(bf16)
    cdx.paged_qkv_append(qkv, k, v, table, _ints([768]), _ints([0]), nq, _table(1, D))
    assert torch.equal(v[pages - 2, :, 255], qkv.view(-1, D)[nq + nkv:])


# ---- eviction -----------------------------------------------------------------

def _tracked(L, B, nkv, cap, lens, seed, kind="random"):
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(L, B, nkv, cap, generator=g).pow(4)
    if kind == "ties":
        w = torch.randint(0, 3, (L, B, nkv, cap), generator=g).float()
    if kind == "odd":
        pool = torch.tensor([0.0, -0.0, math.nan, math.inf, -math.inf, 1.0, -1.0, 1e-45, 3e38])
        w = pool[torch.randint(0, len(pool), (L, B, nkv, cap), generator=g)]
    pos = torch.argsort(torch.rand(L, B, nkv, cap, generator=g), -1)
    for b, n in enumerate(lens):  # a permutation of 0 .. n - 1 over the slots in use
        n = max(0, min(n, cap))
        pos[:, b] = torch.argsort(torch.argsort(torch.where(torch.arange(cap) < n, pos[:, b], pos[:, b] + cap)))
    return w, pos.to(torch.int32)


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("L,nkv,D,page,lens,keep,recent", [
    (2, 2, 64, 16, [40, 41, 39, 0, -1, 48, 1], 40, 8), (None, 4, 40, 32, [33, 2, 64], 1, 0),
    (None, 1, 128, 64, [1, 2], 1, 1), (3, 2, 8, 16, [600, 700, 1300], 600, 600), (1, 3, 80, 32, [1000, 999], 100, 99),
    (None, 2, 64, 256, [256, 200], 256, 3),
    (None, 2, 8, 64, [2048, 2000, 1999], 1999, 100), (None, 1, 8, 256, [5000, 8192], 3000, 10),
    (None, 1, 8, 128, [9000, 8200], 4500, 4000),
])
def test_evict(cdx, L, nkv, D, page, lens, keep, recent, kind):
    print(f"evict layers={L} nkv={nkv} D={D} page={page} lengths={lens} keep={keep} recent={recent} {kind}", flush=True)
    B, width, layers = len(lens), -(-max(lens) // page), L or 1
    cap = width * page
    k, v, table = ref.cache(B, nkv, D, page, width, layers=L, seed=keep)
    w, pos = _tracked(layers, B, nkv, cap, lens, keep + recent, kind)
    last = [max(0, min(n, cap)) - 1 for n in lens]
    want_len, want_w, want_p, moves = ref.evict(lens, last, w, pos, keep, recent)
    ek, ev = k.cpu().view(layers, *k.shape[-4:]).clone(), v.cpu().view(layers, *v.shape[-4:]).clone()
    t = table.cpu()
    for (l, b, h), i, j in moves:
        for e in (ek, ev):
            e[l, t[b, i // page], h, i % page] = e[l, t[b, j // page], h, j % page]
    dw, dp = (x.cuda() if L else x[0].cuda() for x in (w, pos))
    w0, p0 = dw.clone(), dp.clone()
    n, nw, np_ = cdx.paged_evict(k, v, table, _ints(lens), _ints(last), dw, dp, keep, recent)
    assert n.tolist() == want_len
    assert torch.equal(np_.cpu().view_as(want_p), want_p)
    assert torch.equal(nw.cpu().view_as(want_w).nan_to_num(nan=-7.0), want_w.nan_to_num(nan=-7.0))
    assert torch.equal(k.cpu().view_as(ek), ek) and torch.equal(v.cpu().view_as(ev), ev)
    assert torch.equal(dw.nan_to_num(nan=-7.0), w0.nan_to_num(nan=-7.0)) and torch.equal(dp, p0)


def test_evict_positions_given_twice(cdx):
    """More recent slots than `keep`: the largest weights among them stay."""
    print("evict: every slot recent", flush=True)
    k, v, table = ref.cache(1, 2, 64, 16, 4)
    w, pos = _tracked(1, 1, 2, 64, [64], 3)
    pos.fill_(63)
    want_len, want_w, want_p, _ = ref.evict([64], [63], w, pos, 20, 5)
    n, nw, np_ = cdx.paged_evict(k, v, table, _ints([64]), _ints([63]), w[0].cuda(), pos[0].cuda(), 20, 5)
    assert n.tolist() == want_len and torch.equal(nw.cpu(), want_w[0]) and torch.equal(np_.cpu(), want_p[0])


def test_evict_with_missing_pages(cdx):
    print("evict: pages outside the pool", flush=True)
    k, v, table = ref.cache(1, 1, 64, 16, 4)
    k0, v0 = k.clone(), v.clone()
    table[0, 0], table[0, 3] = -1, k.shape[0]  # holes 0 .. 15 and movers 48 .. 63 cannot move
    w = torch.arange(64, device="cuda").float().view(1, 1, 64)  # the last 20 stay
    pos = torch.arange(64, device="cuda").int().view(1, 1, 64)
    n, nw, _ = cdx.paged_evict(k, v, table, _ints([64]), _ints([63]), w, pos, 20, 0)
    assert n.tolist() == [20] and nw[0, 0, :20].tolist() == list(range(44, 64))
    changed = {int(table[0, 1])}
    rest = [i for i in range(k.shape[0]) if i not in changed]
    assert torch.equal(k[rest], k0[rest]) and torch.equal(v[rest], v0[rest])


# ---- together -----------------------------------------------------------------

def test_a_bounded_generation_of_one_layer(cdx):
    """Prompts, then steps that append, attend with weights and evict, against the same in 64 bits
    on plain lists; then the captured step, replayed."""
    print("paged: prompt, append, attend, evict", flush=True)
    B, nq, nkv, D, page, width, keep, recent = 3, 8, 4, 64, 16, 3, 40, 8
    g = torch.Generator().manual_seed(7)
    k, v, table = ref.cache(B, nkv, D, page, width, fill=float("nan"))
    cap, prompt = width * page, [40, 17, 1]
    lengths, positions = _ints(prompt), _ints(prompt) - 1
    nk, nv = (torch.randn(B, nkv, 40, D, generator=g).to(bf16).cuda() for _ in range(2))
    cdx.paged_write(nk, nv, k, v, table, lengths)
    weights = torch.zeros(B, nkv, cap, device="cuda")
    at = torch.arange(cap, device="cuda", dtype=torch.int32)
    slot_pos = torch.where(at < lengths.view(B, 1, 1), at, -1).expand(B, nkv, cap).contiguous()
    cs = _table(200, D)
    qkv = torch.empty(B, (nq + 2 * nkv) * D, dtype=bf16, device="cuda")
    w_q = (1 + 0.1 * torch.randn(D, generator=g)).to(bf16).cuda()

    def step():
        lengths.add_(1), positions.add_(1)
        slot = (lengths.long() - 1).view(B, 1, 1).expand(B, nkv, 1)
        slot_pos.scatter_(-1, slot, positions.view(B, 1, 1).expand(B, nkv, 1))
        q = cdx.paged_qkv_append(qkv, k, v, table, lengths, positions, nq, cs, w_q, w_q)
        out, _ = cdx.paged_attention(q, k, v, table, lengths, weights=weights, weights_out=weights)
        n, w, p = cdx.paged_evict(k, v, table, lengths, positions, weights, slot_pos, keep, recent)
        lengths.copy_(n), weights.copy_(w), slot_pos.copy_(p)
        return q, out

    def check(q, out, before):
        """The step's output from the cache as it was, and the cache as it has to be now."""
        lens, pos = [n + 1 for n in before["len"]], [p + 1 for p in before["pos"]]
        rk, rv = before["k"], before["v"]
        x = qkv.view(B, -1, D)
        for b in range(B):
            pg, row = int(table[b, (lens[b] - 1) // page]), (lens[b] - 1) % page
            want = x[b, nq:nq + nkv].double().cpu()
            want = want * torch.rsqrt(want.square().mean(-1, keepdim=True) + 1e-6) * w_q.double().cpu()
            got = torch.stack([ref.rope(want[h], pos[b]) for h in range(nkv)])
            rk[pg, :, row], rv[pg, :, row] = got.to(bf16).cuda(), x[b, nq + nkv:]
        added = _check_attention(out, q, rk, rv, table, _ints(lens))
        w, p = before["w"].double().cpu() + added, before["sp"].cpu().clone()
        for b in range(B):
            p[b, :, lens[b] - 1] = pos[b]
        # (The eviction's choice is checked on the weights that the kernel summed: test_evict.)
        assert lengths.tolist() == [min(n, keep) for n in lens] and positions.tolist() == pos
        for b in range(B):
            n = min(lens[b], keep)
            for h in range(nkv):
                held = slot_pos[b, h, :n].tolist()
                assert len(set(held)) == n and set(range(pos[b] - recent + 1, pos[b] + 1)) & set(range(pos[b] + 1)) <= \
                    set(held)
                back = {int(s): i for i, s in enumerate(p[b, h].tolist()) if s >= 0}
                for i in (0, n // 2, n - 1):  # rows, weights and positions moved together
                    j = back[held[i]]
                    assert torch.allclose(weights[b, h, i].double().cpu(), w[b, h, j], rtol=1e-4, atol=1e-7)
                    assert torch.equal(ref.slots(k, table, b, n)[h, i], k_row(rk, b, h, j, got=k, i=i))

    def k_row(pages, b, h, j, got, i):
        row = ref.slots(pages, table, b, j + 1)[h, j]
        mine = ref.slots(got, table, b, i + 1)[h, i]
        # the appended row within a rounding, any other bit for bit
        return mine if bool(((row.float() - mine.float()).abs() <= 2.0 ** -7 * row.float().abs() + 1e-6).all()) else row

    def state():
        return {"len": lengths.tolist(), "pos": positions.tolist(), "k": k.clone(), "v": v.clone(),
                "w": weights.clone(), "sp": slot_pos.clone()}

    for _ in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        before = state()
        check(*step(), before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the same on a stream of its own
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        before = state()
        q, out = step()
    torch.cuda.current_stream().wait_stream(side)
    check(q, out, before)
    graph = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in (lengths, positions, k, v, weights, slot_pos)]
    with torch.cuda.graph(graph):
        q, out = step()
    for t, s in zip((lengths, positions, k, v, weights, slot_pos), saved):
        t.copy_(s)
    for i in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        before = state()
        graph.replay()
        torch.cuda.synchronize()
        check(q, out, before)


# ---- refusals -----------------------------------------------------------------

def test_refusals(cdx):
    print("paged: refused calls", flush=True)
    B, nq, nkv, D, page = 2, 4, 2, 64, 16
    k, v, table = ref.cache(B, nkv, D, page, 2)
    lens, cs = _ints([3, 4]), _table(40, D)
    qkv = torch.randn(B, (nq + 2 * nkv) * D, device="cuda").to(bf16)
    q = torch.randn(B, nq, D, device="cuda").to(bf16)
    w = torch.zeros(B, nkv, 32, device="cuda")
    sp = torch.zeros(B, nkv, 32, device="cuda").int()
    new = torch.randn(B, nkv, 20, D, device="cuda").to(bf16)
    paged = dict(k_pages=k, v_pages=v, block_table=table, lengths=lens)

    def append(**a):
        cdx.paged_qkv_append(**{**paged, **dict(qkv=qkv, positions=lens, num_heads=nq, cos_sin=cs), **a})

    def attend(**a):
        cdx.paged_attention(**{**paged, **dict(q=q), **a})

    def write(**a):
        cdx.paged_write(**{**paged, **dict(k=new, v=new), **a})

    def evict(**a):
        cdx.paged_evict(**{**paged, **dict(positions=lens, weights=w, slot_positions=sp, keep=2, recent=1), **a})

    bad = [
        (append, dict(qkv=qkv[:, :-8])), (append, dict(qkv=qkv.half())), (append, dict(num_heads=3)),
        (append, dict(num_heads=0)), (append, dict(lengths=lens.long())), (append, dict(positions=lens[:1])),
        (append, dict(cos_sin=cs.double())), (append, dict(cos_sin=cs[:, :16])), (append, dict(q_norm_w=qkv[0, :D])),
        (append, dict(q_norm_w=qkv[0, :8], k_norm_w=qkv[0, :8])), (append, dict(eps=-1.0)),
        (append, dict(k_pages=k.transpose(1, 2))), (append, dict(v_pages=v[:1])),
        (append, dict(block_table=table.long())),
        (append, dict(qkv=qkv.cpu())), (append, dict(lengths=lens.cpu())),
        (write, dict(k=new[:, :1])), (write, dict(v=new[:, :, :3])), (write, dict(k=new.float())),
        (write, dict(lengths=lens.float())), (write, dict(block_table=table[:1])),
        (attend, dict(q=q[:, :3])), (attend, dict(q=q.float())), (attend, dict(q=q[:1])), (attend, dict(scale=0.0)),
        (attend, dict(scale=float("nan"))), (attend, dict(scale=float("inf"))), (attend, dict(weights=w[..., :31])),
        (attend, dict(weights=w.double())), (attend, dict(weights_out=w)), (attend, dict(block_table=table[:, :0])),
        (attend, dict(weights=w, weights_out=w.transpose(0, 1).contiguous().transpose(0, 1))),
        (attend, dict(k_pages=k[..., :8, :], v_pages=v[..., :8, :])),
        (attend, dict(k_pages=k.float(), v_pages=v.float())),
        (evict, dict(keep=0)), (evict, dict(keep=2, recent=3)), (evict, dict(recent=-1)), (evict, dict(keep=1.5)),
        (evict, dict(weights=w.half())), (evict, dict(slot_positions=sp.long())), (evict, dict(slot_positions=sp[:1])),
        (evict, dict(positions=lens.cpu())), (evict, dict(weights=w[None])),
    ]
    before = [t.clone() for t in (k, v, w, sp)]
    for call, args in bad:
        with pytest.raises((ValueError, RuntimeError)):
            call(**args)
    for t, b in zip((k, v, w, sp), before):
        assert torch.equal(t, b)
    with pytest.raises(NotImplementedError, match="forward-only"):
        attend(q=q.clone().requires_grad_())
    with torch.no_grad():
        attend(q=q.clone().requires_grad_())


# ---- values and sizes at the ends of their ranges --------------------------------

@pytest.mark.parametrize("nq,nkv,D,page,lens", [(4, 2, 64, 16, [1, 2, 40, 700]), (16, 8, 128, 64, [1, 33, 5000]),
                                                (8, 4, 40, 32, [1, 64, 300]), (16, 4, 80, 16, [3, 100])])
def test_attention_over_infinite_values(cdx, nq, nkv, D, page, lens):
    """An infinite value that has a weight makes its column infinite (both signs, or a NaN: NaN) and
    leaves the others as they are."""
    print(f"attention: infinite values, {nq}/{nkv} D={D} lengths={lens}", flush=True)
    k, v, table = ref.cache(len(lens), nkv, D, page, -(-max(lens) // page))
    q = torch.randn(len(lens), nq, D, device="cuda").to(bf16)
    lengths = _ints(lens)
    clean = cdx.paged_attention(q, k, v, table, lengths).view(len(lens), nq, D)
    inf, want = math.inf, {3: math.inf, 5: -math.inf, 6: math.inf, 7: math.nan}
    for at in (0, -1):  # the first slot in use, the last one
        w = v.clone()
        for b, n in enumerate(lens):
            t = at % n
            for col, value in want.items():
                w[int(table[b, t // page]), :, t % page, col] = value
            if n > 1:  # a second one: the sum of two signs has no value
                t = n // 2 if at == 0 else 0
                w[int(table[b, t // page]), :, t % page, 5:7] = torch.tensor([-inf, -inf], device="cuda").to(bf16)
        out = cdx.paged_attention(q, k, w, table, lengths).view(len(lens), nq, D)
        for b, n in enumerate(lens):
            sixth = math.nan if n > 1 else inf
            for col, value in {**want, 6: sixth}.items():
                got = out[b, :, col].float()
                assert bool(got.isnan().all() if math.isnan(value) else (got == value).all()), (b, n, col, got)
        rest = [c for c in range(D) if c not in want]
        assert torch.equal(out[..., rest], clean[..., rest])


def test_attention_repeats_bit_for_bit(cdx):
    """Long sequences over many splits, with other calls between."""
    print("attention: repeated", flush=True)
    k, v, table = ref.cache(4, 8, 128, 128, 65, spare=20)
    g = torch.Generator().manual_seed(2)
    q, other = ((1.5 * torch.randn(4, 16, 128, generator=g)).to(bf16).cuda() for _ in range(2))
    lengths = _ints([8320, 8192, 8191, 4097])
    first = cdx.paged_attention(q, k, v, table, lengths)
    for _ in range(20):
        cdx.paged_attention(other, k, v, table, lengths)
        assert torch.equal(cdx.paged_attention(q, k, v, table, lengths), first)


def test_evict_of_many_heads(cdx):
    """More heads than one launch has threads for."""
    print("evict: 9 x 2^20 heads of 64 slots", flush=True)
    L, B, nkv, D, page, cap, keep = 9, 1 << 17, 8, 8, 64, 64, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.empty(L, B, nkv, page, D, dtype=bf16, device="cuda")
    k.view(torch.int16).random_(0, 1 << 14, generator=g)
    v = k + 1
    table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    lengths = torch.full((B,), cap, dtype=torch.int32, device="cuda")
    # Half of the slots, and always the upper half of every second sequence, weigh more than the others.
    heavy = torch.rand(L, B, nkv, cap, generator=g, device="cuda").argsort(-1) < keep
    heavy[:, ::2] = torch.arange(cap, device="cuda") >= keep
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(L, B, nkv, cap).contiguous()
    k0 = k.clone()
    n, w, p = cdx.paged_evict(k, v, table, lengths, lengths - 1, heavy.float(), pos, keep, 0)
    assert bool((n == keep).all()) and bool((w[..., :keep] == 1).all()) and bool((w[..., keep:] == 0).all())
    assert bool((p[..., keep:] == -1).all())
    held = p[..., :keep].long()
    assert bool(torch.gather(heavy, -1, held).all()) and bool((held.sort(-1).values.diff(dim=-1) > 0).all())
    for l in range(L):  # the rows moved with their positions
        for pages, start in ((k, k0), (v, k0 + 1)):
            want = torch.gather(start[l], 2, held[l].unsqueeze(-1).expand(B, nkv, keep, D))
            assert torch.equal(pages[l, :, :, :keep], want)


def test_append_of_many_sequences(cdx):
    """More heads than one launch has threads for: what two calls of half of them give."""
    print("append: 2^20 sequences of 256 heads", flush=True)
    B, nq, nkv, D, page = 1 << 20, 254, 1, 8, 16
    k = torch.zeros(B, nkv, page, D, dtype=bf16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.empty(B, (nq + 2 * nkv) * D, dtype=bf16, device="cuda").uniform_(-1, 1)
    at = torch.arange(B, dtype=torch.int32, device="cuda")
    table, lengths, positions, cs = at.flip(0).view(B, 1), at % page + 1, at % 40, _table(40, D)
    q = cdx.paged_qkv_append(qkv, k, v, table, lengths, positions, nq, cs)
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    for part in (slice(0, B // 2), slice(B // 2, B)):
        half = cdx.paged_qkv_append(qkv[part], k2, v2, table[part], lengths[part], positions[part], nq, cs)
        assert torch.equal(q[part], half)
    assert torch.equal(k, k2) and torch.equal(v, v2)
