"""The operators of several new tokens per sequence on a paged cache against plain forms
(tests/_paged_chunk.py): pages from a pool and back, the append of rows, and their attention."""

from __future__ import annotations

import random

import pytest
import torch

import _paged as ref
import _paged_chunk as chunk

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(n, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    return torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()


# ---- pages and rows -----------------------------------------------------------

def _check_reserve(cdx, counts, lengths, positions, table, page, rows, stride=None, free=None, room=None):
    t = _ints(table)
    pool = {}
    if free is not None:
        room = len(free) + 3 if room is None else room
        pool = {"free_pages": _ints((free + [77] * room)[:room]), "free_count": _ints([len(free)])}
        before = pool["free_pages"].clone()
    got = cdx.paged_reserve(_ints(counts), _ints(lengths), _ints(positions), t, page, rows, stride=stride, **pool)
    want = chunk.reserve(counts, lengths, positions, table, page, rows, stride, free)
    for name, g, w in zip(got._fields, got, want):
        w = [w] if name == "free_count" and w is not None else w
        assert (g is None and w is None) or g.tolist() == w, (name, g, w)
    assert got.row_slots.dtype == torch.int64 and t.tolist() == want[-1]
    if pool:
        assert torch.equal(pool["free_pages"], before) and pool["free_count"].tolist() == [len(free)]
    return got


def test_reserve_by_hand(cdx):
    print("reserve: by hand", flush=True)
    # Two sequences that lack a page each, one that lacks none, one without new tokens.
    got = _check_reserve(cdx, [3, 2, 1, 0], [15, 16, 4, 9], [15, 20, 4, 8], [[5, -1], [6, -1], [7, -1], [8, -1]], 16, 8,
                         free=[9, 3, 2])
    assert got.row_slots.tolist() == [5 * 16 + 15, 2 * 16, 2 * 16 + 1, 3 * 16, 3 * 16 + 1, 7 * 16 + 4, -1, -1]
    assert got.row_positions.tolist() == [16, 17, 18, 21, 22, 5, -1, -1]
    assert got.free_count.tolist() == [1] and got.lengths.tolist() == [18, 18, 5, 9]


@pytest.mark.parametrize("page", [16, 64, 256])
def test_reserve_refusals_on_the_device(cdx, page):
    print(f"reserve: sequences that are refused, page={page}", flush=True)
    full = [[1, 2], [3, -1], [4, -1], [5, -1], [6, -1]]
    # Past the capacity; a pool that has one page for two; one behind them that needs none.
    _check_reserve(cdx, [1, page, 2 * page, 1, page - 1], [2 * page, 1, 0, page, 1], [5] * 5, full, page, 5 * page,
                   free=[9])
    # An empty pool, and one whose count is out of range.
    _check_reserve(cdx, [1, 1], [0, 1], [-1, 0], [[-1, -1], [3, -1]], page, 2, free=[])
    t = _ints([[0, -1]])
    for count, left in ((-4, 0), (100, 2)):
        got = cdx.paged_reserve(_ints([1]), _ints([page]), _ints([page - 1]), t.clone(), page, 1,
                                free_pages=_ints([7, 8, 9]), free_count=_ints([count]))
        assert got.free_count.tolist() == [left] and got.counts.tolist() == [1 if left else 0]
    # More tokens than rows: the first that do not fit, and all behind them.
    _check_reserve(cdx, [3, 5, 2, 0], [0] * 4, [-1] * 4, full[:4], page, 7, free=list(range(20)))
    _check_reserve(cdx, [3, 4, 2], [0] * 3, [-1] * 3, full[:3], page, 8, stride=3, free=list(range(20)))
    _check_reserve(cdx, [3, 3, 2], [0] * 3, [-1] * 3, full[:3], page, 8, stride=3)
    # Negative counts and lengths.
    _check_reserve(cdx, [-3, 2, 2 ** 31 - 1, 1], [4, -7, 0, 0], [3, -1, -1, -1], full[:4], page, 4, free=[1, 2, 3])
    # Sums past 32 bits.
    _check_reserve(cdx, [2 ** 31 - 1] * 3 + [1], [0] * 4, [-1] * 4, full[:4], page, 4, free=[1, 2, 3])


@pytest.mark.parametrize("seed", range(12))
def test_reserve_and_truncate_random(cdx, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 2, 7, 64, 511, 512, 513, 1100])
    page, width = rng.choice([16, 32, 64, 128, 256]), rng.choice([1, 2, 9])
    padded = rng.random() < 0.4
    most = rng.choice([1, 2, 30, page * width])
    lengths = [rng.choice([0, rng.randint(0, page * width), -1]) for _ in range(B)]
    counts = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(B)]
    positions = [rng.randint(-1, 10 ** 6) for _ in range(B)]
    used = sum(chunk.pages(max(n, 0), page) for n in lengths)
    need = sum(max(0, chunk.pages(max(n, 0) + c, page) - chunk.pages(max(n, 0), page)) for n, c in zip(lengths, counts))
    free = rng.sample(range(used + need + 50), max(0, rng.choice([need // 2, need + 5, need])))
    table = [[rng.randint(0, 10 ** 6) for _ in range(width)] for _ in range(B)]
    rows = B * most if padded else max(0, sum(max(c, 0) for c in counts) + rng.choice([0, 5, -3]))
    print(f"reserve {B} x {most}, page={page} width={width} padded={padded} rows={rows} free={len(free)}/{need}", flush=True)
    pool = rng.random() < 0.8
    _check_reserve(cdx, counts, lengths, positions, table, page, rows, most if padded else None, free if pool else None)

    to = [rng.choice([0, rng.randint(-2, page * width), 10 ** 6, max(n, 0)]) for n in lengths]
    room = rng.choice([len(free) + used + 9, len(free) + used // 2])
    have = _ints((free + [-5] * room)[:room])
    got = cdx.paged_truncate(_ints(to), _ints(lengths), _ints(positions), _ints(table), page, have, _ints([len(free)]))
    want = chunk.truncate(to, lengths, positions, table, page, free, room)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == [len(want[2])]
    assert have.tolist() == (want[2] + [-5] * room)[:room]


def test_a_pool_without_pages(cdx):
    print("reserve: an empty list of free pages", flush=True)
    free, count, table = _ints([]), _ints([0]), _ints([[3, -1], [4, -1]])
    rows = cdx.paged_reserve(_ints([2, 1]), _ints([15, 3]), _ints([14, 2]), table, 16, 3, free_pages=free,
                             free_count=count)
    assert rows.counts.tolist() == [0, 1] and rows.row_slots.tolist() == [-1, -1, 67]
    new = cdx.paged_truncate(_ints([0, 9]), rows.lengths, rows.positions, table, 16, free, rows.free_count)
    assert [t.tolist() for t in new] == [[0, 4], [-1, 3], [0]]


def test_truncate_undoes_reserve(cdx):
    print("truncate undoes reserve", flush=True)
    rng = random.Random(5)
    B, page, width = 40, 16, 6
    lengths = [rng.randint(0, 40) for _ in range(B)]
    counts = [rng.randint(0, 50) for _ in range(B)]
    free = _ints(rng.sample(range(1000), 300))
    count, table = _ints([300]), torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    before = free.clone()
    rows = cdx.paged_reserve(_ints(counts), _ints(lengths), _ints(lengths) - 1, table, page, sum(counts),
                             free_pages=free, free_count=count)
    assert rows.counts.tolist() == counts
    free[int(rows.free_count):300] = -9  # what was taken is not read again
    new = cdx.paged_truncate(_ints(lengths), rows.lengths, rows.positions, table, page, free, rows.free_count)
    assert new[0].tolist() == lengths and new[1].tolist() == [n - 1 for n in lengths] and new[2].tolist() == [300]
    assert torch.equal(free, before)


def test_pages_strided_and_wide_tables(cdx):
    print("reserve: a table inside a wider one, strided counts", flush=True)
    wide = torch.full((3, 9), -7, dtype=torch.int32, device="cuda")
    both = _ints([[2, 5], [17, 3], [1, 40]])
    free, count = _ints([4, 5, 6, 7, 8]), _ints([5])
    rows = cdx.paged_reserve(both[:, 0], both[:, 1], both[:, 1] - 1, wide[:, 2:6], 16, 20, free_pages=free,
                             free_count=count)
    want = chunk.reserve([2, 17, 1], [5, 3, 40], [4, 2, 39], [[-7] * 4] * 3, 16, 20, None, [4, 5, 6, 7, 8])
    assert rows.row_slots.tolist() == want[5] and wide[:, 2:6].tolist() == want[-1]
    assert bool((wide[:, :2] == -7).all()) and bool((wide[:, 6:] == -7).all())
    with pytest.raises(ValueError, match="rows of its own"):
        cdx.paged_reserve(both[:, 0], both[:, 1], both[:, 1], wide.t()[:3], 16, 20)
    with pytest.raises(ValueError, match="rows of its own"):
        cdx.paged_reserve(both[:, 0], both[:, 1], both[:, 1], wide[:1].expand(3, 9), 16, 20)


# ---- the append ---------------------------------------------------------------

@pytest.mark.parametrize("nq,nkv,D,page,norm,dtype", [
    (16, 8, 128, 64, True, bf16), (12, 4, 64, 16, True, torch.float32), (16, 4, 80, 32, True, bf16),
    (8, 4, 40, 256, True, torch.float32), (4, 2, 64, 128, False, bf16), (3, 1, 8, 16, True, bf16),
    (5, 5, 104, 32, False, torch.float32),
])
def test_chunk_append(cdx, nq, nkv, D, page, norm, dtype):
    print(f"chunk append {nq}/{nkv} D={D} page={page} norm={norm} {dtype}", flush=True)
    R, P = 19, 5
    g = torch.Generator().manual_seed(D + nq)
    k, v, _ = ref.cache(1, nkv, D, page, P, spare=0, seed=D)
    k0, v0 = k.clone(), v.clone()
    qkv = torch.randn(R, (nq + 2 * nkv) * D, generator=g).to(dtype)
    wq, wk = ((1 + 0.1 * torch.randn(2, D, generator=g)).to(bf16)) if norm else (None, None)
    slots = torch.randperm(P * page, generator=g)[:R].tolist()
    slots[:6] = [0, P * page - 1, -1, P * page, -2 ** 40, 2 ** 40]
    slots[6:] = [s for s in slots[6:] if s not in (0, P * page - 1)] + [-1] * sum(s in (0, P * page - 1) for s in slots[6:])
    pos = torch.randint(0, 9001, (R,), generator=g).tolist()
    pos[7], pos[8] = 9000, 0
    q = cdx.paged_chunk_append(qkv.cuda(), k, v, _ints(slots, torch.int64), _ints(pos), nq, _table(9001, D),
                               wq.cuda() if norm else None, wk.cuda() if norm else None)
    x = qkv.double().view(R, nq + 2 * nkv, D)
    ek, ev = k0.cpu().clone(), v0.cpu().clone()
    for r in range(R):
        def head(i, w):
            y = x[r, i]
            if w is not None:
                y = y * torch.rsqrt(y.square().mean() + 1e-6) * w.double()
            return ref.rope(y, pos[r])

        def close(got, want):
            # One rounding of the result, and fp32 arithmetic (and a table rounded to fp32) on
            # values of the row's size.
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().max()
            assert bool(((got.double().cpu() - want).abs() <= tol).all())

        if not 0 <= slots[r] < P * page:
            assert not q[r].any()
            continue
        for i in range(nq):
            close(q[r, i], head(i, wq))
        pg, row = divmod(slots[r], page)
        for h in range(nkv):
            close(k[pg, h, row], head(nq + h, wk))
            ek[pg, h, row] = k[pg, h, row].cpu()
            ev[pg, h, row] = x[r, nq + nkv + h].to(bf16)
    assert torch.equal(k.cpu(), ek) and torch.equal(v.cpu(), ev)  # v exactly, and nothing else written


def test_chunk_append_is_the_append_of_one_token(cdx):
    print("chunk append against paged_qkv_append", flush=True)
    B, nq, nkv, D, page = 9, 12, 4, 64, 32
    k, v, table = ref.cache(B, nkv, D, page, 3, seed=3)
    k1, v1 = k.clone(), v.clone()
    qkv = torch.randn(B, (nq + 2 * nkv) * D, device="cuda").to(bf16)
    w = (1 + 0.1 * torch.randn(2, D, device="cuda")).to(bf16)
    lens, cs = _ints([0, 1, 31, 32, 33, 64, 95, 5, 17]), _table(200, D)
    pos = lens + 3
    pos[2], pos[3] = -1, 500  # no angle: NaN
    rows = cdx.paged_reserve(torch.ones_like(lens), lens, pos - 1, table, page, B)
    assert rows.row_positions.tolist() == pos.tolist()
    a = cdx.paged_qkv_append(qkv, k, v, table, lens + 1, pos, nq, cs, w[0], w[1])
    b = cdx.paged_chunk_append(qkv, k1, v1, rows.row_slots, rows.row_positions, nq, cs, w[0], w[1])
    for x, y in ((a, b), (k, k1), (v, v1)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_chunk_append_takes_strided_rows(cdx):
    print("chunk append: strided operands", flush=True)
    R, nq, nkv, D, page = 4, 4, 2, 64, 16
    k, v, _ = ref.cache(2, nkv, D, page, 2)
    wide = torch.randn(R, 3 * (nq + 2 * nkv) * D + 8, device="cuda").to(bf16)
    slots = torch.stack([_ints([3, 17, 40, 63], torch.int64)] * 2, 1)
    pos, cs = torch.stack([_ints([1, 2, 3, 4])] * 3, 1), _table(40, D)
    for at in (8, 3):
        x = wide[:, at:at + (nq + 2 * nkv) * D]
        k1, v1, k2, v2 = k.clone(), v.clone(), k.clone(), v.clone()
        a = cdx.paged_chunk_append(x.contiguous(), k1, v1, slots[:, 0].contiguous(), pos[:, 1].contiguous(), nq, cs)
        b = cdx.paged_chunk_append(x, k2, v2, slots[:, 0], pos[:, 1], nq, cs)
        assert torch.equal(a, b) and torch.equal(k1, k2) and torch.equal(v1, v2)
    empty = cdx.paged_chunk_append(wide[:0, :(nq + 2 * nkv) * D], k, v, slots[:0, 0], pos[:0, 0], nq, cs)
    assert empty.shape == (0, nq, D)


# ---- attention ----------------------------------------------------------------

def _few(most, group):
    """Whether all of a call's queries fit the tiles of few queries, whose weights keep 16 bits."""
    return most * group <= 16


def _case(B, nq, nkv, D, page, before, counts, gaps=None, seed=0, fill=float("nan")):
    """Operands of a call; every slot past a sequence's length holds ``fill``."""
    g = torch.Generator().manual_seed(seed)
    lengths = [n + c for n, c in zip(before, counts)]
    width = max(1, chunk.pages(max(lengths), page))
    k, v, table = ref.cache(B, nkv, D, page, width, seed=seed, fill=fill)
    for b, n in enumerate(lengths):
        for s in range(0, n, page):
            m = min(page, n - s)
            pg = int(table[b, s // page])
            k[pg, :, :m] = torch.randn(nkv, m, D, generator=g).to(bf16).cuda()
            v[pg, :, :m] = torch.randn(nkv, m, D, generator=g).to(bf16).cuda()
    gaps = gaps or [0] * B
    starts, at = [], 0
    for c, gap in zip(counts, gaps):
        starts.append(at)
        at += c + gap
    q = (1.5 * torch.randn(at, nq, D, generator=g)).to(bf16).cuda()
    return q, k, v, table, starts, counts, lengths


def _run(cdx, q, k, v, table, starts, counts, lengths, **kw):
    return cdx.paged_chunk_attention(q, k, v, table, _ints(starts), _ints(counts), _ints(lengths), **kw)


def _check(out, want, bound):
    got = out.double().view(want.shape)
    ok = ((got - want).abs() <= bound) | (want.isnan() & got.isnan())
    assert bool(ok.all()), f"off by {float(((got - want).abs() / bound.clamp_min(1e-30)).nan_to_num().max())} of the bound"


HEADS = [(16, 8, 128), (16, 4, 80), (12, 4, 64), (8, 4, 40), (8, 8, 32), (4, 2, 16), (2, 1, 8), (5, 1, 96), (3, 3, 104),
         (40, 2, 72), (24, 8, 48), (6, 2, 112), (8, 2, 120), (7, 7, 56), (16, 16, 24), (4, 4, 88)]
RAGGED = [([0, 1, 15, 16, 17, 31, 32, 33], [1, 2, 3, 1, 16, 17, 5, 0]),
          ([0, 5, 63, 64, 65, 200], [200, 129, 64, 65, 1, 33]),
          ([700, 0, 3], [1, 1, 1]),
          ([1021], [7])]


@pytest.mark.parametrize("nq,nkv,D", HEADS)
@pytest.mark.parametrize("ragged", range(len(RAGGED)))
def test_chunk_attention(cdx, nq, nkv, D, ragged):
    before, counts = RAGGED[ragged]
    page = (16, 32, 64, 128, 256)[(D // 8 + ragged) % 5]
    print(f"chunk attention {nq}/{nkv} D={D} page={page} before={before} counts={counts}", flush=True)
    args = _case(len(counts), nq, nkv, D, page, before, counts, gaps=[0, 2, 0, 1, 0, 0, 3, 0][:len(counts)], seed=D + ragged)
    few = _few(max(counts), nq // nkv)
    want, bound = chunk.attention(*args, rounded_p=not few)
    _check(_run(cdx, *args, max_tokens=max(counts)), want, bound)
    if ragged == 0:
        want, bound = chunk.attention(*args, scale=0.02, rounded_p=True)
        _check(_run(cdx, *args, scale=0.02), want, bound)  # (max_tokens not known)


@pytest.mark.parametrize("nq,nkv,D,page,B,before,count", [
    (16, 8, 128, 64, 2, 2000, 700), (16, 4, 80, 16, 3, 999, 257), (12, 4, 64, 256, 1, 5000, 130),
    (8, 4, 40, 32, 5, 17, 300), (16, 8, 128, 128, 1, 20000, 3), (4, 2, 64, 16, 1, 0, 1500), (8, 1, 128, 64, 70, 40, 4),
])
def test_chunk_attention_longer(cdx, nq, nkv, D, page, B, before, count):
    print(f"chunk attention {nq}/{nkv} D={D} page={page} {B} x {before} + {count}", flush=True)
    args = _case(B, nq, nkv, D, page, [before] * B, [count] * B, seed=count)
    want, bound = chunk.attention(*args, rounded_p=not _few(count, nq // nkv))
    out = _run(cdx, *args, max_tokens=count)
    _check(out, want, bound)
    assert torch.equal(out, _run(cdx, *args, max_tokens=count))


@pytest.mark.parametrize("nq,nkv,D,before,count", [(16, 8, 128, 40, 100), (12, 4, 64, 0, 130), (16, 4, 80, 9, 3),
                                                   (8, 4, 40, 64, 64), (2, 2, 128, 4, 5)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_special_values_of_later_tokens_do_not_reach_earlier_ones(cdx, nq, nkv, D, before, count, value):
    print(f"chunk attention: {value} in later tokens, {nq}/{nkv} D={D} {before} + {count}", flush=True)
    args = _case(1, nq, nkv, D, 16, [before], [count], seed=D)
    q, k, v, table, starts, counts, lengths = args
    at = count // 2  # the first token with such a value in v, in one column of each head; the last one has it in k too
    for slot, pages in ((before + at, v), (before + count - 1, v), (before + count - 1, k)):
        pages[int(table[0, slot // 16]), :, slot % 16, D // 3] = value
    want, bound = chunk.attention(*args, rounded_p=not _few(count, nq // nkv))
    out = _run(cdx, *args, max_tokens=count)
    got = out.view(want.shape).double()
    _check(got[:at], want[:at], bound[:at])
    # From it on its column is what it is in 64 bits, the others are finite up to the last token.
    cols = torch.arange(D, device="cuda") != D // 3
    _check(got[at:count - 1][..., cols], want[at:count - 1][..., cols], bound[at:count - 1][..., cols])
    for x, y in ((got[at:count - 1, :, D // 3], want[at:count - 1, :, D // 3]),):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.isinf(), y.isinf())
        assert torch.equal(x[y.isinf()], y[y.isinf()])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("slots,count,gap", [(64, 1, 3), (200, 5, 2), (3000, 2, 3), (90, 1, 200), (900, 150, 40)])
def test_special_values_do_not_reach_rows_without_tokens(cdx, value, slots, count, gap):
    """Rows behind a sequence's are taken along with its last ones; they stay zeros, whatever its cache holds."""
    print(f"chunk attention: {value} in {slots} slots, {count} rows and {gap} without a token", flush=True)
    args = _case(2, 4, 2, 64, 16, [slots - count, 0], [count, 0], gaps=[gap, gap], seed=slots)
    q, k, v, table, starts, counts, lengths = args
    for slot in (3, slots // 2):
        v[int(table[0, slot // 16]), :, slot % 16, 5] = value
    q[count:] = value
    out = _run(cdx, *args, max_tokens=count)
    assert not out[count:].any() and not bool(out[:count].view(count, 4, 64)[..., 5].isfinite().any())


def test_missing_pages(cdx):
    print("chunk attention: pages outside the pool", flush=True)
    for count in (3, 100):
        args = _case(3, 4, 2, 64, 16, [40, 40, 40], [count] * 3, seed=count)
        q, k, v, table, starts, counts, lengths = args
        want, bound = chunk.attention(*args)
        table[0, 1] = -1
        table[1, (40 + count - 1) // 16] = k.shape[0]  # the last one: the tokens before it do not see it
        out = _run(cdx, *args, max_tokens=count).view(want.shape)
        assert bool(out[:count].isnan().all())
        sees = 40 + torch.arange(count) >= (40 + count - 1) // 16 * 16
        mid = out[count:2 * count]
        assert bool(mid[sees].isnan().all())
        keep = torch.cat([torch.zeros(count, dtype=torch.bool), ~sees, torch.ones(count, dtype=torch.bool)])
        _check(out[keep], want[keep], bound[keep])


def test_rows_without_tokens_and_lengths_out_of_range(cdx):
    print("chunk attention: gaps, lengths below the counts and past the capacity", flush=True)
    for most, few in ((4, True), (90, False)):
        args = _case(4, 4, 2, 64, 16, [5, 5, 5, 5], [most, 1, most, 2], gaps=[3, 0, 40, 7], seed=2)
        q, k, v, table, starts, counts, lengths = args
        cap = table.shape[1] * 16
        k.nan_to_num_(0.5), v.nan_to_num_(0.5)  # (every slot counts for the sequence past the capacity)
        lengths = [lengths[0], 0, 2, cap + 1]  # one without slots, one shorter than its tokens, one too long
        want, bound = chunk.attention(q, k, v, table, starts, counts, lengths, rounded_p=not few)
        out = _run(cdx, q, k, v, table, starts, counts, lengths, max_tokens=most)
        _check(out, want, bound)
        gap = torch.ones(q.shape[0], dtype=torch.bool)
        for s, c in zip(starts, counts):
            gap[s:s + c] = False
        assert int(gap.sum()) == 50 and not out[gap.cuda()].any()
        assert not out[starts[1]].any() and not out[starts[2]:starts[2] + most - 2].any()
        # No sequence at all brings a token; negative counts bring none.
        for none in ([0] * 4, [-3] * 4):
            assert not _run(cdx, q, k, v, table, starts, none, [0, 9, -5, 7], max_tokens=most).any()


def test_scores_without_a_finite_one(cdx):
    print("chunk attention: scores of -inf", flush=True)
    for count in (2, 70):
        args = _case(1, 4, 2, 64, 16, [30], [count], seed=1)
        q, k, v, table, starts, counts, lengths = args
        q.fill_(1.0)
        for t in range(20):  # the first slots weigh nothing
            k[int(table[0, t // 16]), :, t % 16] = -float("inf")
        want, bound = chunk.attention(*args)
        rest = [x.clone() for x in (k, v)]
        bound = torch.where(bound.isfinite(), bound, 0.0)
        # The bound of the rest: the scores' sizes of the slots that count.
        for t in range(20):
            rest[0][int(table[0, t // 16]), :, t % 16] = 0.0
        _, bound = chunk.attention(q, rest[0], v, table, starts, counts, lengths)
        _check(_run(cdx, *args, max_tokens=count), want, bound)
        for t in range(30 + count):
            k[int(table[0, t // 16]), :, t % 16] = -float("inf")
        assert bool(_run(cdx, *args, max_tokens=count).isnan().all())


def test_chunk_of_one_is_the_attention_of_one(cdx):
    print("chunk attention against paged_attention", flush=True)
    before = [0, 1, 31, 32, 700, 63]
    args = _case(6, 16, 8, 128, 64, before, [1] * 6, seed=9)
    q, k, v, table, starts, counts, lengths = args
    assert torch.equal(_run(cdx, *args, max_tokens=1), cdx.paged_attention(q, k, v, table, _ints(lengths)))


def test_many_sequences(cdx):
    print("chunk attention: more sequences than one look takes", flush=True)
    rng = random.Random(3)
    for B in (63, 64, 65, 200, 4100):
        before = [rng.randint(0, 20) for _ in range(B)]
        counts = [rng.choice([0, 0, 1, 2, 30 if B < 300 else 3]) for _ in range(B)]
        counts[0] = 1
        args = _case(B, 4, 2, 32, 16, before, counts, seed=B)
        want, bound = chunk.attention(*args)
        _check(_run(cdx, *args), want, bound)


@pytest.mark.parametrize("nq,nkv,counts,before", [
    (4, 4, [129, 129], [0, 0]), (4, 4, [129, 1, 193, 300], [0, 60, 0, 0]), (8, 4, [65, 64, 129], [0, 127, 0]),
    (6, 2, [43, 43, 86], [62, 0, 20]), (4, 1, [33, 1, 65, 97, 2], [0, 255, 0, 31, 500]), (12, 4, [500], [0]),
    (20, 1, [7, 40, 13], [0, 0, 64]), (128, 1, [1, 2, 3], [0, 9, 300]), (150, 1, [1, 2, 3], [0, 9, 300]),
])
def test_every_tile_once(cdx, nq, nkv, counts, before):
    """Sequences whose tiles end past their tokens, at and around steps of the order that tiles are taken in."""
    print(f"chunk attention: tiles {nq}/{nkv} {counts} over {before}", flush=True)
    args = _case(len(counts), nq, nkv, 16, 16, before, counts, seed=nq)
    want, bound = chunk.attention(*args)
    _check(_run(cdx, *args, max_tokens=max(counts)), want, bound)
    _check(_run(cdx, *args, max_tokens=0), want, bound)  # a wrong hint chooses another kernel, no other result


@pytest.mark.parametrize("seed", range(10))
def test_random_batches(cdx, seed):
    rng = random.Random(seed)
    nq, nkv = rng.choice([(4, 4), (4, 2), (6, 2), (8, 2), (16, 1), (3, 1)])
    D, page = rng.choice([8, 32, 40, 64, 80, 128]), rng.choice([16, 32, 64, 128, 256])
    B = rng.choice([1, 2, 5, 30, 64, 65, 130])
    most, old = rng.choice([1, 4, 40, 300, 1000 // B + 1]), rng.choice([0, 1, 70, 600, 4000 // B])
    counts = [rng.choice([0, 1, most, rng.randint(0, most)]) for _ in range(B)]
    counts[rng.randrange(B)] = most
    before = [rng.choice([0, old, rng.randint(0, old)]) for _ in range(B)]
    gaps = [rng.choice([0, 0, 0, rng.randint(0, 9)]) for _ in range(B)]
    print(f"chunk attention: random {nq}/{nkv} D={D} page={page} B={B} most={most} old={old}", flush=True)
    args = _case(B, nq, nkv, D, page, before, counts, gaps=gaps, seed=seed)
    want, bound = chunk.attention(*args, rounded_p=not _few(most, nq // nkv))
    out = _run(cdx, *args, max_tokens=most)
    _check(out, want, bound)
    gap = torch.ones(out.shape[0], dtype=torch.bool)
    for s, c in zip(args[4], counts):
        gap[s:s + c] = False
    assert not out[gap.cuda()].any()


def test_strided_operands_and_streams(cdx):
    print("chunk attention: strided operands, another stream", flush=True)
    args = _case(3, 4, 2, 64, 16, [9, 40, 0], [40, 3, 5], seed=4)
    q, k, v, table, starts, counts, lengths = args
    want = _run(cdx, *args)
    wide_q = torch.empty(q.shape[0], 4, 130, dtype=bf16, device="cuda")
    wide_q[..., 1:65] = q
    wide_t = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    wide_t[:, 2:2 + table.shape[1]] = table
    three = torch.stack([_ints(starts), _ints(counts), _ints(lengths)], 1)
    got = cdx.paged_chunk_attention(wide_q[..., 1:65], k, v, wide_t[:, 2:2 + table.shape[1]], three[:, 0], three[:, 1],
                                    three[:, 2])
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(cdx, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert _run(cdx, q[:0], k, v, table, [0] * 3, [0] * 3, lengths).shape == (0, 4 * 64)


def test_pool_past_32_bits(cdx):
    print("chunk attention and append: a pool of more than 2^31 values", flush=True)
    nq, nkv, D, page = 4, 2, 128, 256
    P = 2 ** 31 // (nkv * page * D) + 40
    k = torch.zeros(P, nkv, page, D, dtype=bf16, device="cuda")
    v = torch.zeros_like(k)
    small = _case(1, nq, nkv, D, page, [300], [60], seed=8)
    q, ks, vs, table, starts, counts, lengths = small
    far = _ints([[P - 1, P - 7]])
    k[far[0].long()], v[far[0].long()] = ks[table[0].long()], vs[table[0].long()]
    want = _run(cdx, *small)
    assert torch.equal(_run(cdx, q, k, v, far, starts, counts, lengths), want)
    rows = cdx.paged_reserve(_ints([2]), _ints([360]), _ints([359]), far, page, 2)
    qkv = torch.randn(2, (nq + 2 * nkv) * D, device="cuda").to(bf16)
    cdx.paged_chunk_append(qkv, k, v, rows.row_slots, rows.row_positions, nq, _table(400, D))
    assert torch.equal(v[P - 7, :, 104:106].transpose(0, 1), qkv.view(2, -1, D)[:, nq + nkv:])


# ---- together -----------------------------------------------------------------

def test_a_run_of_calls_on_a_shared_pool(cdx):
    """Prompts, steps, speculated tokens taken back and sequences that end and begin: every call's attention
    against one computed from the tokens of each sequence."""
    nq, nkv, D, page, B, width = 8, 4, 64, 16, 4, 8
    print("a run of calls on a shared pool", flush=True)
    g = torch.Generator(device="cuda").manual_seed(0)
    P = 14  # fewer than B * width
    k = torch.full((P, nkv, page, D), float("nan"), dtype=bf16, device="cuda")
    v = k.clone()
    free, left = torch.randperm(P, generator=g, device="cuda").to(torch.int32), _ints([P])
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    lengths, positions = _ints([0] * B), _ints([-1] * B)
    cs = _table(width * page, D)
    told = [[] for _ in range(B)]  # every sequence's (k, v) rows, in 64 bits of their bf16 values

    def call(counts, stride=None):
        nonlocal lengths, positions, left
        R = B * stride if stride else sum(counts)
        qkv = torch.randn(R, (nq + 2 * nkv) * D, generator=g, device="cuda").to(bf16)
        rows = cdx.paged_reserve(_ints(counts), lengths, positions, table, page, R, stride=stride, free_pages=free,
                                 free_count=left)
        lengths, positions, left = rows.lengths, rows.positions, rows.free_count
        q = cdx.paged_chunk_append(qkv, k, v, rows.row_slots, rows.row_positions, nq, cs)
        out = cdx.paged_chunk_attention(q, k, v, table, rows.starts, rows.counts, rows.lengths, max_tokens=max(counts))
        want = torch.zeros(R, nq, D, dtype=torch.float64)
        x = qkv.double().cpu().view(R, -1, D)
        for b, (s, n) in enumerate(zip(rows.starts.tolist(), rows.counts.tolist())):
            for i in range(n):
                pos = len(told[b])
                kk = torch.stack([ref.rope(x[s + i, nq + h], pos) for h in range(nkv)]).to(bf16).double()
                told[b].append((kk, x[s + i, nq + nkv:]))
                ks, vs = (torch.stack(t, 1) for t in zip(*told[b]))
                qq = torch.stack([ref.rope(x[s + i, h], pos) for h in range(nq)]).to(bf16).double()
                for h in range(nq):
                    p = torch.softmax(D ** -0.5 * (ks[h // 2] @ qq[h]), 0)
                    want[s + i, h] = p @ vs[h // 2]
        # q and k rounded to bf16 may differ by a step from those here (fp32 arithmetic before the rounding):
        # 2^-7 of some; the attention's own error as elsewhere.  Values are of size 1, sums of 2.
        assert float((out.double().cpu().view(want.shape) - want).abs().max()) <= 2.0 ** -5
        return rows

    call([20, 1, 33, 0])                       # 2 + 1 + 3 pages
    call([1, 1, 1, 40], stride=40)             # a padded batch; 0 + 0 + 0 + 3 pages
    assert int(left) == P - 9
    rows = call([5, 5, 5, 5])                  # speculated
    keep = _ints([2, 0, 5, 1])
    told = [t[:len(t) - 5 + n] for t, n in zip(told, keep.tolist())]
    lengths, positions, left = cdx.paged_truncate(lengths - rows.counts + keep, lengths, positions, table, page, free, left)
    call([1] * 4)
    lengths, positions, left = cdx.paged_truncate(_ints([10 ** 6, 10 ** 6, 0, 10 ** 6]), lengths, positions, table, page,
                                                  free, left)
    told[2] = []                               # the third has ended; another one takes its place
    call([1, 30, 90, 1])
    assert lengths.tolist() == [len(t) for t in told]
    refused = call([128, 1, 1, 1])             # the first lacks the pages; the others go on
    assert refused.counts.tolist()[0] == 0 and lengths.tolist() == [len(t) for t in told]


def test_captured_and_replayed(cdx):
    """A step of reserve, append and attention in a graph, replayed with eager calls between."""
    print("captured and replayed", flush=True)
    nq, nkv, D, page, B, width, P = 8, 4, 64, 16, 3, 6, 18
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros(P, nkv, page, D, dtype=bf16, device="cuda")
    v = torch.zeros_like(k)
    free, cs = torch.randperm(P, generator=gen, device="cuda").to(torch.int32), _table(width * page, D)
    state = torch.cat([_ints([0] * B), _ints([-1] * B), _ints([P])])
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    counts, R = _ints([7, 1, 3]), 12
    qkv = torch.randn(R, (nq + 2 * nkv) * D, generator=gen, device="cuda").to(bf16)

    def step(k, v, table, state):
        rows = cdx.paged_reserve(counts, state[:B], state[B:2 * B], table, page, R, free_pages=free,
                                 free_count=state[2 * B:])
        q = cdx.paged_chunk_append(qkv, k, v, rows.row_slots, rows.row_positions, nq, cs)
        out = cdx.paged_chunk_attention(q, k, v, table, rows.starts, rows.counts, rows.lengths)
        state.copy_(torch.cat([rows.lengths, rows.positions, rows.free_count]))
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k.clone(), v.clone(), table.clone(), state.clone())
    torch.cuda.current_stream().wait_stream(side)
    eager = [t.clone() for t in (k, v, table, state)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k, v, table, state)
    for i in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager)
        assert torch.equal(out, want), i
        assert all(torch.equal(a, b) for a, b in zip((k, v, table, state), eager)), i
