"""The kernel of few queries, whose weights keep 16 bits, held to its own bound where values and pages are special."""

from __future__ import annotations

import pytest
import torch

import _paged as ref
import _paged_chunk as chunk
from test_gpu_paged_chunk import _case, _check, _few, _run

pytestmark = pytest.mark.gpu
HEADS = [(4, 2, 64), (16, 8, 128), (8, 4, 40)]


@pytest.mark.parametrize("nq,nkv,D", HEADS)
@pytest.mark.parametrize("before,count", [(40, 3), (46, 4), (900, 8), (0, 1)])
def test_missing_pages(cdx, nq, nkv, D, before, count):
    print(f"few queries: pages outside the pool, {nq}/{nkv} D={D} {before} + {count}", flush=True)
    assert _few(count, nq // nkv)
    args = _case(3, nq, nkv, D, 16, [before] * 3, [count] * 3, seed=count)
    q, k, v, table, starts, counts, lengths = args
    want, bound = chunk.attention(*args, rounded_p=False)
    last = (before + count - 1) // 16
    table[0, last // 2] = -1
    table[1, last] = k.shape[0]  # (the tokens before the last page do not see it)
    out = _run(cdx, *args, max_tokens=count).view(want.shape)
    sees = before + torch.arange(count) >= last * 16
    first = before + torch.arange(count) >= last // 2 * 16
    gone = torch.cat([first, sees, torch.zeros(count, dtype=torch.bool)]).cuda()
    assert bool(out[gone].isnan().all())
    _check(out[~gone], want[~gone], bound[~gone])


@pytest.mark.parametrize("nq,nkv,D", HEADS)
@pytest.mark.parametrize("before,count", [(30, 2), (700, 8)])
def test_scores_without_a_finite_one(cdx, nq, nkv, D, before, count):
    """The first slots weigh nothing: the definition and its bound (as in _paged_chunk.attention) over the others."""
    print(f"few queries: scores of -inf, {nq}/{nkv} D={D} {before} + {count}", flush=True)
    args = _case(1, nq, nkv, D, 16, [before], [count], seed=1)
    q, k, v, table, starts, counts, lengths = args
    q.fill_(1.0)
    none = before * 2 // 3
    for t in range(none):
        k[int(table[0, t // 16]), :, t % 16] = -float("inf")
    ks, vs = (ref.slots(x, table, 0, before + count).double()[:, none:] for x in (k, v))
    want = torch.zeros(count, nq, D, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    sums = ((before + count) / 32 + 64) * 2.0 ** -23
    for i in range(count):
        for h in range(nq):
            kk, vv = (x[h // (nq // nkv), :before + i + 1 - none] for x in (ks, vs))
            p = torch.softmax(D ** -0.5 * kk.sum(1), 0)
            delta = (D + 8) * 2.0 ** -24 * D ** -0.5 * kk.abs().sum(1).max() + 2.0 ** -19
            want[i, h] = p @ vv
            bound[i, h] = (2.0 ** -16 + 2 * delta + sums) * (p @ vv.abs()) + 2.0 ** -8 * want[i, h].abs()
    _check(_run(cdx, *args, max_tokens=count), want, bound)
    for t in range(before + count):
        k[int(table[0, t // 16]), :, t % 16] = -float("inf")
    assert bool(_run(cdx, *args, max_tokens=count).isnan().all())
