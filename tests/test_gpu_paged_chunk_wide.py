"""Attention of several new tokens in block tables wider than the sequences, as a cache's are: how a call is cut up goes
by the table's width, what it computes does not."""

from __future__ import annotations

import pytest
import torch

import _paged_chunk as chunk
from test_gpu_paged_chunk import _case, _check, _few, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq,nkv,D,page,before,counts", [
    (16, 8, 128, 64, [900, 0, 300], [128, 5, 70]), (12, 4, 64, 16, [0], [500]), (16, 4, 80, 32, [700, 65], [9, 200]),
    (16, 8, 128, 64, [3000], [8]), (8, 4, 40, 16, [63, 0, 1], [1, 1, 4]), (4, 2, 64, 16, [5] * 70, [3] * 69 + [90]),
])
@pytest.mark.parametrize("wide", [4, 16, 300])
def test_wide_tables(cdx, nq, nkv, D, page, before, counts, wide):
    print(f"wide tables: {nq}/{nkv} D={D} {before[:3]} + {counts[:3]} x {wide}", flush=True)
    args = _case(len(counts), nq, nkv, D, page, before, counts, gaps=[2] * len(counts), seed=D)
    q, k, v, table, starts, counts, lengths = args
    B, width = table.shape
    table = torch.cat([table, torch.full((B, width * (wide - 1)), -1, dtype=torch.int32, device="cuda")], 1)
    want, bound = chunk.attention(*args, rounded_p=not _few(max(counts), nq // nkv))
    out = _run(cdx, q, k, v, table, starts, counts, lengths, max_tokens=max(counts))
    _check(out, want, bound)
    gap = torch.ones(q.shape[0], dtype=torch.bool)
    for s, n in zip(starts, counts):
        gap[s:s + n] = False
    assert not out[gap.cuda()].any()
