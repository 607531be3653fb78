"""Calls of a model on a PagedKVCache after captured and replayed ones, against an eager cache of the same tokens."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_model import _model

pytestmark = pytest.mark.gpu


def _graph(call, warm):
    """call() captured, after warm() on another stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        warm()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out = call()
    return graph, out


@torch.inference_mode()
def test_calls_after_replayed_prompts(cdx):
    print("counts: replayed prompts", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S = 2, 20
    cache, eager, other = (cdx.PagedKVCache(m.config, B, 32, page_size=16) for _ in range(3))
    gen = torch.Generator().manual_seed(4)
    ids, more = (torch.randint(0, 600, (B, n), generator=gen).cuda() for n in (S, 14))
    prompts, logits = _graph(lambda: m(ids, past_key_values=cache).logits, lambda: m(ids, past_key_values=other))
    for i in range(4):
        ids.copy_(torch.randint(0, 600, (B, S), generator=gen))
        for c in (cache, eager):
            c.release([0, 1])
        prompts.replay()
        assert torch.equal(logits, m(ids, past_key_values=eager).logits)
        if i % 2 == 0:
            for c in (cache, eager):
                with pytest.raises(ValueError, match="full"):
                    m(more, past_key_values=c, token_counts=[14, 1])
            got, want = (m(more[:, :12], past_key_values=c, token_counts=[12, 1]).logits for c in (cache, eager))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1, 0], want[1, 0])
        else:
            got, want = (m(more[:, :1], past_key_values=c).logits for c in (cache, eager))
            assert torch.equal(got, want)
        assert cache.lengths.tolist() == eager.lengths.tolist() == ([32, 21] if i % 2 == 0 else [21, 21])


@pytest.mark.parametrize("pages", [None, 4])
@torch.inference_mode()
def test_calls_after_replayed_cuts(cdx, pages):
    print(f"counts: replayed truncate, pages={pages}", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache, eager, other = (cdx.PagedKVCache(m.config, 2, 32, page_size=16, pages=pages) for _ in range(3))
    ids = torch.randint(0, 600, (2, 90), generator=torch.Generator().manual_seed(4)).cuda()
    to = torch.tensor([5, 3]).cuda()
    for c in (cache, eager):
        m(ids[:, :20], past_key_values=c, token_counts=[20, 18])
    graph, _ = _graph(lambda: cache.truncate(to), lambda: other.truncate(to))
    for i in range(4):
        graph.replay()
        eager.truncate(to)
        assert cache.lengths.tolist() == eager.lengths.tolist() == [5, 3]
        got, want = (m(ids[:, 20 + i:47 + i], past_key_values=c, token_counts=[27, 26]).logits for c in (cache, eager))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, :26], want[1, :26])
        assert torch.equal(cache._state, eager._state) and cache.lengths.tolist() == [32, 29]
