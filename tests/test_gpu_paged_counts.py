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


@torch.inference_mode()
def test_counts_on_the_device_past_their_rows(cdx):
    print("counts: on the device, past their rows", flush=True)
    m = _model(cdx, 64, 4, 2)
    ids = torch.randint(0, 600, (2, 40), generator=torch.Generator().manual_seed(4)).cuda()
    cache = cdx.PagedKVCache(m.config, 2, 48, page_size=16, pages=4)
    for _ in range(2):
        for rows, counts in ((ids, [41, 1]), (ids, [1, 41]), (ids[0], [30, 11])):
            with pytest.raises(ValueError, match="token_counts"):
                m(rows, past_key_values=cache, token_counts=torch.tensor(counts).cuda())
            assert cache.lengths.tolist() == [0, 0] and int(cache.free_count) == 4
        m(ids, past_key_values=cache, token_counts=torch.tensor([30, 20]).cuda())
        assert cache.lengths.tolist() == [30, 20]
        m(ids[:, :3], past_key_values=cache, token_counts=torch.tensor([2, 3]).cuda())
        assert cache.lengths.tolist() == [32, 23]
        cache.release([0, 1])
    # Nothing has to be read: the first sequence's rows attend to nothing, the second's are as ever.
    cache, other = (cdx.PagedKVCache(m.config, 2, 48, page_size=16) for _ in range(2))
    got = m(ids[:, :9], past_key_values=cache, token_counts=torch.tensor([10, 5]).cuda()).logits
    # (On the device too: 9 rows for a bound take another kernel, which rounds its weights to 8 bits, than 5 do.)
    want = m(ids[:, :9], past_key_values=other, token_counts=torch.tensor([0, 5]).cuda()).logits
    assert torch.equal(got[1, :5], want[1, :5]) and cache.lengths.tolist() == [0, 5] and cache.longest >= 5
    m(ids, past_key_values=cache, token_counts=[40, 40])
    assert cache.lengths.tolist() == [40, 45]


@torch.inference_mode()
def test_graphs_of_more_rows_than_the_capacity(cdx):
    """Each graph's rows count for the host's bound, which stays within the capacity: the rotary table need not grow,
    which no capture can do."""
    print("counts: graphs of many rows", flush=True)
    m = _model(cdx, 64, 4, 2, layers=1, max_position_embeddings=128)
    cache, eager, other = (cdx.PagedKVCache(m.config, 2, 128, page_size=16) for _ in range(3))
    ids = torch.randint(0, 600, (2, 60), generator=torch.Generator().manual_seed(4)).cuda()
    counts = torch.tensor([20, 11]).cuda()
    graphs = [_graph(lambda: m(ids, past_key_values=cache, token_counts=counts).logits,
                     lambda: m(ids, past_key_values=other, token_counts=counts)) for _ in range(4)]
    for graph, logits in graphs:
        graph.replay()
        want = m(ids, past_key_values=eager, token_counts=counts).logits
        assert torch.equal(logits[0, :20], want[0, :20]) and torch.equal(logits[1, :11], want[1, :11])
        assert cache.lengths.tolist() == eager.lengths.tolist()


@pytest.mark.parametrize("pages", [None, 4])
@torch.inference_mode()
def test_replayed_prompts_begin_the_batch_anew(cdx, pages):
    print(f"counts: prompts replayed over others, pages={pages}", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache, eager, other = (cdx.PagedKVCache(m.config, 2, 32, page_size=16, pages=pages) for _ in range(3))
    gen = torch.Generator().manual_seed(4)
    ids, n = torch.empty(2, 20, dtype=torch.int64, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
    ids.zero_(), n.fill_(20)
    prompts, logits = _graph(lambda: m(ids, past_key_values=cache, prompt_lengths=n).logits,
                             lambda: m(ids, past_key_values=other, prompt_lengths=n))
    for held in ([20, 7], [16, 20], [3, 17], [20, 20]):
        ids.copy_(torch.randint(0, 600, (2, 20), generator=gen)), n.copy_(torch.tensor(held))
        prompts.replay()
        eager.reset()
        want = m(ids, past_key_values=eager, prompt_lengths=n).logits
        for b, c in enumerate(held):
            assert torch.equal(logits[b, :c], want[b, :c])
        for _ in range(2):
            got, want = (m(ids[:, :1], past_key_values=c).logits for c in (cache, eager))
            assert torch.equal(got, want)
        assert cache.lengths.tolist() == eager.lengths.tolist() == [c + 2 for c in held]
        assert pages is None or int(cache.free_count) == int(eager.free_count)


def _no_waits(call):
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        return call()
    finally:
        torch.cuda.set_sync_debug_mode("default")


@pytest.mark.parametrize("pages", [None, 20])
@torch.inference_mode()
def test_counts_of_the_host_do_not_wait(cdx, pages):
    print(f"counts: no wait for the host's, pages={pages}", flush=True)
    m = _model(cdx, 64, 4, 2)
    ids = torch.randint(0, 600, (3, 40), generator=torch.Generator().manual_seed(4)).cuda()
    cache, other = (cdx.PagedKVCache(m.config, 3, 96, page_size=16, pages=pages) for _ in range(2))
    lens = torch.tensor([9, 4, 30])
    got, held = [], [torch.zeros(2 ** 26, device="cuda") for _ in range(2)]
    for c in (other, cache):
        def calls():
            for t in held:  # (work that is still queued when the counts are given)
                t.add_(1.0)
            c.reset()
            out = [m(ids[:, :30], past_key_values=c, prompt_lengths=lens).logits[2]]
            out.append(m(ids[:, :9], past_key_values=c, token_counts=[9, 1, 5]).logits[0])
            out.append(m(ids[0, :9], past_key_values=c, token_counts=torch.tensor([2, 0, 7])).logits)
            c.truncate([15, 5, 40])
            c.release([1])
            out.append(m(ids[:, :1], past_key_values=c).logits)
            c.reset()
            out.append(m._prompts_in_pieces(ids, None, c, 16))
            c.reset()
            out.append(m._prompts_in_pieces(ids, lens, c, 16))
            return out
        got.append(calls() if c is other else _no_waits(calls))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert cache.lengths.tolist() == [9, 4, 30]


@torch.inference_mode()
def test_counts_of_the_host_in_a_captured_call(cdx):
    """A graph would copy them at every replay from where they were: they are refused, and the capture goes on."""
    print("counts: the host's in a captured call", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache, eager, other = (cdx.PagedKVCache(m.config, 2, 64, page_size=16, pages=8) for _ in range(3))
    ids = torch.randint(0, 600, (2, 3), generator=torch.Generator().manual_seed(4)).cuda()
    counts = torch.tensor([3, 2]).cuda()

    def captured():
        for call in (lambda: m(ids, past_key_values=cache, token_counts=[3, 2]), lambda: cache.truncate([1, 1]),
                     lambda: cache.release([0]),
                     lambda: m(ids, past_key_values=cache, prompt_lengths=counts.new_zeros(2, device="cpu"))):
            with pytest.raises(ValueError, match="captured"):
                call()
        return m(ids, past_key_values=cache, token_counts=counts).logits

    graph, logits = _graph(captured, lambda: m(ids, past_key_values=other, token_counts=counts))
    for i in range(3):
        graph.replay()
        want = m(ids, past_key_values=eager, token_counts=counts).logits
        assert torch.equal(logits[0], want[0]) and torch.equal(logits[1, :2], want[1, :2])
        assert torch.equal(cache._state, eager._state) and cache.lengths.tolist() == [3 * i + 3, 2 * i + 2]


@torch.inference_mode()
def test_replayed_prompts_of_a_bounded_cache(cdx):
    """Cuts go by the weights of the batch at hand, not by those of the last one."""
    print("counts: prompts replayed on a bounded cache", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache, eager, other = (cdx.PagedKVCache(m.config, 2, 32, page_size=16, keep=14, recent=4) for _ in range(3))
    gen = torch.Generator().manual_seed(4)
    ids = torch.zeros(2, 12, dtype=torch.int64, device="cuda")
    prompts, logits = _graph(lambda: m(ids, past_key_values=cache).logits, lambda: m(ids, past_key_values=other))
    for _ in range(3):
        ids.copy_(torch.randint(0, 600, (2, 12), generator=gen))
        prompts.replay()
        eager.reset()
        assert torch.equal(logits, m(ids, past_key_values=eager).logits)
        for i in range(45):
            x = torch.randint(0, 600, (2, 1), generator=gen).cuda()
            got, want = (m(x, past_key_values=c).logits for c in (cache, eager))
            assert torch.equal(got, want) and torch.equal(cache.lengths, eager.lengths), i
        assert torch.equal(cache.slot_positions[..., :14], eager.slot_positions[..., :14])
        assert int(cache.lengths.max()) < 32 and cache.positions.tolist() == [56, 56]


def test_reserve_without_rows_by_the_entry_point(cdx):
    """Results of no bytes lie over nothing, wherever their pointers are."""
    print("counts: reserve without rows", flush=True)
    from complexity_deep import _native as nat
    x = torch.tensor([[0, 0], [5, 9], [4, 8]], dtype=torch.int32, device="cuda")  # counts, lengths, positions
    table = torch.tensor([[3, 4], [1, 2]], dtype=torch.int32, device="cuda")
    out = torch.empty(4, 2, dtype=torch.int32, device="cuda")
    nat.check(nat.lib().cdx_paged_reserve(
        *(t.data_ptr() for t in x), 2, 0, 0, table.data_ptr(), 2, 2, 16, None, 0, None, *(t.data_ptr() for t in out), None,
        x.data_ptr() + 4, x.data_ptr() + 4, nat.stream_of(x)), "cdx_paged_reserve")
    assert out.tolist() == [[0, 0], [0, 0], [5, 9], [4, 8]]
