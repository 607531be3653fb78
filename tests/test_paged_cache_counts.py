"""What PagedKVCache counts on the host and on the device, on the CPU (tests/_paged_sim.py): calls after captured ones,
counts that do not fit, and bounds."""

from __future__ import annotations

import pytest
import torch

from _paged_sim import Sim


@pytest.mark.parametrize("lengths", [None, [20, 7]])
def test_a_call_after_replayed_prompts(monkeypatch, lengths):
    """Prompts on pages of the cache's own, captured and replayed on an emptied cache."""
    given = None if lengths is None else Sim.device(lengths)
    sim = Sim(monkeypatch, 2, 32, page_size=16)
    cache = sim.cache
    prompts = sim.capture(lambda c: c.begin(2, 20, given))
    sim.holds([0, 0])
    held = lengths or [20, 20]
    for _ in range(2):
        cache.release([0, 1])
        sim.replay(prompts)
        sim.holds(held)
        with pytest.raises(ValueError, match="full"):  # 20 + 14 of 32
            cache.begin(2, 14, token_counts=[14, 1])
        sim.holds(held)
        cache.begin(2, 12, token_counts=[12, 1])
        assert cache.rows.counts.tolist() == [12, 1]
        sim.holds([32, held[1] + 1])
        # A call of one token each is a step behind the replayed prompts, no prompt of its own.
        cache.reset()
        sim.replay(prompts)
        cache.begin(2, 1)
        assert not cache.prompt
        sim.holds([n + 1 for n in held])


@pytest.mark.parametrize("pages", [None, 4])
@pytest.mark.parametrize("cut", ["truncate", "reset"])
def test_a_call_after_replayed_cuts(monkeypatch, pages, cut):
    """The host's lengths are too large after them: they are read, not gone by."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=pages)
    cache = sim.cache
    cache.begin(2, 20, token_counts=[20, 18])
    sim.holds([20, 18], pages)
    graph = sim.capture(lambda c: c.truncate(Sim.device([5, 3])) if cut == "truncate" else c.reset())
    sim.holds([20, 18], pages)
    held = [5, 3] if cut == "truncate" else [0, 0]
    for i in range(3):
        cache.begin(2, 11, token_counts=[11, 11])
        sim.holds([31, 29] if i == 0 else [n + 11 for n in held], pages)
        sim.replay(graph)
        sim.holds(held, pages)
        with pytest.raises(ValueError, match="full"):
            cache.begin(2, 33, token_counts=[33 - held[0], 1])
        cache.begin(2, 32, token_counts=[27, 26])
        sim.holds([held[0] + 27, held[1] + 26], pages)
        sim.replay(graph)
        sim.holds(held, pages)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("pages", [None, 3])
def test_counts_on_the_device_that_do_not_fit_their_rows(monkeypatch, pages, packed):
    """Where a call reads them, they are held against its rows as the host's are; where it does not, the device leaves
    such a sequence out and the host's bounds stay bounds."""
    capacity = 48 if packed else 32
    sim = Sim(monkeypatch, 2, capacity, page_size=16, pages=pages)
    cache = sim.cache
    rows = 33 if packed else 20
    bad = [30, 4]  # past 20 rows each, and past 33 in all
    for _ in range(2):
        with pytest.raises(ValueError, match="token_counts"):
            cache.begin(2, rows, token_counts=bad, packed=packed)
        if pages is not None:  # (a pool of fewer pages than could be asked for: read)
            with pytest.raises(ValueError, match="token_counts"):
                cache.begin(2, rows, token_counts=Sim.device(bad), packed=packed)
            sim.holds([0, 0], pages)
        cache.begin(2, rows, token_counts=Sim.device([16, 17]), packed=packed)
        sim.holds([16, 17], pages)
        # A bound of the lengths past the capacity: read.
        with pytest.raises(ValueError, match="token_counts"):
            cache.begin(2, rows, token_counts=Sim.device([31, 3]), packed=packed)
        sim.holds([16, 17], pages)
        cache.begin(2, rows, token_counts=Sim.device([0, 15]), packed=packed)
        sim.holds([16, 32], pages)
        cache.reset()
    if pages is None:
        cache.begin(2, rows, token_counts=Sim.device(bad), packed=packed)
        assert cache.rows.counts.tolist() == ([30, 0] if packed else [0, 4])
        sim.holds(cache.rows.counts.tolist())
        assert cache.longest >= max(cache.rows.counts.tolist())
        cache.begin(2, 60, token_counts=[18, 40] if packed else [32, 28], packed=packed)
        sim.holds([48, 40] if packed else [32, 32])


@pytest.mark.parametrize("pages,step", [(None, False), (5, False), (5, True)])
def test_captured_calls_do_not_move_the_bounds_past_the_capacity(monkeypatch, pages, step):
    """No sequence has more tokens than its capacity, however many graphs are made of a cache's calls."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=pages)
    cache = sim.cache
    cache.begin(2, 20, token_counts=[20, 3])
    for _ in range(20):
        sim.capture(lambda c: c.begin(2, 1) if step else c.begin(2, 7, token_counts=Sim.device([7, 2])))
        assert cache.longest <= 32 and cache.newest <= 32
    assert cache.lengths.tolist() == [20, 3]
    cache.begin(2, 12, token_counts=[12, 9])
    sim.holds([32, 12], pages)


@pytest.mark.parametrize("keep", [None, 16])
def test_a_step_after_replays_that_emptied_a_full_cache(monkeypatch, keep):
    """A step is refused as full, or cuts the cache, by the lengths that the device has."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, keep=keep)
    cache = sim.cache
    prompts = sim.capture(lambda c: c.begin(2, 20))
    for _ in range(2):
        sim.replay(prompts)
        for n in range(21, 33):
            cache.begin(2, 1)
            sim.holds([n, n])
        if keep is None:
            with pytest.raises(ValueError, match="full"):
                cache.begin(2, 1)
            sim.holds([32, 32])


@pytest.mark.parametrize("pages", [None, 4])
@pytest.mark.parametrize("lengths", [None, [20, 7]])
def test_replayed_prompts_begin_the_batch_anew(monkeypatch, pages, lengths):
    """Captured prompts are prompts at every replay, also where sequences still hold the tokens of the last."""
    given = None if lengths is None else Sim.device(lengths)
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=pages)
    prompts = sim.capture(lambda c: c.begin(2, 20, given))
    held = lengths or [20, 20]
    for _ in range(3):
        sim.replay(prompts)
        sim.holds(held, pages)
        sim.cache.begin(2, 1)
        sim.holds([n + 1 for n in held], pages)


def test_captured_calls_take_no_counts_of_the_host(monkeypatch):
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=4)
    cache = sim.cache
    for call in (lambda c: c.begin(2, 3, torch.tensor([3, 2])), lambda c: c.begin(2, 3, token_counts=[3, 2]),
                 lambda c: c.truncate([1, 1]), lambda c: c.release([0])):
        with pytest.raises(ValueError, match="captured"):
            sim.capture(call)
        assert cache.longest == cache.newest == 0
    sim.holds([0, 0], 4)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_prompt_lengths_of_any_integers(monkeypatch, dtype):
    """Lengths in types that hold them, but not the prompts' rows nor what is left of them."""
    import complexity_deep as cdx
    S, lens = 300, torch.tensor([3, 120, 64, 1], dtype=dtype)
    sim = Sim(monkeypatch, 4, 320, page_size=16)
    sim.cache.begin(4, S, lens)
    sim.holds([3, 120, 64, 1])
    assert sim.cache.longest == 120
    sim.cache.reset()
    taken = []

    class Model:
        def forward(self, ids, past_key_values, token_counts):
            past_key_values.begin(*ids.shape, token_counts=token_counts)
            taken.append(token_counts.tolist())
            return cdx.CausalLMOutput(loss=None, logits=ids.unsqueeze(-1).float())

    ids = torch.arange(4 * S).view(4, S)
    last = cdx.ComplexityModel._prompts_in_pieces(Model(), ids, lens, sim.cache, 50)
    assert [sum(c) for c in zip(*taken)] == [3, 120, 64, 1] and taken[1] == [0, 50, 14, 0]
    assert last[:, 0].tolist() == [2, S + 119, 2 * S + 63, 3 * S]
    sim.holds([3, 120, 64, 1])
    for bad in (lens.float(), lens[:3], lens > 3):
        with pytest.raises(ValueError, match="prompt_lengths"):
            cdx.ComplexityModel._prompts_in_pieces(Model(), ids, bad, sim.cache, 50)
        sim.cache.reset()
        with pytest.raises(ValueError, match="prompt_lengths"):
            sim.cache.begin(4, S, bad)


def test_prompts_in_pieces_need_an_unbounded_cache():
    """Refused before the cache is emptied."""
    import complexity_deep as cdx
    cfg = cdx.ComplexityConfig.complexity_tiny()
    cache = cdx.PagedKVCache(cfg, 2, 40, keep=10, device="cpu")
    cache.begin(2, 12)
    with pytest.raises(ValueError, match="keep"):
        cdx.ComplexityModel.generate_paged(None, torch.zeros(2, 12, dtype=torch.int64), 3, cache=cache, chunk=4)
    assert cache.lengths.tolist() == [12, 12]


@pytest.mark.parametrize("pages", [None, 6])
def test_a_captured_call_of_one_token_each_on_a_cache_that_replays_may_have_filled(monkeypatch, pages):
    """A step or a prompt of one token: the host cannot know which, and must not guess."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=pages)
    cache = sim.cache
    first = sim.capture(lambda c: c.begin(2, 1))  # nothing was captured before: a prompt
    assert cache.prompt
    cache.reset()
    prompts = sim.capture(lambda c: c.begin(2, 20))
    cache.reset()
    sim.replay(prompts)
    with pytest.raises(ValueError, match="token_counts"):
        sim.capture(lambda c: c.begin(2, 1))
    sim.holds([20, 20], pages)
    counted = sim.capture(lambda c: c.begin(2, 1, token_counts=Sim.device([1, 1])))
    sim.replay(counted)
    sim.holds([21, 21], pages)
    cache.begin(2, 1)  # (an eager call reads the lengths: after it a captured one is a step)
    step = sim.capture(lambda c: c.begin(2, 1))
    sim.replay(step)
    sim.holds([23, 23], pages)
    sim.replay(first)
    sim.holds([1, 1], pages)


@pytest.mark.parametrize("pages", [None, 4])
@pytest.mark.parametrize("replayed", [False, True])
def test_prompts_of_a_cache_that_the_device_has_emptied(monkeypatch, pages, replayed):
    """By a cut whose lengths the host does not know."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, pages=pages)
    cache = sim.cache
    cache.begin(2, 20)
    cut = sim.capture(lambda c: c.truncate(Sim.device([0, 0]))) if replayed else None
    for prompts in ((20, None), (1, torch.tensor([1, 1])), (9, torch.tensor([2, 9])), (32, None)):
        with pytest.raises(ValueError, match="after the prompts"):
            cache.begin(2, *prompts)
        if replayed:
            sim.replay(cut)
        else:
            cache.truncate(Sim.device([0, 0]))
        sim.holds([0, 0], pages)
        cache.begin(2, *prompts)
        assert cache.prompt
        sim.holds([prompts[0]] * 2 if prompts[1] is None else prompts[1].tolist(), pages)


def test_replayed_prompts_of_a_bounded_cache_have_no_weights_of_the_last_batch(monkeypatch):
    """The weights say what a later cut keeps."""
    sim = Sim(monkeypatch, 2, 32, page_size=16, keep=20)
    cache = sim.cache
    cache.weights.fill_(3.0)  # (as steps leave them)
    prompts = sim.capture(lambda c: c.begin(2, 9))
    assert bool((cache.weights == 3.0).all())
    for _ in range(2):
        sim.replay(prompts)
        sim.holds([9, 9])
        assert not cache.weights.any()
        assert cache.slot_positions[..., :9].eq(torch.arange(9)).all() and cache.slot_positions[..., 9:].eq(-1).all()
        cache.weights.fill_(2.0)
