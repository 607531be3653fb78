"""What PagedKVCache counts on the host and on the device, on the CPU (tests/_paged_sim.py): calls after captured ones,
counts that do not fit, and bounds."""

from __future__ import annotations

import pytest
import torch

from _paged_sim import Sim


@pytest.mark.parametrize("lengths", [None, [20, 7]])
def test_a_call_after_replayed_prompts(monkeypatch, lengths):
    """Prompts on pages of the cache's own, captured and replayed on an emptied cache."""
    given = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
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
