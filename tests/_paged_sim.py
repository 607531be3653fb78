"""PagedKVCache on the CPU: its page operators replaced by the plain forms of tests/_paged_chunk.py, and calls captured
and replayed as a graph does it, by their work on tensors alone."""

from __future__ import annotations

import torch

import _paged_chunk as chunk

HOST = ("longest", "newest", "_exact", "_lengths", "prompt", "_step", "rows", "most", "_before", "_saved",
        "_replays")


def _side_by_side(*lists):
    whole = torch.tensor([x for part in lists for x in part], dtype=torch.int32)
    return whole.split([len(part) for part in lists])


def reserve(counts, lengths, positions, block_table, page_size, rows, *, stride=None, free_pages=None, free_count=None):
    from complexity_deep.paged import PagedRows
    n = None if free_count is None else int(free_count)
    out = chunk.reserve(counts.tolist(), lengths.tolist(), positions.tolist(), block_table.tolist(), page_size, rows,
                        stride, None if n is None else free_pages.tolist()[:n])
    starts, new_counts, new_lengths, new_positions, left, slots, where_to, table = out
    block_table.copy_(torch.tensor(table, dtype=torch.int32))
    parts = _side_by_side(starts, new_counts, new_lengths, new_positions, [0 if left is None else left])
    return PagedRows(*parts[:4], None if n is None else parts[4], torch.tensor(slots, dtype=torch.int64),
                     torch.tensor(where_to, dtype=torch.int32))


def truncate(to, lengths, positions, block_table, page_size, free_pages, free_count):
    room = free_pages.numel()
    n, pos, free = chunk.truncate(to.tolist(), lengths.tolist(), positions.tolist(), block_table.tolist(), page_size,
                                  free_pages.tolist()[:int(free_count)], room)
    free_pages[:len(free)] = torch.tensor(free, dtype=torch.int32)
    return _side_by_side(n, pos, [len(free)])


class _Device(torch.Tensor):
    """Taken for a tensor on the GPU, with what is computed from it."""
    is_cuda = property(lambda self: True)


class Sim:
    """``cache`` (a PagedKVCache on the CPU) with ``capture`` and ``replay`` of its calls."""

    def __init__(self, monkeypatch, batch_size, max_length, **kw):
        import complexity_deep as cdx
        from complexity_deep import paged
        self.capturing = False
        monkeypatch.setattr(paged, "paged_reserve", reserve)
        monkeypatch.setattr(paged, "paged_truncate", truncate)
        monkeypatch.setattr(paged, "_capturing", lambda t: self.capturing)
        self.cache = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), batch_size, max_length, device="cpu", **kw)

    @staticmethod
    def device(values):
        """Integers that the host does not know."""
        return torch.tensor(values).as_subclass(_Device)

    def _tensors(self):
        c = self.cache
        return [t for t in (c._state, c._undo, c.block_table, c.free_pages, c.weights, c.slot_positions)
                if t is not None]

    def _host(self):
        return {name: getattr(self.cache, name) for name in HOST}

    def capture(self, call):
        """The graph of call(cache): counted on the host, not on the device."""
        before, host = [t.clone() for t in self._tensors()], self._host()
        self.capturing = True
        try:
            call(self.cache)
        finally:
            self.capturing = False
            for t, b in zip(self._tensors(), before):
                t.copy_(b)
        return call, host

    def replay(self, graph):
        """The graph's work on tensors, with the host's side as it was (the branches are the captured ones)."""
        call, host = graph
        now = self._host()
        for name, value in host.items():
            setattr(self.cache, name, value)
        self.capturing = True
        try:
            call(self.cache)
        finally:
            self.capturing = False
            for name, value in now.items():
                setattr(self.cache, name, value)

    def holds(self, lengths, pages=None):
        """The device's lengths, and what a pool of so many pages must have left and in use then."""
        c = self.cache
        assert c.lengths.tolist() == lengths and c.positions.tolist() == [n - 1 for n in lengths]
        if pages is not None:
            used = [row[:chunk.pages(n, c.page_size)] for row, n in zip(c.block_table.tolist(), lengths)]
            used = sum(used, [])
            assert int(c.free_count) == pages - len(used)
            assert sorted(used + c.free_pages.tolist()[:pages - len(used)]) == list(range(pages))
