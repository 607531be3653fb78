"""A ComplexityModel on a PagedKVCache with any number of tokens per sequence and call (token_counts), on
pages of its own and on a shared pool, against the fp32 oracle's forward over the whole sequences."""

from __future__ import annotations

import pytest
import torch

from _metrics import errors
from test_gpu_paged_model import MAX_REL, REL_RMS, _model, _oracle_logits

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


class _Run:
    """A model's calls on one cache, with the oracle's logits of every token beside them."""

    def __init__(self, cdx, oracle, m, B, total, **cache):
        self.m, self.B = m, B
        self.ids = torch.randint(0, 600, (B, total), generator=torch.Generator().manual_seed(B + total))
        self.want = _oracle_logits(oracle, m, self.ids)
        self.cache = cdx.PagedKVCache(m.config, B, total, **cache)
        self.cache.k_pages.fill_(float("nan")), self.cache.v_pages.fill_(float("nan"))
        self.at = [0] * B
        self.got, self.expected = [], []

    def call(self, counts, packed, on_device=True, **kw):
        n = torch.tensor(counts)
        if packed:
            ids = torch.cat([self.ids[b, a:a + c] for b, (a, c) in enumerate(zip(self.at, counts))])
        else:
            ids = torch.full((self.B, max(counts)), 599)
            for b, (a, c) in enumerate(zip(self.at, counts)):
                ids[b, :c] = self.ids[b, a:a + c]
        with torch.no_grad():
            out = self.m(ids.cuda(), past_key_values=self.cache, token_counts=n.cuda() if on_device else counts, **kw)
        row = 0
        for b, c in enumerate(counts):
            logits = out.logits[row:row + c] if packed else out.logits[b, :c]
            row += c
            self.got.append(logits)
            self.expected.append(self.want[b, self.at[b]:self.at[b] + c])
            self.at[b] += c
        assert self.cache.lengths.tolist() == self.at
        assert self.cache.positions.tolist() == [n - 1 for n in self.at]

    def step(self):
        at = torch.tensor(self.at)
        with torch.no_grad():
            out = self.m(self.ids[torch.arange(self.B), at].view(self.B, 1).cuda(), past_key_values=self.cache)
        self.got.append(out.logits[:, 0])
        self.expected.append(self.want[torch.arange(self.B), at])
        self.at = [n + 1 for n in self.at]
        assert self.cache.lengths.tolist() == self.at

    def back(self, to, **kw):
        self.cache.truncate(to, **kw)
        self.at = [min(a, max(0, int(t))) for a, t in zip(self.at, to)]
        assert self.cache.lengths.tolist() == self.at

    def check(self):
        e = errors(torch.cat(self.got), torch.cat(self.expected))
        print(e, flush=True)
        assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e


@pytest.mark.parametrize("D,nq,nkv,page,pages,kw", [
    (64, 4, 2, 16, None, {}), (128, 4, 2, 64, 5, {}), (40, 8, 4, 16, 14, {}), (80, 8, 2, 32, None, {}),
    (64, 12, 4, 16, 14, {"use_mu_guidance": False}), (32, 4, 4, 16, None, {"use_qk_norm": False}),
    (64, 4, 1, 16, 14, {"use_token_routed_mlp": False}),
])
@pytest.mark.parametrize("packed", [False, True])
def test_calls_of_any_size_match_the_whole_sequence(cdx, oracle, D, nq, nkv, page, pages, kw, packed):
    print(f"chunks D={D} heads={nq}/{nkv} page={page} pages={pages} packed={packed} {kw}", flush=True)
    r = _Run(cdx, oracle, _model(cdx, D, nq, nkv, **kw), 3, 90, page_size=page, pages=pages)
    r.call([21, 1, 0], packed)
    r.call([1, 33, 17], packed, on_device=False)
    r.step()
    r.call([2, 3, 1], packed)  # (few rows in all)
    r.step()
    r.call([40, 0, 1], packed)
    r.check()
    if pages is not None:
        used = sum(-(-n // page) for n in r.at)
        assert int(r.cache.free_count) == pages - used
        live = torch.cat([r.cache.block_table[b, :-(-n // page)] for b, n in enumerate(r.at)])
        free = r.cache.free_pages[:pages - used]
        assert sorted(torch.cat([live, free]).tolist()) == list(range(pages))


@pytest.mark.parametrize("pages", [None, 11])
def test_tokens_taken_back_and_sequences_released(cdx, oracle, pages):
    print(f"chunks: truncate and release, pages={pages}", flush=True)
    r = _Run(cdx, oracle, _model(cdx, 64, 4, 2), 3, 80, page_size=16, pages=pages)
    r.call([30, 20, 40], True)
    r.call([5, 5, 5], False)
    r.back(torch.tensor([33, 25, 41]).cuda())  # of the speculated five, three, five and one are kept
    r.call([1, 1, 1], True)
    r.step()
    r.cache.release([1])
    r.at[1] = 0
    assert r.cache.lengths.tolist() == r.at
    r.call([3, 50, 2], False)  # another sequence in its place
    r.back([10 ** 9, -5, 40])
    r.call([1, 17, 1], True)
    r.check()
    r.cache.release(range(3))
    r.at = [0, 0, 0]
    assert r.cache.lengths.tolist() == [0, 0, 0] and r.cache.newest == 0
    r.cache.reset()
    r.call([9, 40, 9], False)
    r.check()


def test_prompts_by_the_other_path_on_a_pool(cdx, oracle):
    """Prompts and steps without token_counts take their pages from the pool too."""
    print("pool: prompts and steps", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S = 3, 37
    ids = torch.randint(0, 600, (B, S + 12), generator=torch.Generator().manual_seed(2)).cuda()
    want = _oracle_logits(oracle, m, ids)
    lens = torch.tensor([37, 5, 18])
    for given in (lens, lens.cuda()):
        cache = cdx.PagedKVCache(m.config, B, S + 12, page_size=16, pages=9)
        got, expected, rows = [], [], torch.arange(B)
        with torch.no_grad():
            out = m(ids[:, :S], past_key_values=cache, prompt_lengths=given)
            assert int(cache.free_count) == 9 - (3 + 1 + 2)
            got.append(out.logits[rows.cuda(), cache.positions.long()])
            expected.append(want[rows, lens - 1])
            for i in range(11):
                at = lens + i
                got.append(m(ids[rows.cuda(), at.cuda()].view(B, 1), past_key_values=cache).logits[:, 0])
                expected.append(want[rows, at])
        assert cache.lengths.tolist() == (lens + 11).tolist() and int(cache.free_count) == 9 - (3 + 1 + 2)
        e = errors(torch.stack(got), torch.stack(expected))
        assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e


def test_refusals_leave_the_cache(cdx):
    print("chunks: refusals", flush=True)
    m = _model(cdx, 64, 4, 2)
    ids = torch.randint(0, 600, (2, 40)).cuda()
    for pages in (None, 4):
        cache = cdx.PagedKVCache(m.config, 2, 48, page_size=16, pages=pages)
        with torch.no_grad():
            for bad in ([41, 1], [-1, 3], [1], [1.5, 2], torch.tensor([1.0, 2.0]), torch.tensor([True, False])):
                with pytest.raises((ValueError, TypeError)):
                    m(ids, past_key_values=cache, token_counts=bad)
            with pytest.raises(ValueError):
                m(ids[0], past_key_values=cache, token_counts=[30, 11])  # 41 tokens in 40 rows
            with pytest.raises(ValueError):
                m(ids, past_key_values=cache, token_counts=[1, 1], prompt_lengths=torch.tensor([1, 1]))
            with pytest.raises(ValueError):
                m(ids, token_counts=[1, 1])
            with pytest.raises(ValueError):
                m(ids[0], past_key_values=cache, token_counts=[20, 20], labels=ids[0])
            assert cache.lengths.tolist() == [0, 0] and cache.newest == 0
            m(ids, past_key_values=cache, token_counts=[30, 20])
            before = cache._state.clone()
            for counts in ([19, 0], torch.tensor([19, 0]).cuda()):
                with pytest.raises(ValueError, match="full"):
                    m(ids[:, :19], past_key_values=cache, token_counts=counts)
            if pages:
                with pytest.raises(ValueError, match="1 pages are needed, and 0 of 4 are free"):
                    m(ids[:, :3], past_key_values=cache, token_counts=[3, 0])
            # A call that raises inside the model, with and without token_counts.
            attn = m.layers[1].self_attn
            attn.train(), setattr(attn, "attention_dropout", 0.1)
            for kw in (dict(token_counts=[1, 2]), {}):
                with pytest.raises(NotImplementedError):
                    m(ids[:, :2 if kw else 1], past_key_values=cache, **kw)
                assert torch.equal(cache._state, before) and (cache.longest, cache.newest) == (30, 30)
            attn.eval()
            m(ids[:, :2], past_key_values=cache, token_counts=torch.tensor([2, 2]).cuda())
            assert cache.lengths.tolist() == [32, 22]
            m(ids[:, :10], past_key_values=cache, token_counts=[0, 10])
            assert cache.lengths.tolist() == [32, 32]
            if pages:
                with pytest.raises(ValueError, match="free"):
                    m(ids[:, :1], past_key_values=cache)
                cache.release([0])
                m(ids[:, :1], past_key_values=cache)
                assert cache.lengths.tolist() == [1, 33]


def test_generation_with_prompts_in_pieces(cdx, oracle):
    print("generate_paged in pieces", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S = 3, 41
    ids = torch.randint(0, 600, (B, S), generator=torch.Generator().manual_seed(5)).cuda()
    want = _oracle_logits(oracle, m, ids)
    for lens in (None, torch.tensor([41, 7, 16]), torch.tensor([3, 32, 33]).cuda()):
        end = torch.full((B,), S) if lens is None else lens.cpu()
        for chunk in (1, 16, 64):
            cache = cdx.PagedKVCache(m.config, B, S + 8, page_size=16, pages=10)
            with torch.no_grad():
                got = m._prompts_in_pieces(ids, lens, cache, chunk)
            e = errors(got, want[torch.arange(B), end - 1])
            assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, (chunk, e)
            assert cache.lengths.tolist() == end.tolist()
        new = m.generate_paged(ids, 6, prompt_lengths=lens, chunk=16, cache=cache, eos_token_id=-1)
        assert new.shape == (B, 6) and cache.lengths.tolist() == (end + 5).tolist()
    with pytest.raises(ValueError):
        m.generate_paged(ids, 2, chunk=0)
    with pytest.raises(ValueError):
        m.generate_paged(ids[:, :0], 2, chunk=4)


def test_a_captured_call(cdx):
    """A call of given shape with its counts on the device, replayed with other ids and counts, against an
    eager cache of the same calls."""
    print("chunks: captured", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, T = 3, 24
    gen = torch.Generator().manual_seed(3)
    caches = [cdx.PagedKVCache(m.config, B, 200, page_size=16, pages=40) for _ in range(3)]
    ids = torch.randint(0, 600, (T,), generator=gen).cuda()
    counts = torch.tensor([10, 9, 5]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        for _ in range(2):
            m(ids, past_key_values=caches[2], token_counts=counts)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        logits = m(ids, past_key_values=caches[0], token_counts=counts).logits
    for i in range(5):
        ids.copy_(torch.randint(0, 600, (T,), generator=gen))
        counts.copy_(torch.tensor([[10, 9, 5], [0, 1, 20], [24, 0, 0], [1, 1, 1], [8, 8, 8]][i]))
        graph.replay()
        torch.cuda.synchronize()
        with torch.inference_mode():
            want = m(ids, past_key_values=caches[1], token_counts=counts).logits
        n = int(counts.sum())
        assert torch.equal(logits[:n], want[:n]), i
        assert torch.equal(caches[0]._state, caches[1]._state)


@pytest.mark.parametrize("pages", [None, 12])
def test_a_call_after_replayed_ones(cdx, pages):
    """Replays count on the device alone: the calls after them go by its lengths."""
    print(f"chunks: eager after replays, pages={pages}", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache = cdx.PagedKVCache(m.config, 2, 32, page_size=16, pages=pages)
    ids = torch.randint(0, 600, (2, 1), generator=torch.Generator().manual_seed(3)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        m(ids.expand(2, 18), past_key_values=cache, token_counts=[18, 18])
        m(ids, past_key_values=cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        m(ids, past_key_values=cache)
    with torch.inference_mode():
        for want in (22, 23, 24):
            if want == 22:
                for _ in range(3):
                    graph.replay()
            else:
                graph.replay()
            cache.truncate([want, want])
            assert cache.lengths.tolist() == [want, want]
            with pytest.raises(ValueError, match="full"):
                m(ids.expand(2, 33 - want), past_key_values=cache, token_counts=[1, 33 - want])
            assert cache.lengths.tolist() == [want, want]
        m(ids.expand(2, 8), past_key_values=cache, token_counts=[8, 0])
        assert cache.lengths.tolist() == [32, 24]
        # An emptied cache takes prompts, but not where replays have brought tokens meanwhile.
        cache.release([0, 1])
        graph.replay()
        with pytest.raises(ValueError):
            m(ids.expand(2, 8), past_key_values=cache)
        assert cache.lengths.tolist() == [1, 1]
        cache.release([0, 1])
        m(ids.expand(2, 8), past_key_values=cache)
        graph.replay()
        m(ids, past_key_values=cache)
    assert cache.lengths.tolist() == [10, 10] and cache.positions.tolist() == [9, 9]
    with pytest.raises(TypeError):
        cache.release([0.5])


@pytest.mark.parametrize("B", [2, 12])
def test_replayed_steps_of_a_pool_that_runs_out(cdx, B):
    """A step that a replay finds no page for is neither counted nor stored, and leaves the tokens that are there."""
    print(f"chunks: replayed steps of a pool that runs out, B={B}", flush=True)
    m = _model(cdx, 64, 4, 2)
    cache = cdx.PagedKVCache(m.config, B, 64, page_size=16, pages=B + 1)
    ids = torch.randint(0, 600, (B, 13), generator=torch.Generator().manual_seed(3)).cuda()
    new = ids[:, :1].clone()
    with torch.inference_mode():
        m(ids, past_key_values=cache)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(new, past_key_values=cache)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = m(new, past_key_values=cache).logits
        for _ in range(3):  # 14 -> 16, then the first sequence takes the page that is left
            graph.replay()
        assert cache.lengths.tolist() == [17] + [16] * (B - 1) and int(cache.free_count) == 0
        table = cache.block_table[:, 0].long()
        kept = [t[:, table].clone() for t in (cache.k_pages, cache.v_pages)]
        for n in range(18, 22):
            new.copy_(ids[:, n - 16:n - 15])
            graph.replay()
            assert cache.lengths.tolist() == [n] + [16] * (B - 1)
            assert cache.positions.tolist() == [n - 1] + [15] * (B - 1)
            for t, k in zip((cache.k_pages, cache.v_pages), kept):
                assert torch.equal(t[:, table], k)
        with pytest.raises(ValueError, match="pages"):
            m(new, past_key_values=cache)
        # An eager cache of the first sequence's tokens gives its logits.
        alone = cdx.PagedKVCache(m.config, 1, 64, page_size=16)
        want = m(torch.cat([ids[:1], *[ids[:1, :1]] * 4, ids[:1, 2:6]], 1), past_key_values=alone).logits[:, -1]
        e = errors(logits[:1, -1], want)
        assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e
        assert bool(logits.isfinite().all())
        cache.release(range(1, B))
        m(new, past_key_values=cache)
        assert cache.lengths.tolist() == [22] + [1] * (B - 1)


def test_modules_by_themselves(cdx):
    print("chunks: an attention module by itself", flush=True)
    m = _model(cdx, 64, 4, 2)
    attn = m.layers[0].self_attn
    x = torch.randn(1, 20, 256, device="cuda").to(bf16)
    with torch.no_grad():
        want = attn(x)[0]
        cache = cdx.PagedKVCache(m.config, 1, 40, page_size=16)
        for at, n in ((0, 13), (13, 1), (14, 6)):
            cache.begin(1, n, token_counts=[n])
            out, kv = attn(x[:, at:at + n], past_key_value=cache[0])
            e = errors(out, want[:, at:at + n])
            assert kv is None and e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e
        cache.begin(1, 3, token_counts=[3])
        with pytest.raises(ValueError):
            attn(x[:, :4], past_key_value=cache[0])
