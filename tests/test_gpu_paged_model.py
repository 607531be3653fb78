"""A ComplexityModel on a PagedKVCache: prompts, then one token per sequence and call, against the
fp32 oracle's forward over the whole sequences (every token attends to all before it)."""

from __future__ import annotations

import pytest
import torch

import _paged as ref
from _metrics import errors

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16

# As for the model's forward without a cache (tests/test_gpu_model.py).
MAX_REL, REL_RMS = 3e-2, 2e-2


def _model(cdx, D, nq, nkv, layers=3, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = cdx.ComplexityConfig(vocab_size=600, hidden_size=nq * D, intermediate_size=256, num_hidden_layers=layers,
                               num_attention_heads=nq, num_key_value_heads=nkv, num_experts=4, **kw)
    m = cdx.ComplexityModel(cfg)
    with torch.no_grad():
        for layer in m.layers:
            if layer.mu_guidance is not None:
                layer.mu_guidance.mu_proj.weight.normal_(0, 0.02)
        for n, p in m.named_parameters():
            if "norm" in n:
                p.add_(0.1 * torch.randn_like(p))
        if cfg.use_mu_guidance:
            m.mu_init.normal_(0, 0.5)
    return m.to("cuda", bf16).eval()


def _oracle_logits(oracle, m, ids):
    sd = {k: v.detach().float().cpu() for k, v in m.state_dict().items()}
    return oracle.forward(sd, m.config.to_dict(), ids.cpu())


@pytest.mark.parametrize("D,nq,nkv,B,page,kw", [
    (64, 4, 2, 3, 16, {}), (128, 4, 2, 1, 64, {}), (40, 8, 4, 2, 32, {}), (80, 8, 2, 9, 16, {}),
    (64, 12, 4, 2, 16, {"use_mu_guidance": False}), (32, 4, 4, 4, 128, {"use_qk_norm": False}),
    (64, 4, 1, 2, 16, {"use_token_routed_mlp": False}), (64, 2, 2, 70, 32, {}),
])
def test_prompts_and_steps_match_the_whole_sequence(cdx, oracle, D, nq, nkv, B, page, kw):
    print(f"paged model D={D} heads={nq}/{nkv} B={B} page={page} {kw}", flush=True)
    m = _model(cdx, D, nq, nkv, **kw)
    S, steps = 37, 12
    ids = torch.randint(0, 600, (B, S + steps), generator=torch.Generator().manual_seed(B)).cuda()
    want = _oracle_logits(oracle, m, ids)
    lens = torch.tensor([S - (5 * b) % S for b in range(B)], dtype=torch.int32)
    cache = cdx.PagedKVCache(m.config, B, S + steps, page_size=page)
    cache.k_pages.fill_(float("nan")), cache.v_pages.fill_(float("nan"))
    got, expected = [], []
    with torch.no_grad():
        out = m(ids[:, :S], past_key_values=cache, prompt_lengths=lens.cuda())
        assert out.past_key_values is cache
        rows = torch.arange(B)
        got.append(out.logits[rows.cuda(), cache.positions.long()])
        expected.append(want[rows, lens.long() - 1])
        for i in range(steps):  # each sequence's own next tokens
            at = lens.long() + i
            got.append(m(ids[rows.cuda(), at.cuda()].view(B, 1), past_key_values=cache).logits[:, 0])
            expected.append(want[rows, at])
    assert cache.lengths.tolist() == [int(n) + steps for n in lens]
    e = errors(torch.stack(got), torch.stack(expected))
    print(e, flush=True)
    assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e


def test_a_bounded_cache(cdx):
    """The same logits as without a bound until the cache is first cut, finite and bounded after."""
    print("paged model: bounded", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S = 3, 20
    ids = torch.randint(0, 600, (B, S + 60), generator=torch.Generator().manual_seed(1)).cuda()
    lens = torch.tensor([20, 3, 11]).cuda()
    cache = cdx.PagedKVCache(m.config, B, 32, page_size=16, keep=24, recent=8)
    free = cdx.PagedKVCache(m.config, B, S + 60, page_size=16)
    with torch.no_grad():
        a, b = (m(ids[:, :S], past_key_values=c, prompt_lengths=lens).logits for c in (cache, free))
        assert torch.equal(a, b)
        for i in range(60):
            tok = ids[:, S + i].view(B, 1)
            a, b = (m(tok, past_key_values=c).logits for c in (cache, free))
            if i < 12:
                e = errors(a, b)  # (the split of a row's keys follows the capacity)
                assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, (i, e)
            assert bool(torch.isfinite(a).all()) and int(cache.lengths.max()) <= 32
            assert cache.longest == int(cache.lengths.max()) and cache.newest == S + i + 1
            # Every slot in use has a position of its own, the newest tokens among them.
            for r in range(B):
                n, last = int(cache.lengths[r]), int(cache.positions[r])
                assert last == int(lens[r]) + i
                held = cache.slot_positions[:, r, :, :n]
                assert bool((held.sort(-1).values.diff(dim=-1) > 0).all()) and bool((held >= 0).all())
                for p in range(max(0, last - 7), last + 1):
                    assert bool((held == p).any(-1).all())
                # What each query head gave, over all its steps, is one a step.
                total = cache.weights[:, r].sum()
                assert bool(torch.isfinite(total)) and float(total) <= (i + 1) * 4 * 3 * 1.001
    assert int(cache.lengths.min()) >= 24


def test_generate_paged(cdx):
    print("generate_paged", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S, n = 3, 9, 24
    ids = torch.randint(1, 600, (B, S), generator=torch.Generator().manual_seed(2)).cuda()
    out = m.generate_paged(ids, n, temperature=0.0, eos_token_id=-5)
    assert out.shape == (B, n) and out.dtype == torch.int64
    cache = cdx.PagedKVCache(m.config, B, S + n)
    with torch.no_grad():
        logits = m(ids, past_key_values=cache).logits[:, -1]
        for i in range(n):
            assert torch.equal(logits.float().argmax(-1), out[:, i])
            logits = m(out[:, i:i + 1], past_key_values=cache).logits[:, -1]
    # Given random numbers, the same tokens, also on a cache that is used again.
    u = torch.rand(B, n, device="cuda")
    a = m.generate_paged(ids, n, uniforms=u, min_p=0.01, eos_token_id=-5, cache=cache)
    assert torch.equal(a, m.generate_paged(ids, n, uniforms=u, min_p=0.01, eos_token_id=-5, cache=cache))
    with torch.inference_mode():
        assert torch.equal(a, m.generate_paged(ids, n, uniforms=u, min_p=0.01, eos_token_id=-5))
        made_inside = cdx.PagedKVCache(m.config, B, S + n)
    assert torch.equal(a, m.generate_paged(ids, n, uniforms=u, min_p=0.01, eos_token_id=-5, cache=made_inside))
    # A right-padded prompt generates what it does on its own.
    lens = torch.tensor([S, 4, 6]).cuda()
    ragged = m.generate_paged(ids, n, temperature=0.0, prompt_lengths=lens, eos_token_id=-5)
    for r, k in enumerate(lens.tolist()):
        alone = m.generate_paged(ids[r:r + 1, :k], n, temperature=0.0, eos_token_id=-5)
        assert ragged[r, :3].tolist() == alone[0, :3].tolist()  # (later ones may differ by a rounding's argmax)
    # A sequence that ended repeats the end, and the generation stops with the last one.
    eos = int(out[0, 2])
    ended = m.generate_paged(ids, n, temperature=0.0, eos_token_id=eos)
    firsts = [(out[r] == eos).nonzero() for r in range(B)]
    stop = max(int(f[0]) + 1 if len(f) else n for f in firsts)
    assert ended.shape == (B, stop)
    for r, f in enumerate(firsts):
        k = int(f[0]) + 1 if len(f) else n
        assert torch.equal(ended[r, :k], out[r, :k]) and bool((ended[r, k:] == eos).all())
    bounded = cdx.PagedKVCache(m.config, B, 16, page_size=16, keep=8)
    assert m.generate_paged(ids, 40, uniforms=torch.rand(B, 40, device="cuda"), eos_token_id=-5,
                            cache=bounded).shape == (B, 40)
    assert int(bounded.lengths.max()) <= 16 and m.generate_paged(ids, 0).shape == (B, 0)


@pytest.mark.parametrize("B,keep", [(2, None), (9, None), (9, 24), (70, None)])
def test_steps_while_launches_are_timed(cdx, B, keep):
    """The Python launch sites compute what the native call paths do: the same bits, or for up to 8
    rows (whose norms are folded into the products otherwise) the same numbers."""
    print(f"paged model: launch hook, B={B} keep={keep}", flush=True)
    from complexity_deep import _native as nat
    m = _model(cdx, 64, 4, 2)
    ids = torch.randint(0, 600, (B, 30), generator=torch.Generator().manual_seed(4)).cuda()
    outs, names = [], set()
    for hook in (None, lambda name, *a: names.add(name)):
        cache = cdx.PagedKVCache(m.config, B, 32, page_size=16, keep=keep)
        try:
            nat.set_launch_hook(hook)
            with torch.no_grad():
                m(ids[:, :25], past_key_values=cache)
                outs.append(torch.stack([m(ids[:, i:i + 1], past_key_values=cache).logits for i in range(5)]))
        finally:
            nat.set_launch_hook(None)
    assert {"paged_write", "paged_attention"} <= names
    if B > 8:
        assert torch.equal(*outs)
    e = errors(*outs)
    assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e


def test_a_captured_step(cdx):
    """A step (with its tokens' choice) in a HIP graph, replayed, against eager steps."""
    print("paged model: captured step", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S, n = 2, 20, 8
    ids = torch.randint(0, 600, (B, S), generator=torch.Generator().manual_seed(3)).cuda()
    u = torch.rand(n, B, device="cuda")
    caches = [cdx.PagedKVCache(m.config, B, 64, page_size=16) for _ in range(2)]
    with torch.no_grad():
        first = [m(ids, past_key_values=c).logits[:, -1] for c in caches]
        assert torch.equal(*first)
        tok, uni = first[0].float().argmax(-1).view(B, 1), torch.zeros(B, device="cuda")
        eager = [tok.clone()]
        for i in range(n):
            logits = m(eager[-1], past_key_values=caches[0]).logits[:, -1]
            eager.append(cdx.sample_tokens(logits, u[i], top_k=50, top_p=0.9).view(B, 1))
        graph, counts = torch.cuda.CUDAGraph(), caches[1]._counts.clone()
        with torch.cuda.graph(graph):
            logits = m(tok, past_key_values=caches[1]).logits[:, -1]
            tok.copy_(cdx.sample_tokens(logits, uni, top_k=50, top_p=0.9).view(B, 1))
        caches[1]._counts.copy_(counts)
        for i in range(n):
            uni.copy_(u[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(tok, eager[i + 1]), i
    assert torch.equal(caches[0].lengths, caches[1].lengths)
    for r in range(B):
        for i in range(len(caches[0])):
            a, b = (ref.slots(c.layer(i)[0], c.block_table, r, S + n) for c in caches)
            assert torch.equal(a, b)


def test_refusals(cdx):
    print("paged model: refused calls", flush=True)
    m = _model(cdx, 64, 4, 2, layers=2)
    cfg, ids = m.config, torch.zeros(2, 5, dtype=torch.long, device="cuda")
    for bad in (dict(page_size=48), dict(max_length=0), dict(batch_size=0), dict(keep=0), dict(keep=32),
                dict(keep=8, recent=9)):
        with pytest.raises(ValueError):
            cdx.PagedKVCache(cfg, **{**dict(batch_size=2, max_length=32), **bad})
    odd = cdx.ComplexityConfig(hidden_size=64 * 3, num_attention_heads=16, num_key_value_heads=4)
    with pytest.raises(ValueError):
        cdx.PagedKVCache(odd, 2, 32)  # heads of 12
    cache = cdx.PagedKVCache(cfg, 2, 6, page_size=16)
    with torch.no_grad():
        for args in (dict(attention_mask=torch.ones(5, 5, dtype=torch.bool, device="cuda")),
                     dict(prompt_lengths=torch.tensor([1])), dict(prompt_lengths=torch.tensor([1.0, 2.0]))):
            with pytest.raises(ValueError):
                m(ids, past_key_values=cache, **args)
        with pytest.raises(ValueError):
            m(ids[:1], past_key_values=cache)
        with pytest.raises(ValueError):
            m(torch.zeros(2, 17, dtype=torch.long, device="cuda"), past_key_values=cache)
        with pytest.raises(ValueError):
            m(ids, prompt_lengths=torch.tensor([1, 2]))
        with pytest.raises(ValueError):
            m(ids, past_key_values=cdx.PagedKVCache(cdx.ComplexityConfig(
                hidden_size=256, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=3), 2, 32))
        assert cache.lengths.tolist() == [0, 0]  # nothing counted
        # A call that raises inside the model counts nothing either.
        attn = m.layers[1].self_attn
        attn.train(), setattr(attn, "attention_dropout", 0.1)
        with pytest.raises(NotImplementedError):
            m(ids, past_key_values=cache)
        assert cache.lengths.tolist() == [0, 0] and cache.newest == 0
        attn.eval()
        m(ids, past_key_values=cache)
        attn.train()
        with pytest.raises(NotImplementedError):
            m(ids[:, :1], past_key_values=cache)
        assert cache.lengths.tolist() == [5, 5] and cache.positions.tolist() == [4, 4] and cache.newest == 5
        attn.eval()
        with pytest.raises(ValueError):
            m(ids, past_key_values=cache)  # a second prompt
        for _ in range(11):
            m(ids[:, :1], past_key_values=cache)
        with pytest.raises(ValueError, match="full"):
            m(ids[:, :1], past_key_values=cache)
        with pytest.raises(ValueError):
            cache.evict()
        cache.reset()
        m(ids, past_key_values=cache)
        with pytest.raises(ValueError):
            m.generate_paged(ids, 4, uniforms=torch.rand(2, 3, device="cuda"))


def test_modules_by_themselves(cdx):
    """An attention module and a block on one layer of a cache, after begin."""
    print("paged model: modules by themselves", flush=True)
    m = _model(cdx, 64, 4, 2, layers=1, use_mu_guidance=False)
    B, S = 3, 12
    x = torch.randn(B, S + 1, 256, device="cuda").to(bf16)
    ids = torch.randint(0, 600, (B, S + 1), device="cuda")
    for module, kw in ((m.layers[0].self_attn, {}), (m.layers[0], {"token_ids": True})):
        args = lambda a, b: {k: ids[:, a:b].contiguous() for k in kw}  # noqa: E731
        cache = cdx.PagedKVCache(m.config, B, S + 1, page_size=16)
        with torch.no_grad():
            whole = module(x, **args(0, S + 1))[0]
            cache.begin(B, S)
            first = module(x[:, :S].contiguous(), past_key_value=cache[0], **args(0, S))[0]
            cache.begin(B, 1)
            last = module(x[:, S:].contiguous(), past_key_value=cache[0], **args(S, S + 1))[0]
        e = errors(torch.cat([first, last], 1), whole)
        assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, e


def test_a_cache_with_pages_of_its_own_order(cdx):
    """A pool whose pages a server handed out in another order, one prefix shared."""
    print("paged model: block table replaced", flush=True)
    m = _model(cdx, 64, 4, 2, layers=2)
    B, S = 2, 16
    ids = torch.randint(0, 600, (1, S), device="cuda").expand(B, S).contiguous()
    nxt = torch.randint(0, 600, (B, 6), device="cuda")
    plain = cdx.PagedKVCache(m.config, B, 48, page_size=16)
    mixed = cdx.PagedKVCache(m.config, B, 48, page_size=16)
    mixed.block_table = torch.tensor([[5, 0, 3], [5, 4, 1]], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        a, b = (m(ids, past_key_values=c).logits for c in (plain, mixed))
        assert torch.equal(a, b)
        for i in range(6):
            a, b = (m(nxt[:, i:i + 1], past_key_values=c).logits for c in (plain, mixed))
            assert torch.equal(a, b)


@pytest.mark.parametrize("B", [2, 9])
def test_block_tables_of_any_stride(cdx, B):
    """A block table whose columns are not neighbours in memory, as a view of a server's wider one."""
    print(f"paged model: strided block table, B={B}", flush=True)
    m = _model(cdx, 64, 4, 2, layers=2)
    ids = torch.randint(0, 600, (B, 20), generator=torch.Generator().manual_seed(8)).cuda()
    plain, strided = (cdx.PagedKVCache(m.config, B, 48, page_size=16) for _ in range(2))
    wide = torch.zeros(B, 6, dtype=torch.int32, device="cuda")
    wide[:, ::2] = plain.block_table
    wide[:, 1::2] = plain.block_table.flip(0)  # (pages of the other sequences)
    strided.block_table = wide[:, ::2]
    with torch.no_grad():
        a, b = (m(ids[:, :14], past_key_values=c).logits for c in (plain, strided))
        assert torch.equal(a, b)
        for i in range(14, 20):
            a, b = (m(ids[:, i:i + 1], past_key_values=c).logits for c in (plain, strided))
            e = errors(a, b)  # (the norms are folded, or not, by the call path)
            assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, (i, e)
    for r in range(B):
        for i in range(2):
            for x, y in zip(plain.layer(i)[:2], strided.layer(i)[:2]):
                a, b = (ref.slots(t, plain.block_table, r, 20).float() for t in (x, y))
                assert torch.equal(a[:, :14], b[:, :14])
                assert float((a - b).abs().max()) <= MAX_REL * float(a.abs().max())


def test_block_tables_of_other_types_are_refused(cdx):
    """Before anything is written, in the native call path and in the other one."""
    print("paged model: block tables of other types", flush=True)
    from complexity_deep.attention import qkv_paged
    m = _model(cdx, 64, 4, 2, layers=2)
    ids = torch.randint(0, 600, (2, 8), generator=torch.Generator().manual_seed(8)).cuda()
    cache = cdx.PagedKVCache(m.config, 2, 48, page_size=16)
    table = cache.block_table
    attn = m.layers[0].self_attn
    with torch.no_grad():
        m(ids[:, :5], past_key_values=cache)
        before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache._counts)]
        for bad in (table.long(), table.cpu(), table.float(), table[:1], table[0]):
            cache.block_table = bad
            with pytest.raises((ValueError, RuntimeError)):
                m(ids[:, 5:6], past_key_values=cache)
        cache.block_table = table
        x = torch.randn(2, 1, 256, device="cuda").to(bf16)
        args = dict(x=x, mu=None, w_x=attn.qkv_weights()[0], w_mu=attn.qkv_weights()[1], H=256, nq=4, q_norm_w=None,
                    k_norm_w=None, eps=1e-6, cos_sin=attn.rotary_emb.cos_sin_table(48, x.device),
                    k_pages=cache.k_pages[0], v_pages=cache.v_pages[0], block_table=table, lengths=cache.lengths,
                    positions=cache.positions)
        for name, bad in (("lengths", cache.lengths.long()), ("lengths", cache.lengths[:1]),
                          ("positions", cache.positions.cpu()), ("positions", cache.positions.float()),
                          ("cos_sin", args["cos_sin"].double()), ("cos_sin", args["cos_sin"][:, :16]),
                          ("q_norm_w", x[0, 0, :64]), ("k_pages", cache.k_pages[0].transpose(1, 2)),
                          ("v_pages", cache.v_pages[0][:1])):
            with pytest.raises((ValueError, RuntimeError)):
                qkv_paged(**{**args, name: bad})
        with pytest.raises(ValueError):
            qkv_paged(**{**args, "q_norm_w": x[0, 0, :8], "k_norm_w": x[0, 0, :8]})
        for t, b in zip((cache.k_pages, cache.v_pages, cache._counts), before):
            assert torch.equal(*(x.view(torch.int16) if x.dtype == bf16 else x for x in (t, b)))
        m(ids[:, 5:6], past_key_values=cache)
        assert cache.lengths.tolist() == [6, 6]


@pytest.mark.parametrize("B", [2, 9])
def test_a_step_that_raises_leaves_the_weights(cdx, B):
    """A bounded cache after a step that raised in its second layer is what it was, and the step done
    again gives what it gives on a cache that never saw it raise."""
    print(f"paged model: raised steps, B={B}", flush=True)
    m = _model(cdx, 64, 4, 2)
    ids = torch.randint(0, 600, (B, 40), generator=torch.Generator().manual_seed(6)).cuda()
    caches = [cdx.PagedKVCache(m.config, B, 32, page_size=16, keep=20, recent=4) for _ in range(2)]

    def interrupted(*a):
        raise KeyboardInterrupt

    with torch.no_grad():
        for c in caches:
            m(ids[:, :28], past_key_values=c)
        for i in range(28, 40):  # (the cache is full, and cut, at the fifth of these)
            before = [t.clone() for t in (caches[0].weights, caches[0].slot_positions, caches[0]._counts)]
            cut = caches[0].longest == caches[0].capacity
            attn = m.layers[1].self_attn
            attn.train(), setattr(attn, "attention_dropout", 0.1)
            with pytest.raises(NotImplementedError):
                m(ids[:, i:i + 1], past_key_values=caches[0])
            attn.eval()
            hook = m.layers[1].mlp.register_forward_pre_hook(interrupted)
            with pytest.raises(KeyboardInterrupt):
                m(ids[:, i:i + 1], past_key_values=caches[0])
            hook.remove()
            if not cut:  # (a cut, which the step done again would make too, stays)
                for t, s in zip((caches[0].weights, caches[0].slot_positions, caches[0]._counts), before):
                    assert torch.equal(t, s), i
            a, b = (m(ids[:, i:i + 1], past_key_values=c).logits for c in caches)
            assert torch.equal(a, b), i
            assert caches[0].longest == caches[1].longest and caches[0].newest == caches[1].newest
            for name in ("weights", "slot_positions", "_counts"):
                assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (i, name)


def test_a_captured_step_of_a_bounded_cache(cdx):
    """Replayed, it leaves the weights and positions that eager steps leave."""
    print("paged model: captured step, bounded cache", flush=True)
    m = _model(cdx, 64, 4, 2)
    B, S, n = 2, 20, 8
    ids = torch.randint(0, 600, (B, S + n), generator=torch.Generator().manual_seed(9)).cuda()
    caches = [cdx.PagedKVCache(m.config, B, 64, page_size=16, keep=32) for _ in range(2)]
    with torch.no_grad():
        for c in caches:
            m(ids[:, :S], past_key_values=c)
        tok = ids[:, S:S + 1].clone()
        state = ("_counts", "weights", "slot_positions")
        before = [getattr(caches[1], name).clone() for name in state]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = m(tok, past_key_values=caches[1]).logits
        for name, t in zip(state, before):
            getattr(caches[1], name).copy_(t)
        for i in range(n):
            tok.copy_(ids[:, S + i:S + i + 1])
            eager = m(tok, past_key_values=caches[0]).logits
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits, eager), i
            for name in state:
                assert torch.equal(*(getattr(c, name) for c in caches)), (i, name)


@pytest.mark.parametrize("keep", [None, 12])
def test_padding_takes_no_room(cdx, keep):
    """Right-padded prompts whose padded length nearly fills the cache: each sequence has room for
    its own tokens, and a bounded cache is cut when its longest sequence fills it."""
    print(f"paged model: padded prompts in a small cache, keep={keep}", flush=True)
    m = _model(cdx, 64, 4, 2, layers=2)
    ids = torch.randint(0, 600, (2, 40), generator=torch.Generator().manual_seed(10)).cuda()
    lens = torch.tensor([5, 3], device="cuda")
    small, wide = (cdx.PagedKVCache(m.config, 2, n, page_size=16, keep=keep) for n in (16, 64))
    with torch.no_grad():
        for c in (small, wide):
            m(ids[:, :15], past_key_values=c, prompt_lengths=lens)
        for i in range(11):
            a, b = (m(ids[:, 15 + i:16 + i], past_key_values=c).logits for c in (small, wide))
            e = errors(a, b)  # (the split of a row's keys follows the capacity)
            assert e["max_rel"] <= MAX_REL and e["rel_rms"] <= REL_RMS, (i, e)
            assert small.lengths.tolist() == [6 + i, 4 + i]
        assert small.longest == 16
        if keep is None:
            with pytest.raises(ValueError, match="full"):
                m(ids[:, 26:27], past_key_values=small)
            assert small.lengths.tolist() == [16, 14]
        else:
            for i in range(10):
                m(ids[:, 26 + i:27 + i], past_key_values=small)
                assert small.longest == int(small.lengths.max()) <= 16
            assert small.lengths.tolist() == [14, 14]
