"""sample_tokens against a plain form by sorting, in 64 bits (tests/_paged.py): token for token."""

from __future__ import annotations

import math

import pytest
import torch

import _paged as ref

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def _logits(B, V, seed, dtype, kind="model"):
    g = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(B, V, generator=g)
    if kind == "model":
        x.scatter_add_(1, torch.randint(0, V, (B, 8), generator=g), 4 + 3 * torch.rand(B, 8, generator=g))
    if kind == "ties":
        x = torch.randint(-2, 3, (B, V), generator=g).float()
    if kind == "flat":
        x = torch.zeros(B, V)
    if kind == "masked":
        x = torch.where(torch.rand(B, V, generator=g) < 0.9, -math.inf, x)
        x[:, V // 2] = 0.5
    if kind == "tiny":  # values around 0 among others, too many for the lists at the larger sizes
        pool = torch.tensor([0.0, -0.0, 1e-9, -1e-9, 3e-8, -5e-8, 2.0 ** -24, -2.0 ** -24, 2.0 ** -23])
        x = torch.where(torch.rand(B, V, generator=g) < 0.3, pool[torch.randint(0, 9, (B, V), generator=g)], x)
    if kind == "odd":
        pool = torch.tensor([math.nan, -math.inf, 0.0, -0.0, 1.0, -1.0, 1e-30, -3e38])
        x = pool[torch.randint(0, len(pool), (B, V), generator=g)]
    return x.to(dtype), torch.rand(B, generator=g)


def _check(cdx, x, u, **s):
    got = cdx.sample_tokens(x.cuda(), u.cuda(), **{k: v.cuda() if torch.is_tensor(v) else v for k, v in s.items()})
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    for b in range(x.shape[0]):
        # (Settings are taken in fp32, as numbers and as tensors.)
        row = {k: float(v[b] if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32)) for k, v in s.items()}
        if "top_k" in s:
            row["top_k"] = int(s["top_k"][b] if torch.is_tensor(s["top_k"]) else s["top_k"])
        assert int(got[b]) == ref.sample(x[b], float(u[b]), **row), f"row {b}: {row}"
    return got


SETTINGS = [{}, {"temperature": 0.0}, {"temperature": 0.7, "top_k": 50, "top_p": 0.9}, {"top_p": 0.5}, {"top_k": 1},
            {"min_p": 0.05, "temperature": 1.5}, {"top_k": 7, "min_p": 0.2, "top_p": 0.3}, {"top_p": 0.0},
            {"min_p": 1.0}, {"temperature": 1e-3}, {"temperature": 1e30, "top_p": 0.95}, {"top_k": 1000, "top_p": 0.99}]


@pytest.mark.parametrize("kind", ["model", "ties", "flat", "masked", "tiny", "odd"])
@pytest.mark.parametrize("V,dtype", [(1, bf16), (2, torch.float32), (50, bf16), (511, bf16), (512, torch.float32),
                                     (1000, torch.float32), (5003, bf16)])
def test_sample(cdx, V, dtype, kind):
    print(f"sample V={V} {dtype} {kind}", flush=True)
    for i, s in enumerate(SETTINGS):
        x, u = _logits(5, V, 31 * V + i, dtype, kind)
        u[0], u[1] = 0.0, 1 - 2.0 ** -24
        _check(cdx, x, u, **s)


@pytest.mark.parametrize("V,dtype,B", [(32000, torch.float32, 3), (100000, bf16, 3), (100003, bf16, 2),
                                       (131072, torch.float32, 2), (1 << 20, bf16, 1)])
def test_sample_large_vocabularies(cdx, V, dtype, B):
    print(f"sample V={V} {dtype} B={B}", flush=True)
    for i, s in enumerate(({}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.95}, {"temperature": 1.3, "min_p": 0.01},
                           {"top_k": 5000, "temperature": 2.0}, {"top_k": V // 2, "top_p": 0.999}, {"temperature": 0},
                           {"temperature": 30.0, "top_p": 0.6}, {"top_k": 1000})):
        x, u = _logits(B, V, V + i, dtype, "tiny" if i == 2 else "model")
        _check(cdx, x, u, **s)


def test_sample_settings_of_each_row(cdx):
    print("sample: settings by row", flush=True)
    B, V = 12, 3001
    x, u = _logits(B, V, 5, bf16)
    g = torch.Generator().manual_seed(9)
    _check(cdx, x, u, temperature=torch.tensor([0.0, 0.5, 1, 2, -1, 1e-3, 1, 1, 1, 1, 1, 0.8]),
           top_k=torch.tensor([0, 1, 5, 3000, 3001, 40000, -4, 100, 0, 0, 9, 50], dtype=torch.int32),
           top_p=torch.tensor([1, 0.9, 0, 1.5, -1, 0.5, 0.999, 0.1, 1, 1, 0.7, 0.9]),
           min_p=torch.tensor([0, 0.1, 0, 0, 0, 0, 0.3, -1, 2.0, 1, 0, 0.02]))
    many = torch.rand(B, 2, generator=g)
    _check(cdx, x, u, temperature=many[:, 0].contiguous() + 0.1, top_p=many[:, 1])  # (a strided tensor)


def test_sample_ties_stay_in_the_order_of_their_indices(cdx):
    print("sample: equal logits", flush=True)
    V = 4096
    x = torch.zeros(64, V, dtype=bf16)
    u = torch.arange(64) / 64
    # Half of equal tokens: those before which the sum is at most half, i.e. V/2 + 1 of them.
    got = _check(cdx, x, u, top_p=0.5)
    assert got.tolist() == [int(i / 64 * (V // 2 + 1)) for i in range(64)]
    assert _check(cdx, x, u, top_k=3).tolist() == [i * V // 64 for i in range(64)]  # all tie with the third
    assert _check(cdx, x, u, temperature=0).tolist() == [0] * 64


def test_sample_infinities(cdx):
    print("sample: infinite rows", flush=True)
    x = torch.tensor([[-math.inf] * 4, [math.nan] * 4, [1, math.inf, 2, math.inf],
                      [math.nan, -math.inf, -3e38, math.nan], [-math.inf, 0, -math.inf, 0]])
    u = torch.tensor([0.3, 0.3, 0.7, 0.99, 0.5])
    for s in ({}, {"temperature": 0.0}, {"top_k": 2, "top_p": 0.9, "min_p": 0.1}):
        got = _check(cdx, x, u, **s)
        assert got[:2].tolist() == [-1, -1] and int(got[3]) == 2
    assert cdx.sample_tokens(x.cuda(), u.cuda()).tolist() == [-1, -1, 3, 2, 3]
    # A temperature without bounds: every finite logit weighs the same.
    row = torch.full((5,), math.inf, device="cuda")
    assert cdx.sample_tokens(x.cuda(), u.cuda(), temperature=row).tolist()[4] == 3


def test_sample_uniforms_outside_their_range(cdx):
    print("sample: u of 1, nan, below 0", flush=True)
    x = torch.zeros(4, 10, device="cuda")
    u = torch.tensor([1.0, math.nan, -0.5, 7.0], device="cuda")
    assert cdx.sample_tokens(x, u).tolist() == [9, 0, 0, 9]


def test_sample_strided_rows(cdx):
    """The last position's logits of [B, S, V], and rows at any byte."""
    print("sample: strided and unaligned rows", flush=True)
    for dtype in (bf16, torch.float32):
        for V in (1000, 1001):
            full = torch.randn(6, 3, V + 2, device="cuda").to(dtype)
            u = torch.rand(6, device="cuda")
            for view in (full[:, -1, :V], full[:, 1, 1:V + 1], full[:, 0, 2:], full.transpose(1, 2)[:, :V, 0]):
                for s in ({}, {"top_k": 20, "top_p": 0.8}, {"min_p": 0.1}):
                    a = cdx.sample_tokens(view, u, **s)
                    assert torch.equal(a, cdx.sample_tokens(view.clone(), u, **s))
                    assert int(a[2]) == ref.sample(view[2], float(u[2]), **{k: float(torch.tensor(v)) if k != "top_k"
                                                                            else v for k, v in s.items()})


def test_sample_draws_what_the_weights_say(cdx):
    """Evenly spaced numbers draw each token as often as its share of the sum, to one."""
    print("sample: shares", flush=True)
    n, V = 4096, 37
    x = torch.randn(1, V, device="cuda").float()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(cdx.sample_tokens(x.expand(n, V).contiguous(), u), minlength=V).double().cpu()
    share = torch.softmax(x[0].double().cpu(), 0) * n
    assert bool(((got - share).abs() <= 1.0).all())


def test_sample_in_a_graph_and_on_a_stream(cdx):
    print("sample: captured", flush=True)
    B, V = 4, 20000
    x, u = torch.zeros(B, V, device="cuda", dtype=bf16), torch.zeros(B, device="cuda")
    cdx.sample_tokens(x, u, top_k=40, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cdx.sample_tokens(x, u, top_k=40, top_p=0.9)
    side = torch.cuda.Stream()
    for i in range(4):
        new, uniform = _logits(B, V, i, bf16)
        x.copy_(new), u.copy_(uniform)
        graph.replay()
        eager = cdx.sample_tokens(x, u, top_k=40, top_p=0.9)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = cdx.sample_tokens(x, u, top_k=40, top_p=0.9)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, eager) and torch.equal(out, other)


def test_sample_refusals(cdx):
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    t = torch.ones(2, device="cuda")
    for args, s in [((x.half(), u), {}), ((x[0], u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x.cpu(), u), {}),
                    ((x, u.cpu()), {}), ((x[:, :0], u), {}), ((x, u), {"temperature": -1.0}),
                    ((x, u), {"temperature": math.nan}), ((x, u), {"temperature": math.inf}), ((x, u), {"top_k": -1}),
                    ((x, u), {"top_k": 1.5}), ((x, u), {"top_p": 1.1}), ((x, u), {"top_p": -0.1}),
                    ((x, u), {"min_p": 2}),
                    ((x, u), {"min_p": math.nan}), ((x, u), {"temperature": t[:1]}), ((x, u), {"top_k": t}),
                    ((x, u), {"top_p": t.double()}), ((x, u), {"min_p": t.cpu()}),
                    ((torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1]), {})]:
        with pytest.raises((ValueError, RuntimeError)):
            cdx.sample_tokens(*args, **s)
    assert cdx.sample_tokens(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [bf16, torch.float32])
def test_sample_top_k_that_ends_among_values_around_zero(cdx, dtype):
    """The k-th largest logit lies among values of less than 2^-24, too many for the lists, and top-p
    cuts above them: its total holds what top-k kept of them, and nothing else."""
    print(f"sample: top-k ends around zero, {dtype}", flush=True)
    V, B = 32768, 12
    row = torch.tensor([1e-9, -1e-9]).repeat(V // 2)
    row[1000:9000:1000] = 9 - torch.arange(8) / 16
    x = row.to(dtype).expand(B, V).contiguous()
    u = (torch.arange(B) + 0.5) / B
    for s in ({"top_k": 1000, "top_p": 0.5}, {"top_k": 20000, "top_p": 0.5}, {"top_k": 1000, "top_p": 0.9},
              {"top_k": 1000, "top_p": 0.5, "min_p": 0.7}, {"top_k": 1000, "top_p": 0.7, "temperature": 0.5}):
        _check(cdx, x, u, **s)


def test_sample_of_many_rows(cdx):
    """More rows than one launch has threads for, with settings of each row."""
    print("sample: 2^22 + 5 rows", flush=True)
    B, V = (1 << 22) + 5, 9
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype in (bf16, torch.float32):
        x = torch.rand(B, V, generator=g, device="cuda").argsort(-1).to(dtype)  # (no ties)
        u = torch.rand(B, generator=g, device="cuda")
        best = x.argmax(-1)
        zero, one = torch.zeros(B, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
        assert torch.equal(cdx.sample_tokens(x, u, temperature=0), best)
        assert torch.equal(cdx.sample_tokens(x, u, top_k=one), best)
        assert torch.equal(cdx.sample_tokens(x, u, top_p=zero), best)
        assert torch.equal(cdx.sample_tokens(x, u, min_p=zero + 1), best)
        assert torch.equal(cdx.sample_tokens(x, u, temperature=zero), best)
        some = cdx.sample_tokens(x, u)
        for part in (slice(0, 1000), slice(B - 1000, B)):
            assert torch.equal(cdx.sample_tokens(x[part], u[part]), some[part])
