"""CPU checks of the entry points of several new tokens per sequence: host-side validation rejects bad
calls with the documented status codes before anything is enqueued, and the Python operators
refuse CPU tensors."""

from __future__ import annotations

import math

import pytest
import torch

from test_capi_paged import CDX_EINVAL, CDX_EUNSUPPORTED, CDX_EWORKSPACE, _call, _kw, lib  # noqa: F401


def test_reserve_validation(lib):  # noqa: F811
    call = _call(lib.cdx_paged_reserve,
                 "counts lengths positions B stride rows table table_ld width page free cap count starts new_counts "
                 "new_lengths new_positions new_count slots row_positions stream",
                 [16, 32, 48, 2, 0, 5, 64, 4, 4, 16, 80, 9, 96, 112, 128, 144, 160, 176, 192, 208, None])
    for text, code in [("B=-1", CDX_EINVAL), ("B=0", CDX_EINVAL), ("B=4294967296", CDX_EUNSUPPORTED),
                       ("page=8", CDX_EUNSUPPORTED), ("page=48", CDX_EUNSUPPORTED), ("width=-1", CDX_EINVAL),
                       ("table_ld=3", CDX_EINVAL), ("width=1073741824 table_ld=1073741824", CDX_EUNSUPPORTED),
                       ("rows=-1", CDX_EINVAL), ("rows=2147483647", CDX_EUNSUPPORTED), ("stride=-1", CDX_EINVAL),
                       ("stride=2147483648", CDX_EUNSUPPORTED), ("cap=-1", CDX_EINVAL),
                       ("cap=2147483648", CDX_EUNSUPPORTED), ("counts=None", CDX_EINVAL), ("lengths=None", CDX_EINVAL),
                       ("positions=None", CDX_EINVAL), ("table=None", CDX_EINVAL), ("free=None", CDX_EINVAL),
                       ("count=None", CDX_EINVAL), ("new_count=None", CDX_EINVAL), ("starts=None", CDX_EINVAL),
                       ("new_counts=None", CDX_EINVAL), ("new_lengths=None", CDX_EINVAL),
                       ("new_positions=None", CDX_EINVAL), ("slots=None", CDX_EINVAL),
                       ("row_positions=None", CDX_EINVAL), ("new_counts=16", CDX_EINVAL), ("new_lengths=32", CDX_EINVAL),
                       ("new_positions=48", CDX_EINVAL), ("new_count=96", CDX_EINVAL),
                       ("count=None new_count=None", CDX_EINVAL)]:
        assert call(**_kw(text)) == code, text


def test_truncate_validation(lib):  # noqa: F811
    call = _call(lib.cdx_paged_truncate,
                 "to lengths positions B table table_ld width page free cap count new_lengths new_positions new_count "
                 "stream",
                 [16, 32, 48, 2, 64, 4, 4, 16, 80, 9, 96, 112, 128, 144, None])
    for text, code in [("B=-1", CDX_EINVAL), ("B=0", CDX_EINVAL), ("B=4294967296", CDX_EUNSUPPORTED),
                       ("page=8", CDX_EUNSUPPORTED), ("width=-1", CDX_EINVAL), ("table_ld=3", CDX_EINVAL),
                       ("cap=-1", CDX_EINVAL), ("cap=2147483648", CDX_EUNSUPPORTED), ("to=None", CDX_EINVAL),
                       ("lengths=None", CDX_EINVAL), ("positions=None", CDX_EINVAL), ("table=None", CDX_EINVAL),
                       ("free=None", CDX_EINVAL), ("count=None", CDX_EINVAL), ("new_lengths=None", CDX_EINVAL),
                       ("new_positions=None", CDX_EINVAL), ("new_count=None", CDX_EINVAL),
                       ("new_lengths=32", CDX_EINVAL), ("new_lengths=16", CDX_EINVAL), ("new_positions=48", CDX_EINVAL),
                       ("new_count=96", CDX_EINVAL)]:
        assert call(**_kw(text)) == code, text


def test_chunk_append_validation(lib):  # noqa: F811
    call = _call(lib.cdx_paged_chunk_append_fwd,
                 "qkv fp32 ld rows nq nkv hd qn kn eps cos n_pos slots positions num_pages page k_pages v_pages q "
                 "stream",
                 [16, 0, 512, 5, 4, 2, 64, None, None, 1e-6, 16, 8, 16, 16, 9, 16, 16, 16, 16, None])
    for text, code in [("nkv=0", CDX_EINVAL), ("num_pages=-1", CDX_EINVAL), ("num_pages=4294967296", CDX_EUNSUPPORTED),
                       ("hd=12", CDX_EUNSUPPORTED), ("hd=136", CDX_EUNSUPPORTED), ("hd=0", CDX_EUNSUPPORTED),
                       ("page=8", CDX_EUNSUPPORTED), ("rows=-1", CDX_EINVAL), ("rows=2147483648", CDX_EUNSUPPORTED),
                       ("k_pages=None", CDX_EINVAL), ("v_pages=None", CDX_EINVAL), ("k_pages=24", CDX_EUNSUPPORTED),
                       ("nq=3", CDX_EINVAL), ("nq=0", CDX_EINVAL), ("n_pos=-1", CDX_EINVAL), ("qn=16", CDX_EINVAL),
                       ("ld=504", CDX_EINVAL), ("ld=516", CDX_EUNSUPPORTED), ("n_pos=0", CDX_EINVAL),
                       ("cos=None", CDX_EINVAL), ("q=None", CDX_EINVAL), ("slots=None", CDX_EINVAL),
                       ("positions=None", CDX_EINVAL), ("qkv=18", CDX_EUNSUPPORTED), ("qn=8 kn=16", CDX_EUNSUPPORTED),
                       ("nq=65536 ld=5000000", CDX_EUNSUPPORTED), ("rows=0 qkv=None q=None", 0)]:
        assert call(**_kw(text)) == code, text
    assert call(eps=-1.0) == CDX_EINVAL and call(eps=math.nan) == CDX_EINVAL


def test_chunk_attention_validation(lib):  # noqa: F811
    call = _call(lib.cdx_paged_chunk_attention_fwd,
                 "q rows B nq nkv hd k_pages v_pages table table_ld width num_pages page starts counts lengths most "
                 "scale out work work_bytes stream",
                 [16, 40, 2, 4, 2, 64, 16, 16, 16, 400, 400, 900, 16, 16, 16, 16, 40, 0.125, 16, 16, 1 << 30, None])
    for text, code in [("nkv=0", CDX_EINVAL), ("width=-1", CDX_EINVAL), ("num_pages=-1", CDX_EINVAL),
                       ("table_ld=3", CDX_EINVAL), ("hd=12", CDX_EUNSUPPORTED), ("hd=136", CDX_EUNSUPPORTED),
                       ("page=8", CDX_EUNSUPPORTED), ("page=512", CDX_EUNSUPPORTED),
                       ("num_pages=4294967296", CDX_EUNSUPPORTED), ("B=4294967296", CDX_EUNSUPPORTED),
                       ("B=-1", CDX_EINVAL), ("rows=-1", CDX_EINVAL), ("rows=2147483648", CDX_EUNSUPPORTED),
                       ("most=-1", CDX_EINVAL), ("nq=3", CDX_EINVAL), ("nq=0", CDX_EINVAL), ("width=0", CDX_EINVAL),
                       ("num_pages=0", CDX_EINVAL), ("B=0", CDX_EINVAL), ("q=None", CDX_EINVAL),
                       ("k_pages=None", CDX_EINVAL), ("v_pages=None", CDX_EINVAL), ("table=None", CDX_EINVAL),
                       ("starts=None", CDX_EINVAL), ("counts=None", CDX_EINVAL), ("lengths=None", CDX_EINVAL),
                       ("out=None", CDX_EINVAL), ("out=24", CDX_EUNSUPPORTED), ("k_pages=24", CDX_EUNSUPPORTED),
                       ("work_bytes=64", CDX_EWORKSPACE), ("work=None", CDX_EWORKSPACE), ("rows=0 q=None", 0)]:
        assert call(**_kw(text)) == code, text
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=scale) == CDX_EINVAL
    need = lib.cdx_paged_chunk_attention_workspace_bytes
    assert need(40, 2, 4, 2, 64, 6400, 40) > 0 and need(0, 2, 4, 2, 64, 6400, 40) == 0
    assert need(40, 2, 3, 2, 64, 6400, 40) == 0 and need(40, 2, 4, 2, 64, 6400, -1) == 0


def test_operators_refuse_cpu_tensors():
    import complexity_deep as cdx
    i32 = {"dtype": torch.int32}
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    one, table = torch.zeros(1, **i32), torch.zeros(1, 2, **i32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        cdx.paged_reserve(one, one, one, table, 16, 3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        cdx.paged_truncate(one, one, one, table, 16, one, one)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        cdx.paged_chunk_append(torch.zeros(3, 512, dtype=torch.bfloat16), k, k, torch.zeros(3, dtype=torch.int64),
                               torch.zeros(3, **i32), 4, torch.zeros(8, 32, 2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        cdx.paged_chunk_attention(torch.zeros(3, 4, 64, dtype=torch.bfloat16), k, k, table, one, one, one)


def test_cache_refuses_what_it_cannot_take():
    """Before any memory is taken or a kernel called."""
    import complexity_deep as cdx
    cfg = cdx.ComplexityConfig.complexity_tiny()
    for bad in (dict(pages=0), dict(pages=-3), dict(pages=2.5), dict(pages=True), dict(pages=8, keep=10)):
        with pytest.raises(ValueError, match="PagedKVCache"):
            cdx.PagedKVCache(cfg, 2, 40, device="cpu", **bad)
    bounded = cdx.PagedKVCache(cfg, 2, 40, keep=10, device="cpu")
    with pytest.raises(ValueError, match="bounded"):
        bounded.begin(2, 3, token_counts=[3, 3])
    with pytest.raises(ValueError, match="bounded"):
        bounded.truncate([1, 1])
    c = cdx.PagedKVCache(cfg, 2, 40, page_size=16, device="cpu")
    for args in ((3, [1, 1], False), (2, [1, 1, 1], False), (2, [3, 1], False), (2, [-1, 1], False), (3, [2, 2], True),
                 (0, [0, 0], False)):
        with pytest.raises(ValueError, match="PagedKVCache"):
            c.begin(args[0] if args[0] == 3 and not args[2] else 2, 3 if args[2] else min(args[0], 2),
                    token_counts=args[1], packed=args[2])
    with pytest.raises(ValueError, match="full"):
        c.begin(2, 49, token_counts=[49, 1])
    assert c.lengths.tolist() == [0, 0] and c.newest == 0


def test_cache_without_a_pool_is_cut_anywhere():
    import complexity_deep as cdx
    c = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 3, 40, page_size=16, device="cpu")
    c.begin(3, 9, torch.tensor([9, 4, 0]))
    c.begin(3, 1)
    c.truncate(torch.tensor([5, 50, 0]))
    assert c.lengths.tolist() == [5, 5, 0] and c.positions.tolist() == [4, 4, -1] and c.longest == 5
    c.begin(3, 1)
    assert c.lengths.tolist() == [6, 6, 1] and c.longest == c.newest == 6
    c.release([0])
    assert c.lengths.tolist() == [0, 6, 1] and c.longest == 6
    with pytest.raises(IndexError):
        c.release([3])
    c.release([1, 2])
    assert c.lengths.tolist() == [0, 0, 0] and c.newest == 0 and c.positions.tolist() == [-1, -1, -1]
    c.begin(3, 4)  # prompts again
    assert c.lengths.tolist() == [4, 4, 4] and c.prompt
