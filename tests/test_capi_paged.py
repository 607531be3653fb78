"""CPU checks of the paged and sampling entry points: host-side validation rejects bad calls with
the documented status codes before anything is enqueued (so these run without a GPU), and the
Python operators refuse CPU tensors."""

from __future__ import annotations

import math

import pytest
import torch

CDX_EINVAL, CDX_EUNSUPPORTED, CDX_EWORKSPACE = -1, -2, -4


@pytest.fixture(scope="module")
def lib():
    from complexity_deep import _native
    if not _native.LIB_PATH.exists():
        import importlib.util
        from pathlib import Path
        src = Path(__file__).resolve().parents[1] / "complexity-deep_amd" / "build_native.py"
        spec = importlib.util.spec_from_file_location("build_native", src)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.build()
    return _native.lib()


def _call(fn, names, ok):
    def call(**kw):
        args = dict(zip(names.split(), ok))
        assert set(kw) <= set(args), kw
        args.update(kw)
        return fn(*args.values())
    return call


CACHE = [("nkv=0", CDX_EINVAL), ("width=-1", CDX_EINVAL), ("num_pages=-1", CDX_EINVAL), ("table_ld=3", CDX_EINVAL),
         ("hd=12", CDX_EUNSUPPORTED), ("hd=136", CDX_EUNSUPPORTED), ("hd=0", CDX_EUNSUPPORTED),
         ("page=8", CDX_EUNSUPPORTED), ("page=48", CDX_EUNSUPPORTED), ("page=512", CDX_EUNSUPPORTED),
         ("num_pages=4294967296", CDX_EUNSUPPORTED), ("width=1073741824 table_ld=1073741824", CDX_EUNSUPPORTED),
         ("B=4294967296", CDX_EUNSUPPORTED), ("B=-1", CDX_EINVAL), ("k_pages=None", CDX_EINVAL),
         ("v_pages=None", CDX_EINVAL), ("k_pages=24", CDX_EUNSUPPORTED), ("v_pages=8", CDX_EUNSUPPORTED),
         ("table=None", CDX_EINVAL), ("lengths=None", CDX_EINVAL)]


def _kw(text):
    return {k: None if v == "None" else int(v) for k, v in (p.split("=") for p in text.split())}


def test_append_validation(lib):
    call = _call(lib.cdx_paged_append_fwd,
                 "qkv fp32 ld B nq nkv hd qn kn eps cos n_pos lengths positions table table_ld width num_pages page "
                 "k_pages v_pages q stream",
                 [16, 0, 512, 2, 4, 2, 64, None, None, 1e-6, 16, 8, 16, 16, 16, 4, 4, 9, 16, 16, 16, 16, None])
    for text, code in CACHE:
        assert call(**_kw(text)) == code, text
    assert call(nq=3) == CDX_EINVAL and call(nq=0) == CDX_EINVAL and call(n_pos=-1) == CDX_EINVAL
    assert call(qn=16) == CDX_EINVAL and call(eps=-1.0) == CDX_EINVAL and call(eps=math.nan) == CDX_EINVAL
    assert call(ld=504) == CDX_EINVAL and call(ld=516) == CDX_EUNSUPPORTED
    assert call(n_pos=0) == CDX_EINVAL and call(cos=None) == CDX_EINVAL and call(q=None) == CDX_EINVAL
    assert call(positions=None) == CDX_EINVAL and call(qkv=18) == CDX_EUNSUPPORTED
    assert call(qn=8, kn=16) == CDX_EUNSUPPORTED
    assert call(B=0, qkv=None, q=None) == 0
    assert lib.cdx_last_error() == b""


def test_projection_and_append_validation(lib):
    call = _call(lib.cdx_qkv_paged_fwd,
                 "x ldx xn xeps mu ldmu w w_mu ldw B H nq nkv hd qn kn eps cos n_pos lengths positions table table_ld "
                 "width num_pages page k_pages v_pages q work work_bytes stream",
                 [16, 256, None, 0.0, 16, 256, 16, 16, 512, 2, 256, 4, 2, 64, None, None, 1e-6, 16, 8, 16, 16, 16, 4, 4,
                  9, 16, 16, 16, 16, 16, 1 << 20, None])
    for text, code in CACHE:
        assert call(**_kw(text)) == code, text
    assert call(H=0) == CDX_EINVAL and call(H=96) == CDX_EUNSUPPORTED and call(ldx=128) == CDX_EINVAL
    assert call(ldw=128) == CDX_EINVAL and call(ldmu=128) == CDX_EINVAL and call(ldx=260) == CDX_EUNSUPPORTED
    assert call(w_mu=None) == CDX_EINVAL and call(x=None) == CDX_EINVAL and call(work=None) == CDX_EINVAL
    assert call(work_bytes=4095) == CDX_EWORKSPACE and call(x=18) == CDX_EUNSUPPORTED
    assert call(B=9, xn=16) == CDX_EUNSUPPORTED  # the norm is folded for up to 8 rows
    assert call(xn=16, xeps=-1.0) == CDX_EINVAL and call(qn=16) == CDX_EINVAL and call(n_pos=0) == CDX_EINVAL
    assert call(q=None) == CDX_EINVAL and call(B=0) == 0


def test_write_validation(lib):
    call = _call(lib.cdx_paged_write,
                 "k v B nkv S hd lengths table table_ld width num_pages page k_pages v_pages stream",
                 [16, 16, 2, 2, 5, 64, 16, 16, 4, 4, 9, 16, 16, 16, None])
    for text, code in CACHE:
        assert call(**_kw(text)) == code, text
    assert call(S=-1) == CDX_EINVAL and call(k=None) == CDX_EINVAL and call(v=8) == CDX_EUNSUPPORTED
    assert call(S=1 << 31) == CDX_EUNSUPPORTED and call(B=100000, S=1 << 24) == CDX_EUNSUPPORTED
    assert call(B=0) == 0 and call(S=0, k=None) == 0 and call(width=0, table=None) == 0 and call(num_pages=0) == 0


def test_attention_validation(lib):
    call = _call(lib.cdx_paged_attention_fwd,
                 "q B nq nkv hd k_pages v_pages table table_ld width num_pages page lengths scale out w_in w_out work "
                 "work_bytes stream",
                 [16, 2, 4, 2, 64, 16, 16, 16, 4, 4, 9, 16, 16, 0.125, 16, None, None, 16, 1 << 30, None])
    for text, code in CACHE:
        assert call(**_kw(text)) == code, text
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=scale) == CDX_EINVAL
    assert call(nq=3) == CDX_EINVAL and call(nq=0) == CDX_EINVAL and call(w_in=16) == CDX_EINVAL
    assert call(w_out=16) == CDX_EINVAL and call(width=0) == CDX_EINVAL and call(num_pages=0) == CDX_EINVAL
    assert call(q=None) == CDX_EINVAL and call(out=24) == CDX_EUNSUPPORTED
    assert call(B=0) == 0
    need = lib.cdx_paged_attention_workspace_bytes(2, 4, 2, 64, 64, 1)
    assert need >= 2 * 4 * 64 * 4  # the scores
    assert call(w_in=16, w_out=16, work_bytes=need - 1) == CDX_EWORKSPACE
    assert call(w_in=16, w_out=16, work=None) == CDX_EWORKSPACE
    # A long table of one sequence is split: partial sums.
    assert lib.cdx_paged_attention_workspace_bytes(1, 4, 2, 64, 1 << 16, 0) > 0
    assert lib.cdx_paged_attention_workspace_bytes(0, 4, 2, 64, 64, 1) == 0
    assert lib.cdx_paged_attention_workspace_bytes(1, 3, 2, 64, 64, 1) == 0


def test_evict_validation(lib):
    call = _call(lib.cdx_paged_evict,
                 "layers B nkv hd lengths positions table table_ld width num_pages page k_pages v_pages w sp keep "
                 "recent n_len n_w n_sp work work_bytes stream",
                 [3, 2, 2, 64, 16, 16, 16, 4, 4, 9, 16, 16, 16, 16, 16, 8, 4, 32, 32, 32, 16, 1 << 20, None])
    for text, code in CACHE:
        assert call(**_kw(text)) == code, text
    assert call(layers=-1) == CDX_EINVAL and call(keep=0) == CDX_EINVAL and call(recent=-1) == CDX_EINVAL
    assert call(recent=9) == CDX_EINVAL and call(layers=1 << 17) == CDX_EUNSUPPORTED
    for name in ("positions", "w", "sp", "n_len", "n_w", "n_sp", "work"):
        assert call(**{name: None}) == CDX_EINVAL, name
    assert call(n_w=16) == CDX_EINVAL and call(n_sp=16) == CDX_EINVAL and call(n_len=16) == CDX_EINVAL  # in place
    assert lib.cdx_paged_evict_workspace_bytes(3, 2, 2, 64, 8) == 12 * (1 + 2 * 8) * 4
    assert lib.cdx_paged_evict_workspace_bytes(3, 2, 2, 64, 60) == 12 * (1 + 2 * 4) * 4
    assert lib.cdx_paged_evict_workspace_bytes(3, 2, 2, 64, 64) == 12 * 4
    assert call(work_bytes=12 * 17 * 4 - 1) == CDX_EWORKSPACE
    assert call(layers=0) == 0 and call(B=0) == 0 and call(width=0, table=None) == 0


def test_sample_validation(lib):
    call = _call(lib.cdx_sample_tokens, "logits fp32 ld B V u t t1 k k1 p p1 m m1 tokens stream",
                 [16, 0, 100, 3, 100, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, None])
    assert call(B=-1) == CDX_EINVAL and call(V=0) == CDX_EINVAL and call(ld=99) == CDX_EINVAL
    assert call(V=(1 << 20) + 1, ld=1 << 21) == CDX_EUNSUPPORTED and call(B=1 << 31) == CDX_EUNSUPPORTED
    for bad in ({"t1": -1.0}, {"t1": math.nan}, {"k1": -1}, {"p1": 1.5}, {"p1": -0.5}, {"p1": math.nan}, {"m1": 2.0},
                {"m1": math.nan}, {"logits": None}, {"u": None}, {"tokens": None}):
        assert call(**bad) == CDX_EINVAL, bad
    assert call(B=0, logits=None) == 0


def test_cpu_tensors_raise():
    import complexity_deep as cdx
    bf = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: cdx.paged_attention(q, bf, bf, table, lens),
                 lambda: cdx.paged_write(torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16),
                                         torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), bf, bf, table, lens),
                 lambda: cdx.paged_qkv_append(torch.zeros(1, 512, dtype=torch.bfloat16), bf, bf, table, lens, lens, 4,
                                              torch.zeros(4, 32, 2)),
                 lambda: cdx.paged_evict(bf, bf, table, lens, lens, torch.zeros(1, 2, 32),
                                         torch.zeros(1, 2, 32, dtype=torch.int32), 4, 2),
                 lambda: cdx.sample_tokens(torch.zeros(2, 9), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_cache_arguments():
    """Refused before any memory is taken (so also here)."""
    import complexity_deep as cdx
    cfg = cdx.ComplexityConfig.complexity_tiny()
    for bad in (dict(page_size=17), dict(max_length=0), dict(batch_size=-1), dict(keep=40), dict(keep=-1),
                dict(keep=8, recent=9), dict(keep=8, recent=-1)):
        with pytest.raises(ValueError, match="PagedKVCache"):
            cdx.PagedKVCache(cfg, **{**dict(batch_size=2, max_length=40, device="cpu"), **bad})
    with pytest.raises(ValueError, match="prompt_lengths"):
        cdx.PagedKVCache(cfg, 2, 40, device="cpu").begin(2, 3, torch.tensor([1.0, 2.0]))


def test_cache_counts():
    """The counts of a cache, which any device can hold."""
    import complexity_deep as cdx
    cfg = cdx.ComplexityConfig.complexity_tiny()
    c = cdx.PagedKVCache(cfg, 3, 20, page_size=16, keep=10, device="cpu")
    assert c.capacity == 32 and len(c) == 6 and c.recent == 5 and c.block_table.tolist() == [[0, 1], [2, 3], [4, 5]]
    c.begin(3, 7, torch.tensor([7, 9, -2]))
    assert c.lengths.tolist() == [7, 7, 0] and c.positions.tolist() == [6, 6, -1] and c.prompt
    assert c.slot_positions[2, :, 1, :9].tolist() == [[0, 1, 2, 3, 4, 5, 6, -1, -1],
                                                      [0, 1, 2, 3, 4, 5, 6, -1, -1], [-1] * 9]
    c.begin(3, 1)
    assert c.lengths.tolist() == [8, 8, 1] and c.positions.tolist() == [7, 7, 0] and not c.prompt
    assert c.longest == c.newest == 8 and c.slot_positions[0, :, 0, 7].tolist() == [7, 7, -1]
    assert c.slot_positions[5, 2, 1, :2].tolist() == [0, -1]
    for args in ((2, 1), (3, 2), (3, 1, torch.tensor([1, 1, 1]))):
        with pytest.raises(ValueError, match="PagedKVCache"):
            c.begin(*args)
    with pytest.raises(IndexError):
        c[6]
    c.reset()
    assert c.lengths.tolist() == [0, 0, 0] and c.newest == 0 and bool((c.slot_positions == -1).all())
    full = cdx.PagedKVCache(cfg, 1, 16, page_size=16, device="cpu")
    full.begin(1, 16)
    with pytest.raises(ValueError, match="full"):
        full.begin(1, 1)


def test_a_cache_made_under_inference_mode():
    import complexity_deep as cdx
    with torch.inference_mode():
        c = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 2, 20, page_size=16, keep=10, device="cpu")
    c.begin(2, 5)
    with torch.inference_mode():
        c.begin(2, 1)
    c.begin(2, 1)
    assert c.lengths.tolist() == [7, 7] and not c.lengths.is_inference()


@pytest.mark.parametrize("keep", [None, 8])
def test_a_cache_is_full_when_its_longest_sequence_is(keep):
    """Not when the padded prompts and the steps after them are as long as the capacity."""
    import complexity_deep as cdx
    c = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 3, 16, page_size=16, keep=keep, device="cpu")
    c.begin(3, 15, torch.tensor([3, 0, 6]))
    assert (c.longest, c.newest) == (6, 15)
    for i in range(10):
        c.begin(3, 1)
        assert c.lengths.tolist() == [4 + i, 1 + i, 7 + i] and c.longest == 7 + i
    if keep is None:
        with pytest.raises(ValueError, match="full"):
            c.begin(3, 1)
    assert c.lengths.tolist() == [13, 10, 16] and c.longest == 16


@pytest.mark.parametrize("bad", [dict(keep=10.5), dict(keep=True), dict(keep=8, recent=2.5), dict(keep=8, recent=True)])
def test_a_bound_that_is_no_integer_is_refused_at_once(bad):
    """Not by the first cut, in the middle of a generation."""
    import complexity_deep as cdx
    with pytest.raises(ValueError, match="PagedKVCache"):
        cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 2, 40, device="cpu", **bad)


def test_a_narrower_block_table_is_refused():
    """Tokens past its pages would be dropped, and nobody told."""
    import complexity_deep as cdx
    c = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 2, 40, page_size=16, device="cpu")
    whole = c.block_table
    c.block_table = whole[:, :2]
    with pytest.raises(ValueError, match="block table"):
        c.begin(2, 5)
    c.block_table = torch.cat([whole, whole], 1)  # (a wider one is no harm)
    c.begin(2, 5)
    c.block_table = whole[:, :2]
    with pytest.raises(ValueError, match="block table"):
        c.begin(2, 1)
    assert c.lengths.tolist() == [5, 5] and c.longest == 5


def test_whole_numbers_of_other_types_are_bounds():
    import numpy as np
    import complexity_deep as cdx
    for keep, recent in ((np.int64(8), np.int32(3)), (8.0, 3.0)):
        c = cdx.PagedKVCache(cdx.ComplexityConfig.complexity_tiny(), 2, 40, keep=keep, recent=recent, device="cpu")
        assert (c.keep, c.recent) == (8, 3) and type(c.keep) is type(c.recent) is int


def test_more_threads_than_a_launch_has_are_refused(lib):
    """Where a call is not cut into several launches (operands of hundreds of gigabytes)."""
    write = _call(lib.cdx_paged_write,
                  "k v B nkv S hd lengths table table_ld width num_pages page k_pages v_pages stream",
                  [16, 16, 100000, 2, 1 << 20, 64, 16, 16, 4, 4, 9, 16, 16, 16, None])
    assert write() == CDX_EUNSUPPORTED
    attend = _call(lib.cdx_paged_attention_fwd,
                   "q B nq nkv hd k_pages v_pages table table_ld width num_pages page lengths scale out w_in w_out work "
                   "work_bytes stream",
                   [16, 100000, 4, 2, 64, 16, 16, 16, 4096, 4096, 9, 16, 16, 0.125, 16, 16, 16, 16, 1 << 60, None])
    assert attend() == CDX_EUNSUPPORTED
