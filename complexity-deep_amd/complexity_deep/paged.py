"""The paged KV cache of a generation on the gfx950 kernels: its append, the attention of one new
token over it, and its bound by accumulated attention weight.

The reference keeps k and v of a layer as one tensor each, which every step concatenates into a
longer one, and its cached step keeps the top-left causal mask (core/attention.py:157-175).  Here
k and v lie in pages of a pool, [pages, nkv, page_size, D], a block table names the pages of each
sequence, and a step's one token attends to every slot in use:

  paged_write       prompts' k and v into the pages                     (cdx_paged_write)
  paged_qkv_append  a step's projection: QK norm, RoPE, k and v appended  (cdx_paged_append_fwd)
  paged_attention   softmax(scale q k^T) v over the slots in use         (cdx_paged_attention_fwd)
  paged_evict       the slots with the least accumulated weight go       (cdx_paged_evict)

and, where a call brings any number of tokens of each sequence:

  paged_reserve          pages from a pool, and the slots of the call's rows    (cdx_paged_reserve)
  paged_truncate         sequences cut, pages back to the pool                  (cdx_paged_truncate)
  paged_chunk_append     QK norm, RoPE, k and v into the slots                  (cdx_paged_chunk_append_fwd)
  paged_chunk_attention  each token over the slots up to its own                (cdx_paged_chunk_attention_fwd)

  PagedKVCache      all of it for a model: ComplexityModel.forward takes one as past_key_values

``block_table`` [B, width] and ``lengths`` [B] are int32 tensors on the device and no call waits
for their values: a slot past a sequence's capacity (width * page_size) or on a page outside the
pool is neither read nor written, and attention over such a page is NaN.  A length of 0 (or less)
is an empty sequence.  All of it can be captured into a HIP graph.
"""

from __future__ import annotations

import operator
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as nat
from ._grad import forward_only

PAGE_SIZES = (16, 32, 64, 128, 256)


def _ints(t: torch.Tensor, shape: Tuple[int, ...], like: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != like.device:
        raise ValueError(f"{what} must be an int32 tensor of shape {shape} on {like.device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _page_shapes(k_pages: torch.Tensor, v_pages: torch.Tensor, dims: int, what: str) -> None:
    if k_pages.dim() != dims or v_pages.shape != k_pages.shape:
        raise ValueError(f"{what}: k_pages and v_pages must share one shape of {dims} dimensions, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError(f"{what}: the pages must be contiguous (they are written in place)")
    page, D = k_pages.shape[-2:]
    if page not in PAGE_SIZES:
        raise ValueError(f"{what}: page size {page} is not one of {PAGE_SIZES}")
    if D % 8 != 0 or not 0 < D <= 128:
        raise ValueError(f"{what}: head dim {D} must be a multiple of 8 up to 128")


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, dims: int, what: str) -> torch.Tensor:
    """The block table with unit stride, after checks of the cache's tensors."""
    _page_shapes(k_pages, v_pages, dims, what)
    if table.dtype != torch.int32 or table.dim() != 2 or table.device != k_pages.device:
        raise ValueError(f"{what}: block_table must be an int32 tensor [sequences, pages] on {k_pages.device}, got "
                         f"{table.dtype} {tuple(table.shape)} on {table.device}")
    return table if table.stride(-1) == 1 and (table.shape[0] == 1 or table.stride(0) >= table.shape[1]) \
        else table.contiguous()


def _ld(table: torch.Tensor) -> int:
    return max(table.shape[1], table.stride(0)) if table.shape[0] > 1 else table.shape[1]


def _rotary(cos_sin: torch.Tensor, D: int, what: str) -> None:
    if cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.dim() != 3 \
            or tuple(cos_sin.shape[1:]) != (D // 2, 2) or cos_sin.shape[0] == 0:
        raise ValueError(f"{what}: cos_sin must be a contiguous fp32 table [positions, {D // 2}, 2]")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous at a 16-byte address."""
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def paged_qkv_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                     lengths: torch.Tensor, positions: torch.Tensor, num_heads: int, cos_sin: torch.Tensor,
                     q_norm_w: Optional[torch.Tensor] = None, k_norm_w: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> torch.Tensor:
    """q [B, num_heads, D] of one new token per sequence, its k and v appended to the pages.

    ``qkv`` [B, (num_heads + 2 nkv) D] is the packed projection (mu_qkv_project's columns), bf16
    or fp32.  q and k are normalised per head (weights [D], or neither) and rotated at
    ``positions`` [B] of the fp32 table ``cos_sin`` [n_pos, D/2, 2] (RotaryEmbedding.cos_sin_table; a
    position outside it gives NaN).  k and v go to slot ``lengths - 1``: the lengths count the
    new token already.  Replaces the torch.cat and the norms of core/attention.py:138-161."""
    fast = nat.host()
    if fast is not None:
        q = fast.paged_append(qkv, k_pages, v_pages, block_table, lengths, positions, num_heads, cos_sin, q_norm_w,
                              k_norm_w, eps)
        if q is not None:
            return q
    what = "paged_qkv_append"
    forward_only(what, qkv, k_pages, v_pages, q_norm_w, k_norm_w)
    nat.require_device(k_pages, v_pages, q_norm_w, k_norm_w, what=what)
    nat.require_device(qkv, k_pages, block_table, lengths, positions, cos_sin, dtype=None, what=what)
    table = _pages(k_pages, v_pages, block_table, 4, what)
    pages, nkv, page, D = k_pages.shape
    B, N = table.shape[0], (num_heads + 2 * nkv) * D
    if num_heads <= 0 or nkv == 0 or num_heads % nkv != 0:
        raise ValueError(f"{what}: {num_heads} query heads over {nkv} KV heads")
    if qkv.dtype not in (torch.bfloat16, torch.float32) or tuple(qkv.shape) != (B, N):
        raise ValueError(f"{what}: qkv must be bf16 or fp32 [{B}, {N}], got {qkv.dtype} {tuple(qkv.shape)}")
    _rotary(cos_sin, D, what)
    if (q_norm_w is None) != (k_norm_w is None):
        raise ValueError(f"{what}: pass both QK norm weights or neither")
    if q_norm_w is not None:
        if q_norm_w.numel() != D or k_norm_w.numel() != D:
            raise ValueError(f"{what}: the QK norm weights must have {D} elements")
        q_norm_w, k_norm_w = _aligned(q_norm_w), _aligned(k_norm_w)
    lengths = _ints(lengths, (B,), qkv, f"{what}: lengths")
    positions = _ints(positions, (B,), qkv, f"{what}: positions")
    ld = qkv.stride(0) if B > 1 else N
    if qkv.stride(-1) != 1 or ld < N or ld % 8 != 0 or qkv.data_ptr() % 16 != 0:
        qkv, ld = _aligned(qkv), N
    cos_sin = _aligned(cos_sin)
    q = torch.empty(B, num_heads, D, dtype=torch.bfloat16, device=qkv.device)
    with nat.on_device(qkv), nat.launch_region("paged_append", qkv.device, B=B, nq=num_heads, nkv=nkv, D=D):
        nat.check(nat.lib().cdx_paged_append_fwd(
            qkv.data_ptr(), qkv.dtype == torch.float32, ld, B, num_heads, nkv, D, nat.ptr(q_norm_w), nat.ptr(k_norm_w),
            float(eps), cos_sin.data_ptr(), cos_sin.shape[0], lengths.data_ptr(), positions.data_ptr(),
            table.data_ptr(), _ld(table), table.shape[1], pages, page, k_pages.data_ptr(), v_pages.data_ptr(),
            q.data_ptr(), nat.stream_of(qkv)), "cdx_paged_append_fwd")
    return q


def paged_write(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                block_table: torch.Tensor, lengths: torch.Tensor) -> None:
    """Prompts' k and v [B, nkv, S, D] (normalised and rotated: mu_qkv_rope's, qkv_cache's) into the
    pages: rows t < lengths[b] (all S of them at most) to slot t."""
    fast = nat.host()
    if fast is not None and fast.paged_write(k, v, k_pages, v_pages, block_table, lengths):
        return
    what = "paged_write"
    forward_only(what, k, v, k_pages, v_pages)
    nat.require_device(k, v, k_pages, v_pages, what=what)
    nat.require_device(k, block_table, lengths, dtype=None, what=what)
    table = _pages(k_pages, v_pages, block_table, 4, what)
    pages, nkv, page, D = k_pages.shape
    B = table.shape[0]
    if k.dim() != 4 or k.shape != v.shape or (k.shape[0], k.shape[1], k.shape[3]) != (B, nkv, D):
        raise ValueError(f"{what}: k and v must be [{B}, {nkv}, S, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    lengths = _ints(lengths, (B,), k, f"{what}: lengths")
    k, v = _aligned(k), _aligned(v)
    with nat.on_device(k), nat.launch_region("paged_write", k.device, B=B, S=k.shape[2], nkv=nkv, D=D):
        nat.check(nat.lib().cdx_paged_write(
            k.data_ptr(), v.data_ptr(), B, nkv, k.shape[2], D, lengths.data_ptr(), table.data_ptr(), _ld(table),
            table.shape[1], pages, page, k_pages.data_ptr(), v_pages.data_ptr(), nat.stream_of(k)), "cdx_paged_write")


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, scale: Optional[float] = None, *, weights: Optional[torch.Tensor] = None,
                    weights_out: Optional[torch.Tensor] = None):
    """softmax(scale q k^T) v of one new token per sequence over its slots t < lengths[b], the heads
    merged: [B, nq * D].  q [B, nq, D] bf16; scale defaults to D ** -0.5.  A sequence without slots
    gives zeros.

    With ``weights`` [B, nkv, capacity] fp32, returns (out, weights + what each slot received,
    summed over the query heads of its group); ``weights_out`` may name the result's memory,
    ``weights`` itself among others."""
    if scale is None:
        scale = max(1, k_pages.shape[-1]) ** -0.5
    fast = nat.host()
    if fast is not None:
        done = fast.paged_attention(q, k_pages, v_pages, block_table, lengths, scale, weights, weights_out)
        if done is not None:
            return done if weights is not None else done[0]
    what = "paged_attention"
    forward_only(what, q, k_pages, v_pages, weights)
    nat.require_device(q, k_pages, v_pages, what=what)
    nat.require_device(q, block_table, lengths, weights, weights_out, dtype=None, what=what)
    table = _pages(k_pages, v_pages, block_table, 4, what)
    pages, nkv, page, D = k_pages.shape
    B, cap = table.shape[0], table.shape[1] * page
    if q.dim() != 3 or (q.shape[0], q.shape[2]) != (B, D) or nkv == 0 or q.shape[1] == 0 or q.shape[1] % nkv != 0:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not match {B} sequences with {nkv} KV heads of {D}")
    nq = q.shape[1]
    if table.shape[1] == 0 or pages == 0:
        raise ValueError(f"{what}: empty block table or pool")
    lengths = _ints(lengths, (B,), q, f"{what}: lengths")
    q = _aligned(q)
    if weights is None and weights_out is not None:
        raise ValueError(f"{what}: weights_out without weights")
    if weights is not None:
        for t, name in ((weights, "weights"), (weights_out, "weights_out")):
            if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (B, nkv, cap)):
                raise ValueError(f"{what}: {name} must be fp32 [{B}, {nkv}, {cap}], got {t.dtype} {tuple(t.shape)}")
        if weights_out is None:
            weights_out = torch.empty(B, nkv, cap, dtype=torch.float32, device=q.device)
        elif not weights_out.is_contiguous():
            raise ValueError(f"{what}: weights_out must be contiguous (it is written in place)")
        weights = weights if weights.is_contiguous() else weights.contiguous()
    out = torch.empty(B, nq * D, dtype=q.dtype, device=q.device)
    lib = nat.lib()
    with nat.on_device(q):  # (the splits, and so the size, go by the current device's CUs)
        ws = lib.cdx_paged_attention_workspace_bytes(B, nq, nkv, D, cap, weights is not None)
    work = torch.empty(ws, dtype=torch.uint8, device=q.device) if ws else None
    with nat.on_device(q), nat.launch_region("paged_attention", q.device, B=B, nq=nq, nkv=nkv, D=D):
        nat.check(lib.cdx_paged_attention_fwd(
            q.data_ptr(), B, nq, nkv, D, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), _ld(table),
            table.shape[1], pages, page, lengths.data_ptr(), float(scale),
            out.data_ptr(), nat.ptr(weights), nat.ptr(weights_out), nat.ptr(work), ws, nat.stream_of(q)),
            "cdx_paged_attention_fwd")
    return out if weights is None else (out, weights_out)


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                positions: torch.Tensor, weights: torch.Tensor, slot_positions: torch.Tensor, keep: int, recent: int
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence of more than ``keep`` slots to ``keep``: of each head, the slots whose
    position exceeds positions[b] - recent stay, then those of the largest accumulated weight
    (equal ones by lower slot).

    k_pages, v_pages [layers, pages, nkv, page_size, D] or without the layers; weights (fp32) and
    slot_positions (int32) [(layers,) B, nkv, capacity]; lengths and positions [B], of the newest
    tokens.  Kept rows from slot ``keep`` on move into the evicted slots below it, in the pages;
    returns the new (lengths, weights, slot_positions), with 0 and -1 past the lengths.  The pages
    of a sequence that is cut must not be another's too."""
    fast = nat.host()
    if fast is not None and type(keep) is int and type(recent) is int:
        new = fast.paged_evict(k_pages, v_pages, block_table, lengths, positions, weights, slot_positions, keep, recent)
        if new is not None:
            return new
    what = "paged_evict"
    forward_only(what, k_pages, v_pages, weights)
    nat.require_device(k_pages, v_pages, what=what)
    nat.require_device(k_pages, block_table, lengths, positions, weights, slot_positions, dtype=None, what=what)
    dims = 5 if k_pages.dim() == 5 else 4
    table = _pages(k_pages, v_pages, block_table, dims, what)
    layers = k_pages.shape[0] if dims == 5 else 1
    pages, nkv, page, D = k_pages.shape[-4:]
    B, cap = table.shape[0], table.shape[1] * page
    shape = ((layers,) if dims == 5 else ()) + (B, nkv, cap)
    if isinstance(keep, bool) or isinstance(recent, bool) or int(keep) != keep or int(recent) != recent \
            or keep <= 0 or not 0 <= recent <= keep:
        raise ValueError(f"{what}: keep={keep} must be a positive integer and recent={recent} lie in 0 .. keep")
    keep, recent = int(keep), int(recent)
    if weights.dtype != torch.float32 or tuple(weights.shape) != shape:
        raise ValueError(f"{what}: weights must be fp32 {shape}, got {weights.dtype} {tuple(weights.shape)}")
    weights = weights if weights.is_contiguous() else weights.contiguous()
    slot_positions = _ints(slot_positions, shape, k_pages, f"{what}: slot_positions")
    lengths, positions = (_ints(t, (B,), k_pages, f"{what}: {n}") for t, n in
                          ((lengths, "lengths"), (positions, "positions")))
    if nkv == 0 or table.shape[1] == 0 or pages == 0 or layers == 0 or B == 0:
        raise ValueError(f"{what}: empty cache")
    new = (torch.empty_like(lengths), torch.empty_like(weights), torch.empty_like(slot_positions))
    lib = nat.lib()
    ws = lib.cdx_paged_evict_workspace_bytes(layers, B, nkv, cap, keep)
    work = torch.empty(ws, dtype=torch.uint8, device=k_pages.device)
    with nat.on_device(k_pages), nat.launch_region("paged_evict", k_pages.device, layers=layers, B=B, nkv=nkv, D=D):
        nat.check(lib.cdx_paged_evict(
            layers, B, nkv, D, lengths.data_ptr(), positions.data_ptr(), table.data_ptr(), _ld(table), table.shape[1],
            pages, page, k_pages.data_ptr(), v_pages.data_ptr(), weights.data_ptr(), slot_positions.data_ptr(),
            keep, recent, *(t.data_ptr() for t in new), work.data_ptr(), ws, nat.stream_of(k_pages)),
            "cdx_paged_evict")
    return new


class PagedRows(NamedTuple):
    """What ``paged_reserve`` says of a call's rows; all on the device."""
    starts: torch.Tensor                # [B] int32: the first row of each sequence
    counts: torch.Tensor                # [B] int32: its new tokens, 0 where they were refused
    lengths: torch.Tensor               # [B] int32: its slots in use, the new ones' counted
    positions: torch.Tensor             # [B] int32: of its newest token
    free_count: Optional[torch.Tensor]  # [1] int32: pages left in the pool
    row_slots: torch.Tensor             # [rows] int64: page * page_size + row in the page, or -1
    row_positions: torch.Tensor         # [rows] int32, or -1


def _pool(free_pages: torch.Tensor, free_count: torch.Tensor, like: torch.Tensor, what: str) -> None:
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous() \
            or free_pages.device != like.device:
        raise ValueError(f"{what}: free_pages must be a contiguous int32 list on {like.device}, got {free_pages.dtype} "
                         f"{tuple(free_pages.shape)} on {free_pages.device}")
    if free_count.dtype != torch.int32 or tuple(free_count.shape) != (1,) or free_count.device != like.device:
        raise ValueError(f"{what}: free_count must be one int32 on {like.device}, got {free_count.dtype} "
                         f"{tuple(free_count.shape)} on {free_count.device}")


def _table_rows(table: torch.Tensor, page_size: int, what: str, written: bool) -> None:
    """Checks of a block table that is taken without its pages."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"{what}: page size {page_size} is not one of {PAGE_SIZES}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] == 0:
        raise ValueError(f"{what}: block_table must be an int32 tensor [sequences, pages], got {table.dtype} "
                         f"{tuple(table.shape)}")
    if written and not (table.shape[1] <= 1 or table.stride(1) == 1) or \
            written and table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        raise ValueError(f"{what}: block_table needs rows of its own with unit stride (it is written in place), got "
                         f"strides {table.stride()}")


def paged_reserve(counts: torch.Tensor, lengths: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                  page_size: int, rows: int, *, stride: Optional[int] = None,
                  free_pages: Optional[torch.Tensor] = None, free_count: Optional[torch.Tensor] = None) -> PagedRows:
    """Room for ``counts`` [B] new tokens of each sequence behind its ``lengths`` [B] slots, and where each of
    a call's ``rows`` rows goes.  The rows lie one sequence behind the other, or with ``stride`` those of
    sequence b from row b * stride on (a padded batch).

    With a pool, the pages that a sequence lacks are taken from the end of ``free_pages``, a list whose
    first ``free_count`` [1] entries are pages that nobody has, and written into ``block_table``; without
    one the table names every page already.  A sequence gets all of its tokens or none: none if
    its rows or its capacity do not suffice, or if fewer pages are left than it and the sequences
    before it ask for (one that needs no page is served all the same).

    Nothing but the table is changed: the returned lengths, positions (of the newest tokens) and free_count
    are the new ones, and a call that goes on with the old ones has undone it."""
    fast = nat.host()
    if fast is not None and type(page_size) is int and type(rows) is int and (stride is None or type(stride) is int):
        done = fast.paged_reserve(counts, lengths, positions, block_table, page_size, rows, stride, free_pages,
                                  free_count)
        if done is not None:
            return PagedRows(*done)
    what = "paged_reserve"
    nat.require_device(block_table, counts, lengths, positions, free_pages, free_count, dtype=None, what=what)
    _table_rows(block_table, page_size, what, True)
    B, width = block_table.shape
    if rows < 0 or rows >= 2 ** 31 - 4096:
        raise ValueError(f"{what}: rows={rows} is out of range")
    if stride is not None and not 0 < stride < 2 ** 31:
        raise ValueError(f"{what}: stride={stride} must be positive (None: rows one behind the other)")
    if (free_pages is None) != (free_count is None):
        raise ValueError(f"{what}: pass both free_pages and free_count or neither")
    if free_pages is not None:
        _pool(free_pages, free_count, block_table, what)
    counts, lengths, positions = (_ints(t, (B,), block_table, f"{what}: {n}") for t, n in
                                  ((counts, "counts"), (lengths, "lengths"), (positions, "positions")))
    dev = block_table.device
    small = torch.empty(4 * B + 1, dtype=torch.int32, device=dev)
    starts, new_counts = small[:B], small[B:2 * B]
    new_lengths, new_positions, new_free = small[2 * B:3 * B], small[3 * B:4 * B], small[4 * B:]
    row_slots = torch.empty(rows, dtype=torch.int64, device=dev)
    row_positions = torch.empty(rows, dtype=torch.int32, device=dev)
    pool = free_pages is not None
    with nat.on_device(block_table), nat.launch_region("paged_reserve", dev, B=B, rows=rows):
        nat.check(nat.lib().cdx_paged_reserve(
            counts.data_ptr(), lengths.data_ptr(), positions.data_ptr(), B, stride or 0, rows, block_table.data_ptr(),
            _ld(block_table), width, page_size, nat.ptr(free_pages), free_pages.numel() if pool else 0,
            nat.ptr(free_count), starts.data_ptr(), new_counts.data_ptr(), new_lengths.data_ptr(),
            new_positions.data_ptr(), new_free.data_ptr() if pool else None, row_slots.data_ptr(),
            row_positions.data_ptr(), nat.stream_of(block_table)), "cdx_paged_reserve")
    return PagedRows(starts, new_counts, new_lengths, new_positions, new_free if pool else None, row_slots,
                     row_positions)


def paged_truncate(to: torch.Tensor, lengths: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                   page_size: int, free_pages: torch.Tensor, free_count: torch.Tensor
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence of more than ``to`` [B] slots to that many and give the pages behind them back to
    the pool (``free_pages``, in place): 0 for a sequence that has ended, fewer tokens for one whose
    speculated ones were not accepted.  Returns the new (lengths, positions, free_count).

    The pages must be the sequence's own.  The table keeps its entries: those past the new length name
    pages that may be another's from then on."""
    fast = nat.host()
    if fast is not None and type(page_size) is int:
        done = fast.paged_truncate(to, lengths, positions, block_table, page_size, free_pages, free_count)
        if done is not None:
            return done
    what = "paged_truncate"
    nat.require_device(block_table, to, lengths, positions, free_pages, free_count, dtype=None, what=what)
    _table_rows(block_table, page_size, what, False)
    table = block_table if block_table.stride(-1) == 1 and (
        block_table.shape[0] == 1 or block_table.stride(0) >= block_table.shape[1]) else block_table.contiguous()
    B, width = table.shape
    _pool(free_pages, free_count, table, what)
    to, lengths, positions = (_ints(t, (B,), table, f"{what}: {n}") for t, n in
                              ((to, "to"), (lengths, "lengths"), (positions, "positions")))
    small = torch.empty(2 * B + 1, dtype=torch.int32, device=table.device)
    new = small[:B], small[B:2 * B], small[2 * B:]
    with nat.on_device(table), nat.launch_region("paged_truncate", table.device, B=B):
        nat.check(nat.lib().cdx_paged_truncate(
            to.data_ptr(), lengths.data_ptr(), positions.data_ptr(), B, table.data_ptr(), _ld(table), width, page_size,
            free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), *(t.data_ptr() for t in new),
            nat.stream_of(table)), "cdx_paged_truncate")
    return new


def paged_chunk_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, row_slots: torch.Tensor,
                       row_positions: torch.Tensor, num_heads: int, cos_sin: torch.Tensor,
                       q_norm_w: Optional[torch.Tensor] = None, k_norm_w: Optional[torch.Tensor] = None,
                       eps: float = 1e-6) -> torch.Tensor:
    """q [rows, num_heads, D] of a call's new tokens, their k and v written to the slots ``row_slots`` [rows] of
    the pages (paged_reserve's): what paged_qkv_append does for one token per sequence, at the positions
    ``row_positions`` [rows].  A row without a slot gives zeros and is not stored."""
    fast = nat.host()
    if fast is not None:
        q = fast.paged_chunk_append(qkv, k_pages, v_pages, row_slots, row_positions, num_heads, cos_sin, q_norm_w,
                                    k_norm_w, eps)
        if q is not None:
            return q
    what = "paged_chunk_append"
    forward_only(what, qkv, k_pages, v_pages, q_norm_w, k_norm_w)
    nat.require_device(k_pages, v_pages, q_norm_w, k_norm_w, what=what)
    nat.require_device(qkv, k_pages, row_slots, row_positions, cos_sin, dtype=None, what=what)
    _page_shapes(k_pages, v_pages, 4, what)
    pages, nkv, page, D = k_pages.shape
    R, N = qkv.shape[0] if qkv.dim() == 2 else -1, (num_heads + 2 * nkv) * D
    if num_heads <= 0 or nkv == 0 or num_heads % nkv != 0:
        raise ValueError(f"{what}: {num_heads} query heads over {nkv} KV heads")
    if qkv.dtype not in (torch.bfloat16, torch.float32) or qkv.dim() != 2 or qkv.shape[1] != N:
        raise ValueError(f"{what}: qkv must be bf16 or fp32 [rows, {N}], got {qkv.dtype} {tuple(qkv.shape)}")
    _rotary(cos_sin, D, what)
    if (q_norm_w is None) != (k_norm_w is None):
        raise ValueError(f"{what}: pass both QK norm weights or neither")
    if q_norm_w is not None:
        if q_norm_w.numel() != D or k_norm_w.numel() != D:
            raise ValueError(f"{what}: the QK norm weights must have {D} elements")
        q_norm_w, k_norm_w = _aligned(q_norm_w), _aligned(k_norm_w)
    if row_slots.dtype != torch.int64 or tuple(row_slots.shape) != (R,):
        raise ValueError(f"{what}: row_slots must be int64 [{R}], got {row_slots.dtype} {tuple(row_slots.shape)}")
    row_slots = row_slots if row_slots.is_contiguous() else row_slots.contiguous()
    row_positions = _ints(row_positions, (R,), qkv, f"{what}: row_positions")
    ld = qkv.stride(0) if R > 1 else N
    if qkv.stride(-1) != 1 or ld < N or ld % 8 != 0 or qkv.data_ptr() % 16 != 0:
        qkv, ld = _aligned(qkv), N
    cos_sin = _aligned(cos_sin)
    q = torch.empty(R, num_heads, D, dtype=torch.bfloat16, device=qkv.device)
    with nat.on_device(qkv), nat.launch_region("paged_chunk_append", qkv.device, rows=R, nq=num_heads, nkv=nkv, D=D):
        nat.check(nat.lib().cdx_paged_chunk_append_fwd(
            qkv.data_ptr(), qkv.dtype == torch.float32, ld, R, num_heads, nkv, D, nat.ptr(q_norm_w), nat.ptr(k_norm_w),
            float(eps), cos_sin.data_ptr(), cos_sin.shape[0], row_slots.data_ptr(), row_positions.data_ptr(), pages,
            page, k_pages.data_ptr(), v_pages.data_ptr(), q.data_ptr(), nat.stream_of(qkv)),
            "cdx_paged_chunk_append_fwd")
    return q


def paged_chunk_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                          starts: torch.Tensor, counts: torch.Tensor, lengths: torch.Tensor,
                          scale: Optional[float] = None, *, max_tokens: Optional[int] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of any number of new tokens per sequence, each over the slots up to its own,
    the heads merged: [rows, nq * D].  q [rows, nq, D] bf16: sequence b's ``counts[b]`` tokens, in the last of
    its ``lengths[b]`` slots, are rows ``starts[b]`` on (paged_reserve's; the starts ascend).  scale defaults to
    D ** -0.5.  Rows of no sequence, and tokens without slots, give zeros.

    ``max_tokens``: no sequence brings more than so many, by which the kernels are chosen (the rows, if
    it is not known)."""
    if scale is None:
        scale = max(1, k_pages.shape[-1]) ** -0.5
    fast = nat.host()
    if fast is not None and (max_tokens is None or type(max_tokens) is int):
        out = fast.paged_chunk_attention(q, k_pages, v_pages, block_table, starts, counts, lengths, scale, max_tokens)
        if out is not None:
            return out
    what = "paged_chunk_attention"
    forward_only(what, q, k_pages, v_pages)
    nat.require_device(q, k_pages, v_pages, what=what)
    nat.require_device(q, block_table, starts, counts, lengths, dtype=None, what=what)
    table = _pages(k_pages, v_pages, block_table, 4, what)
    pages, nkv, page, D = k_pages.shape
    B, cap = table.shape[0], table.shape[1] * page
    if q.dim() != 3 or q.shape[2] != D or nkv == 0 or q.shape[1] == 0 or q.shape[1] % nkv != 0:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not match {nkv} KV heads of {D}")
    R, nq = q.shape[:2]
    if B == 0 or table.shape[1] == 0 or pages == 0:
        raise ValueError(f"{what}: empty block table or pool")
    if max_tokens is not None and max_tokens < 0:
        raise ValueError(f"{what}: max_tokens={max_tokens} must not be negative")
    most = R if max_tokens is None else min(R, max_tokens)
    starts, counts, lengths = (_ints(t, (B,), q, f"{what}: {n}") for t, n in
                               ((starts, "starts"), (counts, "counts"), (lengths, "lengths")))
    q = _aligned(q)
    out = torch.empty(R, nq * D, dtype=q.dtype, device=q.device)
    lib = nat.lib()
    with nat.on_device(q):  # (the splits, and so the size, go by the current device's CUs)
        ws = lib.cdx_paged_chunk_attention_workspace_bytes(R, B, nq, nkv, D, cap, most)
    work = torch.empty(ws, dtype=torch.uint8, device=q.device) if ws else None
    with nat.on_device(q), nat.launch_region("paged_chunk_attention", q.device, rows=R, B=B, nq=nq, nkv=nkv, D=D):
        nat.check(lib.cdx_paged_chunk_attention_fwd(
            q.data_ptr(), R, B, nq, nkv, D, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), _ld(table),
            table.shape[1], pages, page, starts.data_ptr(), counts.data_ptr(), lengths.data_ptr(), most, float(scale),
            out.data_ptr(), nat.ptr(work), ws, nat.stream_of(q)), "cdx_paged_chunk_attention_fwd")
    return out


def _capturing(t: torch.Tensor) -> bool:
    """Whether work on t is being captured into a graph."""
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


def _to_device(t: torch.Tensor, device) -> torch.Tensor:
    """t on the device, without a wait: the host's is copied from pinned memory, which the allocator keeps
    until the copy is done."""
    return t if t.is_cuda or torch.device(device).type != "cuda" else t.pin_memory().to(device, non_blocking=True)


class PagedLayer(NamedTuple):
    """One layer of a PagedKVCache, as ComplexityAttention takes it for past_key_value."""
    cache: "PagedKVCache"
    index: int


class PagedKVCache:
    """The KV cache of ``batch_size`` sequences of a ComplexityModel, in pages:
    ``model(ids, past_key_values=cache)`` first takes the prompts, [B, S], then one token per
    sequence and call, [B, 1], and every token attends to all before it (a list of k and v keeps
    the reference's top-left mask instead).

    A call with ``token_counts`` brings any number of tokens of each sequence, none among them: second turns,
    prompts in pieces, prompts of some beside steps of others, speculated tokens at once; ids [B, S],
    right-padded, or [tokens], one sequence behind the other.  ``truncate`` takes tokens back,
    ``release`` empties sequences, whose places others can take.

    Each sequence has room for ``max_length`` tokens (rounded up to whole pages).  With ``pages`` the
    sequences share a pool of so many pages, fewer than batch_size times that: a call takes what its
    tokens need and raises if too few are left.  When the
    longest is full, a call raises, or with ``keep`` first cuts every longer sequence to ``keep``
    slots (paged_evict): the ``recent`` newest tokens (half of ``keep`` by default) stay, and those
    that the steps so far attended to most.  Positions go on counting.  A bounded cache takes its prompts and
    then one token per sequence, and has no shared pool.

    ``lengths`` and ``positions`` (of the newest tokens) live on the device; ``longest`` and ``newest``
    are the host's bounds, and nothing waits for the device but the first call of a batch whose
    bound, of right-padded prompts with prompt_lengths on the device, has reached the capacity: it reads
    how long the longest is; with token_counts on the device, or a pool, such a call reads all lengths, and
    the counts, which must fit their rows.  (For the bound, counts on the device are all rows of a sequence,
    or of the whole call if packed.)  Where it need not read them the device alone leaves out a sequence whose
    tokens do not fit: it brings none, and its rows attend to nothing.  One call at a time may use a cache.

    A call that is captured into a graph, with its counts on the device, counts on the device when it is
    replayed, not here: keep to max_length then (a token past the capacity is not stored).  Captured prompts
    begin the batch anew at every replay.  Once a call of the cache was captured, calls with token_counts, or of a
    pool, prompts, and steps that would be refused as full read the lengths first.  A captured call of one token
    each that could be a prompt or a step, replays having filled the cache or not, is refused.

    A TransformerBlock or ComplexityAttention called by itself takes ``cache[i]``, after ``begin`` has
    counted the call's tokens."""

    def __init__(self, config, batch_size: int, max_length: int, *, page_size: int = 64, keep: Optional[int] = None,
                 recent: Optional[int] = None, pages: Optional[int] = None, device="cuda"):
        nkv, D = config.num_key_value_heads, config.hidden_size // config.num_attention_heads
        if page_size not in PAGE_SIZES:
            raise ValueError(f"PagedKVCache: page size {page_size} is not one of {PAGE_SIZES}")
        if D % 8 != 0 or D > 128 or config.hidden_size % 64 != 0:
            raise ValueError(f"PagedKVCache: heads of {D} in a hidden size of {config.hidden_size} (multiples of 8 up "
                             "to 128, and of 64, are supported)")
        if batch_size <= 0 or max_length <= 0:
            raise ValueError(f"PagedKVCache: bad size {batch_size} x {max_length}")
        if any(isinstance(n, bool) or int(n) != n for n in (keep, recent) if n is not None):
            raise ValueError(f"PagedKVCache: keep={keep} and recent={recent} must be integers")
        keep, recent = (None if n is None else int(n) for n in (keep, recent))
        recent = recent if recent is not None else (keep // 2 if keep is not None else 0)
        if keep is not None and not (0 < keep < max_length and 0 <= recent <= keep):
            raise ValueError(f"PagedKVCache: keep={keep} must lie in 1 .. max_length - 1, recent={recent} in 0 .. keep")
        if pages is not None and (isinstance(pages, bool) or int(pages) != pages or not 0 < pages < 2 ** 31):
            raise ValueError(f"PagedKVCache: pages={pages} must be a positive integer")
        if pages is not None and keep is not None:
            raise ValueError("PagedKVCache: a bounded cache (keep) has pages of its own, not a pool's")
        self.batch_size, self.page_size, self.keep, self.recent = batch_size, page_size, keep, recent
        self.pages = None if pages is None else int(pages)
        width = -(-max_length // page_size)
        self.capacity = width * page_size
        # (Ordinary tensors also under inference_mode: they are written in place wherever the cache is used.)
        with torch.inference_mode(False), torch.no_grad():
            shape = (config.num_hidden_layers, self.pages or batch_size * width, nkv, page_size, D)
            self.k_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
            self.v_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
            device = self.k_pages.device
            own = torch.arange(batch_size * width, dtype=torch.int32, device=device).view(batch_size, width)
            self.block_table = own if self.pages is None else torch.full_like(own, -1)
            # The lengths, the positions, and the count of the pool's free pages, side by side as paged_reserve
            # gives the new ones.
            self._state = torch.zeros(2 * batch_size + 1, dtype=torch.int32, device=device)
            self._counts = self._state[:2 * batch_size].view(2, batch_size)
            self._undo = torch.empty_like(self._state)
            self.free_pages = self.free_count = None
            if self.pages is not None:
                self.free_pages = torch.empty(self.pages, dtype=torch.int32, device=device)
                self.free_count = self._state[2 * batch_size:]
                self._ones = torch.ones(batch_size, dtype=torch.int32, device=device)
            self._tables = {}
            self.weights = self.slot_positions = self._weights_before = None
            if keep is not None:
                shape = (shape[0], batch_size, nkv, self.capacity)
                self.weights = torch.zeros(shape, dtype=torch.float32, device=device)
                self._weights_before = torch.empty_like(self.weights)
                self.slot_positions = torch.empty(shape, dtype=torch.int32, device=device)
        self._replays = False  # whether a call was captured: its replays count on the device alone
        self.reset()

    @property
    def lengths(self) -> torch.Tensor:
        return self._counts[0]

    @property
    def positions(self) -> torch.Tensor:
        return self._counts[1]

    @property
    def step_lengths(self) -> torch.Tensor:
        """What a step of one token per sequence takes for ``lengths``: 0 where the token has no slot."""
        return self.lengths if self._step is None else self._step

    def __len__(self) -> int:
        return self.k_pages.shape[0]

    def __getitem__(self, i: int) -> PagedLayer:
        if not 0 <= i < len(self):
            raise IndexError(f"PagedKVCache: layer {i} of {len(self)}")
        return PagedLayer(self, i)

    def rotary_table(self, rotary, device) -> torch.Tensor:
        """The fp32 (cos, sin) table of a layer's rotary embedding for every position that a call can
        ask for, kept as long as the cache (a captured step reads it where it was)."""
        table = rotary.cos_sin_table(max(self.newest, self.capacity), device)
        self._tables[table.data_ptr()] = table
        return table

    def layer(self, i: int) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
        """(k_pages, v_pages, weights) of layer i."""
        return self.k_pages[i], self.v_pages[i], self.weights[i] if self.weights is not None else None

    def reset(self) -> None:
        """Empty every sequence."""
        self._captured()
        self._counts[0].zero_()
        self._counts[1].fill_(-1)
        if self.pages is not None:
            torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=self.free_pages.device, out=self.free_pages)
            self.free_count.fill_(self.pages)
        if self.weights is not None:
            self.weights.zero_()
            self.slot_positions.fill_(-1)
        self.longest = self.newest = 0  # no sequence has more slots, or has seen more tokens
        self._exact = True              # whether one has as many slots
        self._lengths = [0] * self.batch_size  # the host's, or None if it does not know them
        self.prompt = True              # what the call at hand brings
        self._step = None
        self.rows = None                # (with token_counts: where its rows go
        self.most = 0                   # and the most that a sequence has of them)
        self._before = None             # what ``cancel`` goes back to after a call that took pages
        self._saved = False             # whether _weights_before holds the weights before it

    def _captured(self) -> bool:
        """Whether the call at hand is being captured, which is noted: its replays count on the device alone."""
        capturing = _capturing(self._counts)
        self._replays |= capturing
        return capturing

    def evict(self) -> None:
        """Cut every sequence of more than ``keep`` slots to ``keep``."""
        if self.keep is None:
            raise ValueError("PagedKVCache: made without keep")
        if self.longest <= self.keep:
            return
        self._captured()
        new = paged_evict(self.k_pages, self.v_pages, self.block_table, self.lengths, self.positions, self.weights,
                          self.slot_positions, self.keep, self.recent)
        for t, n in zip((self.lengths, self.weights, self.slot_positions), new):
            t.copy_(n)
        self.longest, self._lengths = self.keep, None

    def begin(self, batch_size: int, tokens: int, prompt_lengths: Optional[torch.Tensor] = None,
              token_counts=None, packed: bool = False) -> None:
        """Make room for a call's tokens and count them: the prompts (of ``prompt_lengths`` tokens
        each, or all of them) of an empty cache, then one token per sequence; or with ``token_counts`` (integers
        [B], on the device or the host) so many of each sequence, in rows of ``tokens`` each or, ``packed``,
        one behind the other in ``tokens`` rows."""
        if batch_size != self.batch_size:
            raise ValueError(f"PagedKVCache: {batch_size} sequences in a cache of {self.batch_size}")
        if self.block_table.shape[-1] * self.page_size < self.capacity:
            raise ValueError(f"PagedKVCache: a block table {tuple(self.block_table.shape)} of pages of {self.page_size} "
                             f"has no room for {self.capacity} tokens")
        self.rows = self._before = None
        replays, capturing = self._replays, self._captured()
        if token_counts is not None:
            if self.keep is not None or prompt_lengths is not None or tokens <= 0:
                raise ValueError("PagedKVCache: token_counts in a bounded cache, beside prompt_lengths, or without rows")
            counts, known = self._integers(token_counts, "token_counts")
            most = tokens if known is None else max(0, *known)
            if known is not None:
                if min(known) < 0:
                    raise ValueError(f"PagedKVCache: token_counts {known} must not be negative")
                self._check_rows(known, tokens, packed)
            self.rows = self._reserve(counts, known, most, tokens if packed else batch_size * tokens,
                                      None if packed else tokens)
            self.most, self.prompt = most, False
            return
        more = tokens != 1 or prompt_lengths is not None
        # (Replays may have brought tokens to an empty cache; prompts are taken if the device has emptied it.)
        if not capturing and (self._replays if self.newest == 0 else more and (self._replays or not self._exact)):
            self._read_longest(self.lengths)
            self.newest = int(self.positions.max()) + 1
        if self.newest == 0:
            if capturing and replays and tokens == 1:
                raise ValueError("PagedKVCache: whether a captured call of one token each is a prompt or a step cannot "
                                 "be known, as replays may have brought tokens: give token_counts, or make a call "
                                 "first")
            if not 0 < tokens <= self.capacity:
                raise ValueError(f"PagedKVCache: prompts of {tokens} tokens in a cache of {self.capacity}")
            n, known = None, [tokens] * batch_size
            if prompt_lengths is not None:
                n = self.prompt_counts(prompt_lengths, tokens)
                known = self._known(n, "prompt_lengths")
                n = _to_device(n.to(torch.int32), self.lengths.device)
            if self.pages is not None:
                if capturing:  # (replayed prompts begin the batch anew, as they do on pages of the cache's own)
                    self._give_back(torch.zeros_like(self.lengths))
                n = torch.full_like(self.lengths, tokens) if n is None else n.to(self.lengths)
                self._reserve(n, known, tokens, batch_size * tokens, tokens)
            elif n is None:
                self._counts[0].fill_(tokens)
            else:
                self._counts[0].copy_(n)
            self._lengths = known
            torch.sub(self._counts[0], 1, out=self._counts[1])
            if self.weights is not None and capturing:  # (replays begin the batch anew)
                self.weights.zero_()
            if self.slot_positions is not None:
                at = torch.arange(self.capacity, dtype=torch.int32, device=self.slot_positions.device)
                self.slot_positions.copy_(torch.where(at < self.lengths.view(-1, 1, 1), at, -1))
            self.longest = self.newest = tokens
            self._exact = prompt_lengths is None
            if prompt_lengths is not None and known is not None:
                self.longest, self._exact = max(known), True
            self.prompt = True
            return
        if more:
            raise ValueError("PagedKVCache: after the prompts a call without token_counts takes one token per sequence "
                             "(reset() empties the cache)")
        if self.pages is not None:
            rows = self._reserve(self._ones, [1] * batch_size, 1, batch_size, None)
            # (A token that a replay finds no page for has no slot, and must not take the newest one's.)
            self._step = rows.counts * rows.lengths if self._replays else None
            self.prompt = False
            return
        if self.longest >= self.capacity and (not self._exact or self._replays) and not capturing:
            self._read_longest(self.lengths)
        if self.longest >= self.capacity:
            if self.keep is None:
                raise ValueError(f"PagedKVCache: full ({self.capacity} tokens)")
            self.evict()
        # Every layer adds to the weights in place: a call that raises is taken back from a copy (1B preset, 32
        # sequences of 2048 slots: 14 us of a step of 2.4 ms).  A step that is captured runs as a whole or not
        # at all, and makes none.
        self._saved = self.weights is not None and not capturing
        if self._saved:
            self._weights_before.copy_(self.weights)
        self._counts.add_(1)
        if self.slot_positions is not None:
            slot = self._new_slot()
            self.slot_positions.scatter_(-1, slot, self.positions.view(-1, 1, 1).expand(slot.shape))
        self.longest += 1
        self.newest += 1
        if self._lengths is not None:
            self._lengths = [n + 1 for n in self._lengths]
        self.prompt = False

    def prompt_counts(self, prompt_lengths: torch.Tensor, tokens: int) -> torch.Tensor:
        """``prompt_lengths`` [B] of prompts in ``tokens`` rows each, as int64 of 0 .. tokens."""
        if prompt_lengths.shape != (self.batch_size,) or prompt_lengths.is_floating_point() \
                or prompt_lengths.is_complex() or prompt_lengths.dtype == torch.bool:
            raise ValueError(f"PagedKVCache: prompt_lengths must be {self.batch_size} integers, got "
                             f"{prompt_lengths.dtype} {tuple(prompt_lengths.shape)}")
        return prompt_lengths.long().clamp(0, tokens)

    def _known(self, values: torch.Tensor, name: str):
        """The values as a list if they are the host's.  A graph would copy those from where they were at its
        capture."""
        if values.is_cuda:
            return None
        if _capturing(self._counts):
            raise ValueError(f"PagedKVCache: {name} of a captured call must be on {self.lengths.device}")
        return values.tolist()

    def _integers(self, values, name: str):
        """(int32 [B] on the device, the same as a list if the host has them) of a tensor or a sequence."""
        if not isinstance(values, torch.Tensor):
            values = torch.tensor([operator.index(n) for n in values], dtype=torch.int64)
        if values.shape != (self.batch_size,) or values.is_floating_point() or values.is_complex() \
                or values.dtype == torch.bool:
            raise ValueError(f"PagedKVCache: {name} must be {self.batch_size} integers, got {values.dtype} "
                             f"{tuple(values.shape)}")
        known = self._known(values, name)
        values = _to_device(values.long().clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32), self.lengths.device)
        return values.to(self.lengths.device), known

    @staticmethod
    def _check_rows(known, rows: int, packed: bool) -> None:
        if (sum(known) if packed else max(known)) > rows:
            raise ValueError(f"PagedKVCache: token_counts {known} in {rows} rows" + (" each" if not packed else ""))

    def _reserve(self, counts: torch.Tensor, known, most: int, rows: int, stride: Optional[int]) -> PagedRows:
        """Pages and rows of ``counts`` tokens (on the host ``known``, or at most ``most`` each), which are counted.
        Raises, with nothing changed, if the capacity or the pool does not suffice; a call that is being captured
        is not looked at, and tokens that do not fit are then neither counted nor stored."""
        capturing = _capturing(self._counts)
        before = (self.longest, self.newest, self._exact, self._lengths)
        lengths = self._lengths if not self._replays else None
        used = self.batch_size * -(-(self.longest + most) // self.page_size)
        if not capturing and (self._replays or self.longest + most > self.capacity
                              or (self.pages is not None and used > self.pages)):
            lengths = self.lengths.tolist() if lengths is None else lengths
            if known is None:
                known = [max(0, n) for n in counts.tolist()]
                self._check_rows(known, rows if stride is None else stride, stride is None)
            if any(c > 0 and n + c > self.capacity for n, c in zip(lengths, known)):
                raise ValueError(f"PagedKVCache: full ({self.capacity} tokens)")
            used, needed = (sum(-(-n // self.page_size) for n in ns)
                            for ns in (lengths, [n + c for n, c in zip(lengths, known)]))
            if self.pages is not None and needed > self.pages:
                raise ValueError(f"PagedKVCache: {needed - used} pages are needed, and {self.pages - used} of "
                                 f"{self.pages} are free")
        new = paged_reserve(counts, self.lengths, self.positions, self.block_table, self.page_size, rows, stride=stride,
                            free_pages=self.free_pages, free_count=self.free_count)
        self._undo.copy_(self._state)
        # (The new lengths, positions and count lie side by side.)
        n = self._state.numel() if self.pages is not None else 2 * self.batch_size
        self._state[:n].copy_(torch.as_strided(new.lengths, (n,), (1,)))
        if lengths is not None and known is not None:
            self._lengths = [n + c for n, c in zip(lengths, known)]
            self.longest, self._exact = max(self._lengths), True
        else:
            self._lengths, self._exact = None, False
            self.longest = min(self.longest + most, self.capacity)  # (tokens past it are refused)
        self.newest = self.longest  # (without a bound by weight a token's position is its slot)
        self._before = before
        return new

    def _give_back(self, to: torch.Tensor) -> None:
        """Cut the sequences of a pool to ``to`` tokens (on the device)."""
        new = paged_truncate(to, self.lengths, self.positions, self.block_table, self.page_size, self.free_pages,
                             self.free_count)
        self._state.copy_(torch.as_strided(new[0], (self._state.numel(),), (1,)))

    def truncate(self, to) -> None:
        """Cut every sequence of more than ``to`` [B] tokens (integers, on the device or the host) to its first so
        many: speculated tokens that were not accepted, 0 for a sequence that has ended.  The pages
        behind go back to the pool."""
        if self.keep is not None:
            raise ValueError("PagedKVCache: a bounded cache does not hold its tokens in order")
        to, known = self._integers(to, "to")
        self._captured()
        if self.pages is not None:
            self._give_back(to)
        else:
            gone = (self.lengths - to.clamp(min=0)).clamp(min=0)
            self._counts.sub_(gone)
        self.rows = self._before = None
        if self._replays:
            self._lengths = None
        if known is not None and (self._lengths is not None or max(known) <= 0):
            self._lengths = [max(0, min(n, t)) for n, t in zip(self._lengths or known, known)]
            self.longest, self._exact = max(self._lengths), True
            self.newest = self.longest  # (0: as after reset())
        else:
            self._lengths, self._exact = None, False

    def release(self, sequences) -> None:
        """Empty these sequences (their numbers); the pages go back to the pool."""
        to = [2 ** 31 - 1] * self.batch_size
        for i in sequences:
            if not 0 <= operator.index(i) < self.batch_size:
                raise IndexError(f"PagedKVCache: sequence {i} of {self.batch_size}")
            to[operator.index(i)] = 0
        self.truncate(to)

    def _read_longest(self, lengths: torch.Tensor) -> None:
        self.longest, self._exact = int(lengths.max()), True

    def _new_slot(self) -> torch.Tensor:
        """The slot of each sequence's newest token, by layer and head (the capacity bounds it here too:
        a replayed step may count past it)."""
        slot = (self.lengths.long() - 1).clamp(max=self.capacity - 1)
        return slot.view(-1, 1, 1).expand(*self.slot_positions.shape[:-1], 1)

    def cancel(self) -> None:
        """Take back the tokens that the last ``begin`` counted, and the weights that they gave to others (a
        call that raised).  A cut that begin made stays: the call made again would make it too."""
        if self.rows is not None or (self._before is not None and not self.prompt):
            self._state.copy_(self._undo)
            self.longest, self.newest, self._exact, self._lengths = self._before
            self.rows = self._before = None
            self.prompt = self.newest == 0
        elif self.prompt:
            self.reset()
        else:
            if self.weights is not None:
                self.slot_positions.scatter_(-1, self._new_slot(), -1)
                if self._saved:
                    self.weights.copy_(self._weights_before)
            self._counts.sub_(1)
            self.longest -= 1
            self.newest -= 1
            if self._lengths is not None:
                self._lengths = [n - 1 for n in self._lengths]
