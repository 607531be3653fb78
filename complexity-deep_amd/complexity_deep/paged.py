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
  PagedKVCache      all of it for a model: ComplexityModel.forward takes one as past_key_values

``block_table`` [B, width] and ``lengths`` [B] are int32 tensors on the device and no call waits
for their values: a slot past a sequence's capacity (width * page_size) or on a page outside the
pool is neither read nor written, and attention over such a page is NaN.  A length of 0 (or less)
is an empty sequence.  All of it can be captured into a HIP graph.
"""

from __future__ import annotations

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


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, dims: int, what: str) -> torch.Tensor:
    """The block table with unit stride, after checks of the cache's tensors."""
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


class PagedLayer(NamedTuple):
    """One layer of a PagedKVCache, as ComplexityAttention takes it for past_key_value."""
    cache: "PagedKVCache"
    index: int


class PagedKVCache:
    """The KV cache of ``batch_size`` sequences of a ComplexityModel, in pages:
    ``model(ids, past_key_values=cache)`` first takes the prompts, [B, S], then one token per
    sequence and call, [B, 1], and every token attends to all before it (a list of k and v keeps
    the reference's top-left mask instead).

    Each sequence has room for ``max_length`` tokens (rounded up to whole pages).  When the
    longest is full, a call raises, or with ``keep`` first cuts every longer sequence to ``keep``
    slots (paged_evict): the ``recent`` newest tokens (half of ``keep`` by default) stay, and those
    that the steps so far attended to most.  Positions go on counting.

    ``lengths`` and ``positions`` (of the newest tokens) live on the device; ``longest`` and ``newest``
    are the host's bounds, and nothing waits for the device but the first call of a batch whose
    bound, of right-padded prompts with prompt_lengths on the device, has reached the capacity: it reads
    how long the longest is.  One call at a time may use a cache.  A
    step that is captured into a graph counts on the device when it is replayed, not here: keep to
    max_length then (a token past the capacity is not stored).  A TransformerBlock or
    ComplexityAttention called by itself takes ``cache[i]``, after ``begin`` has counted the call's
    tokens."""

    def __init__(self, config, batch_size: int, max_length: int, *, page_size: int = 64, keep: Optional[int] = None,
                 recent: Optional[int] = None, device="cuda"):
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
        self.batch_size, self.page_size, self.keep, self.recent = batch_size, page_size, keep, recent
        width = -(-max_length // page_size)
        self.capacity = width * page_size
        # (Ordinary tensors also under inference_mode: they are written in place wherever the cache is used.)
        with torch.inference_mode(False), torch.no_grad():
            shape = (config.num_hidden_layers, batch_size * width, nkv, page_size, D)
            self.k_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
            self.v_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
            device = self.k_pages.device
            pages = torch.arange(batch_size * width, dtype=torch.int32, device=device)
            self.block_table = pages.view(batch_size, width)
            self._counts = torch.zeros(2, batch_size, dtype=torch.int32, device=device)
            self._tables = {}
            self.weights = self.slot_positions = self._weights_before = None
            if keep is not None:
                shape = (shape[0], batch_size, nkv, self.capacity)
                self.weights = torch.zeros(shape, dtype=torch.float32, device=device)
                self._weights_before = torch.empty_like(self.weights)
                self.slot_positions = torch.empty(shape, dtype=torch.int32, device=device)
        self.reset()

    @property
    def lengths(self) -> torch.Tensor:
        return self._counts[0]

    @property
    def positions(self) -> torch.Tensor:
        return self._counts[1]

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
        self._counts[0].zero_()
        self._counts[1].fill_(-1)
        if self.weights is not None:
            self.weights.zero_()
            self.slot_positions.fill_(-1)
        self.longest = self.newest = 0  # no sequence has more slots, or has seen more tokens
        self._exact = True              # whether one has as many slots
        self.prompt = True              # what the call at hand brings
        self._saved = False             # whether _weights_before holds the weights before it

    def evict(self) -> None:
        """Cut every sequence of more than ``keep`` slots to ``keep``."""
        if self.keep is None:
            raise ValueError("PagedKVCache: made without keep")
        if self.longest <= self.keep:
            return
        new = paged_evict(self.k_pages, self.v_pages, self.block_table, self.lengths, self.positions, self.weights,
                          self.slot_positions, self.keep, self.recent)
        for t, n in zip((self.lengths, self.weights, self.slot_positions), new):
            t.copy_(n)
        self.longest = self.keep

    def begin(self, batch_size: int, tokens: int, prompt_lengths: Optional[torch.Tensor] = None) -> None:
        """Make room for a call's tokens and count them: the prompts (of ``prompt_lengths`` tokens
        each, or all of them) of an empty cache, then one token per sequence."""
        if batch_size != self.batch_size:
            raise ValueError(f"PagedKVCache: {batch_size} sequences in a cache of {self.batch_size}")
        if self.block_table.shape[-1] * self.page_size < self.capacity:
            raise ValueError(f"PagedKVCache: a block table {tuple(self.block_table.shape)} of pages of {self.page_size} "
                             f"has no room for {self.capacity} tokens")
        if self.newest == 0:
            if not 0 < tokens <= self.capacity:
                raise ValueError(f"PagedKVCache: prompts of {tokens} tokens in a cache of {self.capacity}")
            if prompt_lengths is None:
                self._counts[0].fill_(tokens)
            else:
                if prompt_lengths.shape != (batch_size,) or prompt_lengths.is_floating_point():
                    raise ValueError(f"PagedKVCache: prompt_lengths must be {batch_size} integers, got "
                                     f"{prompt_lengths.dtype} {tuple(prompt_lengths.shape)}")
                self._counts[0].copy_(prompt_lengths.clamp(0, tokens))
            torch.sub(self._counts[0], 1, out=self._counts[1])
            if self.slot_positions is not None:
                at = torch.arange(self.capacity, dtype=torch.int32, device=self.slot_positions.device)
                self.slot_positions.copy_(torch.where(at < self.lengths.view(-1, 1, 1), at, -1))
            self.longest = self.newest = tokens
            self._exact = prompt_lengths is None
            if prompt_lengths is not None and not prompt_lengths.is_cuda:
                self._read_longest(prompt_lengths.clamp(0, tokens))
            self.prompt = True
            return
        if tokens != 1 or prompt_lengths is not None:
            raise ValueError("PagedKVCache: after the prompts a call takes one token per sequence (reset() empties the "
                             "cache)")
        capturing = self._counts.is_cuda and torch.cuda.is_current_stream_capturing()
        if self.longest >= self.capacity and not self._exact and not capturing:
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
        self.prompt = False

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
        if self.prompt:
            self.reset()
        else:
            if self.weights is not None:
                self.slot_positions.scatter_(-1, self._new_slot(), -1)
                if self._saved:
                    self.weights.copy_(self._weights_before)
            self._counts.sub_(1)
            self.longest -= 1
            self.newest -= 1
